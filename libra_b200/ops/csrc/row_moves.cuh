// Helpers of the kernels that move whole rows (expert_rows.cu, embedding.cu).
//
// A row of H elements is dealt to lanes(H) lanes.  Where the tensors' addresses, strides and widths allow it a lane has
// 16 neighbouring bytes (Wide); else, for odd widths, it has four elements 32 apart (Loose), so that a warp still reads
// whole sectors and has four loads a lane in flight.
#pragma once
#include "vocab_rows.cuh"

// Argument checks: ValueError in Python, as for CPU tensors.
#define ROWS_CHECK(cond, ...)                                     \
  do {                                                            \
    if (!(cond)) {                                                \
      char rows_msg_[768];                                        \
      std::snprintf(rows_msg_, sizeof(rows_msg_), __VA_ARGS__);   \
      throw std::invalid_argument(rows_msg_);                     \
    }                                                             \
  } while (0)

namespace libra {
namespace rows {

using vocab::from_f;
using vocab::to_f;

template <typename E>
struct Wide {
  using T = E;
  static constexpr int V = 16 / sizeof(T);
  uint4 a;
  static __host__ __device__ __forceinline__ int lanes(int H) { return H / V; }
  __device__ __forceinline__ void load(const T* row, int i, int) {
    a = __ldg(reinterpret_cast<const uint4*>(row) + i);
  }
  __device__ __forceinline__ void load_once(const T* row, int i, int) {
    a = __ldcs(reinterpret_cast<const uint4*>(row) + i);
  }
  __device__ __forceinline__ void store(T* row, int i, int) const { reinterpret_cast<uint4*>(row)[i] = a; }
  __device__ __forceinline__ void store_once(T* row, int i, int) const {
    __stcs(reinterpret_cast<uint4*>(row) + i, a);
  }
  __device__ __forceinline__ void zero() { a = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float (&v)[V]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 8) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        v[i] = __uint_as_float(w[i]);
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[V]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (V == 8)
        w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      else
        w[i] = __float_as_uint(v[i]);
    }
    a = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // fp32 rows beside those of T: the lane's V values of one.
  static __device__ __forceinline__ void put_f(float* row, int i, int, const float (&v)[V]) {
#pragma unroll
    for (int q = 0; q < V; q += 4)
      *reinterpret_cast<float4*>(row + i * V + q) = make_float4(v[q], v[q + 1], v[q + 2], v[q + 3]);
  }
  static __device__ __forceinline__ void sum_f(const float* row, int i, int, float (&v)[V]) {
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const float4 x = *reinterpret_cast<const float4*>(row + i * V + q);
      v[q] += x.x;
      v[q + 1] += x.y;
      v[q + 2] += x.z;
      v[q + 3] += x.w;
    }
  }
  static __device__ __forceinline__ void get_f(const float* row, int i, int, float (&v)[V]) {
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const float4 x = *reinterpret_cast<const float4*>(row + i * V + q);
      v[q] = x.x;
      v[q + 1] = x.y;
      v[q + 2] = x.z;
      v[q + 3] = x.w;
    }
  }
};

template <typename E>
struct Loose {
  using T = E;
  static constexpr int V = 4;
  T a[V];
  static __host__ __device__ __forceinline__ int lanes(int H) { return (H + 127) / 128 * 32; }
  static __device__ __forceinline__ int at(int i) { return (i >> 5) * 128 + (i & 31); }
  __device__ __forceinline__ void load(const T* row, int i, int H) {
    const int c = at(i);
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (c + 32 * q < H) a[q] = row[c + 32 * q];
  }
  __device__ __forceinline__ void load_once(const T* row, int i, int H) { load(row, i, H); }
  __device__ __forceinline__ void store(T* row, int i, int H) const {
    const int c = at(i);
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (c + 32 * q < H) row[c + 32 * q] = a[q];
  }
  __device__ __forceinline__ void store_once(T* row, int i, int H) const { store(row, i, H); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int q = 0; q < V; ++q) from_f(a + q, 0.f);
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] = to_f(a[q]);
  }
  __device__ __forceinline__ void set(const float (&v)[V]) {
#pragma unroll
    for (int q = 0; q < V; ++q) from_f(a + q, v[q]);
  }
  static __device__ __forceinline__ void put_f(float* row, int i, int H, const float (&v)[V]) {
    const int c = at(i);
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (c + 32 * q < H) row[c + 32 * q] = v[q];
  }
  static __device__ __forceinline__ void sum_f(const float* row, int i, int H, float (&v)[V]) {
    const int c = at(i);
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (c + 32 * q < H) v[q] += row[c + 32 * q];
  }
  static __device__ __forceinline__ void get_f(const float* row, int i, int H, float (&v)[V]) {
    const int c = at(i);
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] = c + 32 * q < H ? row[c + 32 * q] : 0.f;
  }
};

inline bool row_type(const torch::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat;
}
// Whether every row of t starts on 16 bytes and holds a multiple of them.
inline bool row_vectors(const torch::Tensor& t) {
  const int64_t s = t.element_size();
  return t.size(1) * s % 16 == 0 && (t.size(0) <= 1 || t.stride(0) * s % 16 == 0) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
// t itself, or a copy of it whose inner stride is one.
inline torch::Tensor unit_inner(const torch::Tensor& t) {
  return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous();
}
// go(B) with the lanes' type for t's elements.
template <typename F>
inline void by_lanes(const torch::Tensor& t, bool wide, F&& go) {
  if (t.scalar_type() == at::kFloat) {
    if (wide) go(Wide<float>());
    else go(Loose<float>());
  } else {
    if (wide) go(Wide<__nv_bfloat16>());
    else go(Loose<__nv_bfloat16>());
  }
}

}  // namespace rows
}  // namespace libra
