// Helpers of the kernels that move whole rows (expert_rows.cu, embedding.cu): a row is taken in vectors of 16 bytes
// where its tensor's address, stride and width allow it, else element by element.
#pragma once
#include "vocab_rows.cuh"

namespace libra {
namespace rows {

using vocab::from_f;
using vocab::to_f;

template <int V>
__device__ __forceinline__ void unpack(const uint4& a, float (&v)[V]) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
  if constexpr (V == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
  }
}
template <int V>
__device__ __forceinline__ uint4 pack(const float (&v)[V]) {
  uint32_t w[4];
  if constexpr (V == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(v[i]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The raw bits of V neighbouring elements: 16 bytes, or one element.
template <typename T, int V>
struct Bits {
  uint4 a;
  __device__ __forceinline__ void load(const T* p) { a = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void load_once(const T* p) { a = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = a; }
  __device__ __forceinline__ void store_once(T* p) const { __stcs(reinterpret_cast<uint4*>(p), a); }
  __device__ __forceinline__ void get(float (&v)[V]) const { unpack<V>(a, v); }
  __device__ __forceinline__ void set(const float (&v)[V]) { a = pack<V>(v); }
  __device__ __forceinline__ void zero() { a = make_uint4(0, 0, 0, 0); }
};
template <typename T>
struct Bits<T, 1> {
  T a;
  __device__ __forceinline__ void load(const T* p) { a = *p; }
  __device__ __forceinline__ void load_once(const T* p) { a = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = a; }
  __device__ __forceinline__ void store_once(T* p) const { *p = a; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_f(a); }
  __device__ __forceinline__ void set(const float (&v)[1]) { from_f(&a, v[0]); }
  __device__ __forceinline__ void zero() { from_f(&a, 0.f); }
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

}  // namespace rows
}  // namespace libra
