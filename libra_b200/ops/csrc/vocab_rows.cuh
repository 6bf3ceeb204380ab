// Device helpers shared by the kernels that read whole rows of vocabulary
// logits (logit_controls.cu, top_logprobs.cu, distill.cu).
//
// A row of V logits starts wherever its tensor's strides put it, so it is
// taken as a scalar head up to the next 16-byte boundary, "octets" of eight
// elements (one 16-byte load of bf16, two of fp32) and a scalar tail.
//
// Softmax statistics are a running maximum m and s = sum exp2((z - m) c) with
// c = log2(e) / T.  m starts at the lowest finite float instead of -inf: the
// difference z - m is then never inf - inf, so a -inf logit adds exactly 0, a
// row of the type's lowest value is uniform, and a row with nothing but -inf
// ends with s = 0.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cfloat>
#include <utility>

#include "common.cuh"

namespace libra {
namespace vocab {

constexpr float kLog2e = 1.4426950408889634f;

struct RowSpan {
  int head, octs, tail;
};

template <typename T>
__device__ __forceinline__ RowSpan row_span(const T* p, int V) {
  const int mis = (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
  int head = mis ? (int)(16 / sizeof(T)) - mis : 0;
  if (head > V) head = V;
  const int octs = (V - head) >> 3;
  return {head, octs, V - head - 8 * octs};
}

__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ void from_f(__nv_bfloat16* p, float x) { *p = __float2bfloat16(x); }
__device__ __forceinline__ void from_f(float* p, float x) { *p = x; }

// Raw bits of one octet.
template <typename T>
struct Oct;
template <>
struct Oct<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load_once(const __nv_bfloat16* p) { a = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct Oct<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 4);
  }
  __device__ __forceinline__ void load_once(const float* p) {
    a = __ldcs(reinterpret_cast<const float4*>(p));
    b = __ldcs(reinterpret_cast<const float4*>(p + 4));
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
};

// Eight values to a 16-byte aligned address; bf16 rounds once, to nearest even.
__device__ __forceinline__ void store_oct(__nv_bfloat16* p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ void store_oct(float* p, const float (&v)[8]) {
  __stcs(reinterpret_cast<float4*>(p), make_float4(v[0], v[1], v[2], v[3]));
  __stcs(reinterpret_cast<float4*>(p + 4), make_float4(v[4], v[5], v[6], v[7]));
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// 2^x by the hardware unit (relative error about 2^-22); 2^-inf = 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Key with the order of the float: -inf lowest, NaN above +inf, -0 = +0.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

struct MaxSum {
  float m, s;
};

__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.s * ex2((a.m - m) * c) + b.s * ex2((b.m - m) * c)};
}

__device__ __forceinline__ void add_one(MaxSum& a, float z, float c) {
  const float m = fmaxf(a.m, z);
  a.s = a.s * ex2((a.m - m) * c) + ex2((z - m) * c);
  a.m = m;
}

// Over the block; `sh` holds one entry a warp.  Every thread gets the result, and the merge order is fixed.
template <int kThreads>
__device__ __forceinline__ MaxSum block_merge(MaxSum a, float c, MaxSum* sh) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const MaxSum b = {__shfl_xor_sync(0xffffffffu, a.m, off), __shfl_xor_sync(0xffffffffu, a.s, off)};
    a = merge(a, b, c);
  }
  const int w = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) sh[w] = a;
  __syncthreads();
  a = sh[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) a = merge(a, sh[i], c);
  __syncthreads();
  return a;
}

// The share of a row that CTA `rank` of `n` takes: octets [o0, o1); rank 0 also has the head, the last one the tail.
struct Slice {
  int o0, o1;
  bool first, last;
};
__device__ __forceinline__ Slice row_slice(const RowSpan& sp, int rank, int n) {
  return {(int)((int64_t)sp.octs * rank / n), (int)((int64_t)sp.octs * (rank + 1) / n), rank == 0, rank == n - 1};
}

// Another CTA's shared memory (same cluster), after a cluster barrier.
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster(const int* p, uint32_t rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// Launch with `cluster` CTAs of grid.x to a cluster (1: an ordinary launch).
template <typename... KArgs, typename... Args>
inline void launch_cluster(void (*kern)(KArgs...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t st,
                           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    LIBRA_CHECK(e == cudaSuccess, "libra_b200: shared memory: %s", cudaGetErrorString(e));
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
  LIBRA_CHECK(e == cudaSuccess, "libra_b200: kernel launch failed: %s", cudaGetErrorString(e));
}

// Host checks shared by the three operators.
inline void check_rows(const torch::Tensor& t, const char* op) {
  LIBRA_CHECK(t.is_cuda() && t.dim() == 2 && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat),
              "%s: logits must be a 2-D bf16 or fp32 CUDA tensor", op);
  LIBRA_CHECK(t.size(1) <= 1 || t.stride(1) == 1, "%s: logits need a unit inner stride", op);
  LIBRA_CHECK(t.size(0) < (1ll << 31) && t.size(1) < (1ll << 30), "%s: logits are too large", op);
}
// `out` may be the logits themselves or memory apart from theirs, not another view of it.
inline void check_apart(const torch::Tensor& t, const torch::Tensor& out, const char* op) {
  if (t.numel() == 0) return;
  const char *a = (const char*)t.data_ptr(), *b = (const char*)out.data_ptr();
  if (a == b && t.scalar_type() == out.scalar_type() && (t.size(0) == 1 || t.stride(0) == out.stride(0))) return;
  const auto bytes = [](const torch::Tensor& x) {
    return ((x.size(0) - 1) * x.stride(0) + x.size(1)) * (int64_t)x.element_size();
  };
  LIBRA_CHECK(a + bytes(t) <= b || b + bytes(out) <= a, "%s: out may be the logits, not another view of their memory",
              op);
}
inline bool vec_of(const torch::Tensor& t, const torch::Tensor& like, at::ScalarType ty, int64_t n) {
  return t.device() == like.device() && t.scalar_type() == ty && t.is_contiguous() && t.numel() == n;
}

}  // namespace vocab
}  // namespace libra
