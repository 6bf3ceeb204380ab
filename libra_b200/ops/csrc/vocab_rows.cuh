// Device helpers shared by the kernels that read whole rows of vocabulary
// logits (logit_controls.cu, top_logprobs.cu, distill.cu).
//
// A row of V logits starts wherever its tensor's strides put it, so it is
// taken as a scalar head up to the next 16-byte boundary, "octets" of eight
// elements (one 16-byte load of bf16, two of fp32) and a scalar tail.
//
// Softmax statistics are a running reference m and s = sum exp2((z - m) c) with
// c = log2(e) / T.  m is a logit of the row; it follows the maximum only when
// that is more than 2^kSlack above it in the sum's terms, which happens once or
// twice a thread, where an exact running maximum would rescale almost every
// octet of some lane of a warp.  fp32 holds the larger sums as exactly.  m
// starts at the lowest finite float instead of -inf: the difference z - m is
// then never inf - inf, so a -inf logit adds exactly 0, a row of the type's
// lowest value is uniform, and a row with nothing but -inf ends with s = 0.
#pragma once
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cfloat>
#include <utility>

#include "common.cuh"
#include "tmap.cuh"

namespace libra {
namespace vocab {

constexpr float kSlack = 20.f;
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
  __device__ __forceinline__ float max() const {  // of the numbers in it
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&a);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
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
  __device__ __forceinline__ float max() const {
    return fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w)));
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

// Two fp32 lanes in one instruction.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 c, a, b;\n\t"
      "mov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 c, a, b;\n\t"
      "mov.b64 {%0, %1}, c;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
// exp2((v - m) c) of eight values.
__device__ __forceinline__ void exp_oct(float (&v)[8], float m, float c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 x = mul2(add2(F2{v[2 * i], v[2 * i + 1]}, F2{-m, -m}), F2{c, c});
    v[2 * i] = ex2(x.x);
    v[2 * i + 1] = ex2(x.y);
  }
}
__device__ __forceinline__ F2 sum_oct(const float (&v)[8]) {
  return add2(add2(F2{v[0], v[1]}, F2{v[2], v[3]}), add2(F2{v[4], v[5]}, F2{v[6], v[7]}));
}

struct MaxSum {
  float m, s;
};

// An octet's values into a thread's running (m, s): `lm` is their maximum, `top` is m + kSlack / c.
__device__ __forceinline__ void add_values(MaxSum& a, float& top, float (&v)[8], float lm, float c, float slack) {
  if (lm > top) {
    a.s *= ex2((a.m - lm) * c);
    a.m = lm;
    top = lm + slack;
  }
  exp_oct(v, a.m, c);
  const F2 s = sum_oct(v);
  a.s += s.x + s.y;
}

__device__ __forceinline__ void add_one(MaxSum& a, float z, float c) {
  const float m = fmaxf(a.m, z);
  a.s = a.s * ex2((a.m - m) * c) + ex2((z - m) * c);
  a.m = m;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
// Largest of the numbers (not NaN) in a warp.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Over a warp; every lane gets the same result.
__device__ __forceinline__ MaxSum warp_merge(MaxSum a, float c) {
  const float m = warp_max(a.m);
  return {m, warp_sum(__fmul_rn(a.s, ex2((a.m - m) * c)))};
}

// Over the block, as far as the warps' results in `sh`, which any warp joins with join_warps.
__device__ __forceinline__ void put_warp(MaxSum a, float c, MaxSum* sh) {
  a = warp_merge(a, c);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
}
template <int kWarps>
__device__ __forceinline__ MaxSum join_warps(float c, const MaxSum* sh) {
  const int lane = threadIdx.x & 31;
  return warp_merge(lane < kWarps ? sh[lane] : MaxSum{-FLT_MAX, 0.f}, c);
}

// The share of a row that CTA `rank` of 2^lg takes: octets [o0, o1); rank 0 also has the head, the last one the tail
// and the octets that an even split leaves over (fewer than 2^lg).
struct Slice {
  int o0, o1;
  bool first, last;
};
__device__ __forceinline__ Slice row_slice(const RowSpan& sp, int rank, int lg) {
  const int per = sp.octs >> lg;
  const bool last = rank == (1 << lg) - 1;
  return {rank * per, last ? sp.octs : (rank + 1) * per, rank == 0, last};
}
// Most octets of a slice.
inline int slice_octs(int V, int n) { return V / 8 / n + n - 1; }
inline int log2_of(int n) { return n <= 1 ? 0 : 1 + log2_of(n / 2); }

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

__device__ __forceinline__ unsigned long long ld_cluster(const unsigned long long* p, uint32_t rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_meet() {
  cluster_arrive();
  cluster_wait();
}

// 16 bytes global -> shared without a register; a thread that reads only what it copied itself needs no barrier.
__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Launch of `ctas` CTAs, `cluster` of them to a cluster (1: an ordinary launch).  pdl: the kernel may start while the
// one before it on the stream runs, and waits for it itself (pdl_wait).
template <typename... KArgs, typename... Args>
inline void launch_rows(void (*kern)(KArgs...), int64_t ctas, int threads, size_t smem, int cluster, bool pdl,
                        cudaStream_t st, Args&&... args) {
  LIBRA_CHECK(ctas < (1ll << 31), "libra_b200: too many rows for one launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  if (pdl) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  if (smem > 32 * 1024) {  // with the kernel's static part this may pass the default 48 KB
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    LIBRA_CHECK(e == cudaSuccess, "libra_b200: shared memory: %s", cudaGetErrorString(e));
  }
  if (cluster > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    LIBRA_CHECK(e == cudaSuccess, "libra_b200: cluster size: %s", cudaGetErrorString(e));
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
