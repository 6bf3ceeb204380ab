// top_logprobs — the k largest logits of every row (ties to the lowest index)
// with their logprobs under the temperature-scaled softmax:
//
//   lse = log sum_j exp(z_j / T),   logprob_i = z_i / T - lse
//
// The order is taken on the raw logits, so scaling cannot make new ties.
#include "vocab_rows.cuh"

namespace libra {
namespace vocab {

constexpr int kTopThreads = 512;
constexpr int kTopMax = 256;

struct TopShared {
  MaxSum red[kTopThreads / 32];
  unsigned hist[256];
  unsigned long long best[kTopMax];  // key << 32 | ~index: larger is better
  int n, bin, left;
  int wsum[kTopThreads / 32];
};

// Key of the k-th largest element: radix select from the most significant byte.
template <typename T>
__device__ uint32_t kth_key(const T* z, int V, int k, TopShared& sh) {
  uint32_t prefix = 0u, mask = 0u;
  int left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kTopThreads) sh.hist[i] = 0u;
    __syncthreads();
    for (int j = threadIdx.x; j < V; j += kTopThreads) {
      const uint32_t key = order_key(to_f(z[j]));
      if ((key & mask) == prefix) atomicAdd(&sh.hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int above = 0, bin = 255;
      for (; bin > 0 && above + (int)sh.hist[bin] < left; --bin) above += (int)sh.hist[bin];
      sh.bin = bin;
      sh.left = left - above;
    }
    __syncthreads();
    prefix |= (uint32_t)sh.bin << shift;
    mask |= 255u << shift;
    left = sh.left;
    __syncthreads();
  }
  return prefix;
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads) top_kernel(const T* logits, int64_t ld, int V, int k,
                                                          const float* temps, float temp, int64_t* out_ids,
                                                          float* out_lp, float* out_lse) {
  __shared__ TopShared sh;
  const int row = blockIdx.x;
  const T* z = logits + (int64_t)row * ld;
  float tm = temps ? temps[row] : temp;
  if (!(tm > 0.f)) tm = 1.f;
  const float c = kLog2e / tm;
  MaxSum a = {-FLT_MAX, 0.f};
  for (int j = threadIdx.x; j < V; j += kTopThreads) add_one(a, to_f(z[j]), c);
  put_warp(a, c, sh.red);
  a = join_warps<kTopThreads / 32>(c, sh.red);
  const uint32_t kth = kth_key(z, V, k, sh);
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  for (int j = threadIdx.x; j < V; j += kTopThreads) {
    const uint32_t key = order_key(to_f(z[j]));
    if (key > kth) sh.best[atomicAdd(&sh.n, 1)] = ((unsigned long long)key << 32) | (uint32_t)~j;
  }
  __syncthreads();
  int have = sh.n;
  __syncthreads();
  // the remaining places go to the lowest indices among the ties with the k-th key
  for (int j0 = 0; j0 < V && have < k; j0 += kTopThreads) {
    const int j = j0 + threadIdx.x;
    const bool tie = j < V && order_key(to_f(z[j])) == kth;
    const unsigned ballot = __ballot_sync(0xffffffffu, tie);
    if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = __popc(ballot);
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < kTopThreads / 32; ++w) {
      if (w < (int)(threadIdx.x >> 5)) before += sh.wsum[w];
      total += sh.wsum[w];
    }
    const int at = have + before + __popc(ballot & ((1u << (threadIdx.x & 31)) - 1u));
    if (tie && at < k) sh.best[at] = ((unsigned long long)kth << 32) | (uint32_t)~j;
    have += total;
    __syncthreads();
  }
  const float log_s = logf(a.s);
  const bool none = a.s == 0.f;  // nothing but -inf
  for (int i = threadIdx.x; i < k; i += kTopThreads) {
    const unsigned long long me = sh.best[i];
    int rank = 0;
    for (int j = 0; j < k; ++j) rank += sh.best[j] > me;
    out_ids[(int64_t)row * k + rank] = (int64_t)(uint32_t)~(uint32_t)me;
    const float v = key_value((uint32_t)(me >> 32));
    out_lp[(int64_t)row * k + rank] = none ? -INFINITY : (v - a.m) / tm - log_s;
  }
  if (threadIdx.x == 0) out_lse[row] = none ? -INFINITY : a.m / tm + log_s;
}

// logits [N, V] bf16 / fp32 -> ids [N, k] int64, logprobs [N, k] fp32 (descending), lse [N] fp32.
// temps: optional fp32 [N]; a temperature that is not above 0 counts as 1.
std::vector<torch::Tensor> top_logprobs(torch::Tensor logits, int64_t k, c10::optional<torch::Tensor> temps,
                                        double temperature) {
  check_rows(logits, "top_logprobs");
  const int N = (int)logits.size(0), V = (int)logits.size(1);
  LIBRA_CHECK(k >= 1 && k <= kTopMax && k <= V, "top_logprobs: k must lie in [1, min(%d, V)]", kTopMax);
  if (temps.has_value())
    LIBRA_CHECK(vec_of(*temps, logits, at::kFloat, N), "top_logprobs: temperatures must be contiguous fp32 [N] on the "
                "logits' device");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto ids = torch::empty({N, k}, logits.options().dtype(at::kLong));
  auto lp = torch::empty({N, k}, logits.options().dtype(at::kFloat));
  auto lse = torch::empty({N}, logits.options().dtype(at::kFloat));
  if (N == 0) return {ids, lp, lse};
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const float* tp = temps.has_value() ? temps->data_ptr<float>() : nullptr;
  if (logits.scalar_type() == at::kFloat)
    top_kernel<float><<<N, kTopThreads, 0, st>>>(logits.data_ptr<float>(), logits.stride(0), V, (int)k, tp,
                                                 (float)temperature, ids.data_ptr<int64_t>(), lp.data_ptr<float>(),
                                                 lse.data_ptr<float>());
  else
    top_kernel<__nv_bfloat16><<<N, kTopThreads, 0, st>>>(
        (const __nv_bfloat16*)logits.data_ptr(), logits.stride(0), V, (int)k, tp, (float)temperature,
        ids.data_ptr<int64_t>(), lp.data_ptr<float>(), lse.data_ptr<float>());
  LIBRA_LAUNCH_CHECK();
  return {ids, lp, lse};
}

}  // namespace vocab
}  // namespace libra
