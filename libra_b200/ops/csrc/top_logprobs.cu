// top_logprobs — the k largest logits of every row (ties to the lowest index)
// with their logprobs under the temperature-scaled softmax:
//
//   lse = log sum_j exp(z_j / T),   logprob_i = z_i / T - lse
//
// The order is taken on the raw logits, so scaling cannot make new ties.
//
// One pass over the row gives the softmax sum and the candidates.  Every
// thread keeps the maxima of four classes of its octets.  Where each of w warps
// has k / w maxima of disjoint classes at or above b, k logits are, and b is a
// lower bound of the k-th largest; a warp finds its own by bisection without a
// barrier.  The bound is taken after the first round of loads and again a
// little later; an octet whose maximum reaches it is noted (a few hundred of 19
// thousand), and only noted octets are looked at again, against the final
// bound.  What remains, a little more than k values, is ranked by counting.
// Slices whose values defeat the bound (long ties, ascending rows, NaN) take
// an exact radix select over the slice instead.
//
// Rows are split over a cluster when there are few: every CTA then finds the
// sorted top of its slice and looks up its entries' ranks in the other lists.
#include "vocab_rows.cuh"

namespace libra {
namespace vocab {

constexpr int kTopThreads = 256;
constexpr int kTopWarps = kTopThreads / 32;
constexpr int kTopMax = 256;
constexpr int kClasses = 4;     // of octets a thread; 1024 maxima a block
constexpr int kNoted = 4096;    // octets
constexpr int kChosen = 1024;   // values at or above the final bound
constexpr uint32_t kInfKey = 0x007fffffu;  // order_key(-inf)

struct TopShared {
  unsigned long long chosen[kChosen];  // key << 32 | ~index: larger is better
  unsigned long long list[kTopMax];    // sorted top of the slice, without -inf
  union {
    int noted[kNoted];
    unsigned long long others[kTopMax * 8];  // the cluster's lists, later
  };
  unsigned hist[256];
  float bound[kTopWarps];
  MaxSum red[kTopWarps];
  MaxSum part;
  int n_noted, n_chosen, n_list, bin, left;
  int wsum[kTopWarps];
};

__device__ __forceinline__ unsigned long long entry_of(float v, int j) {
  return ((unsigned long long)order_key(v) << 32) | (uint32_t)~j;
}

// A bound b with at least k of the block's class maxima at or above it: the least over the first `warps` warps (those
// that have octets) of the largest one with k / warps of the warp's maxima at or above it, to the upper 16 bits of its
// key, which are all of a bf16 value's.  The lowest finite float if there is none above -inf.
__device__ __forceinline__ float kth_bound(const float (&cls)[kClasses], int k, int warps, TopShared& sh) {
  const int quota = (k + warps - 1) / warps;
  uint32_t key[kClasses], most = 0u, prefix = 0u;
#pragma unroll
  for (int i = 0; i < kClasses; ++i) {
    key[i] = order_key(cls[i]) >> 16;
    most = max(most, key[i]);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  for (int bit = 31 - __clz(most | 1u); bit >= 0; --bit) {
    const uint32_t trial = prefix | (1u << bit);
    int c = 0;
#pragma unroll
    for (int i = 0; i < kClasses; ++i) c += key[i] >= trial;
    if (__reduce_add_sync(0xffffffffu, c) >= quota) prefix = trial;
  }
  const int w = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) sh.bound[w] = prefix <= (kInfKey >> 16) ? -FLT_MAX : key_value(prefix << 16);
  __syncthreads();
  float b = sh.bound[0];
  for (int i = 1; i < warps; ++i) b = fminf(b, sh.bound[i]);
  __syncthreads();
  return b;
}

// The slice's exact top (at most k) into sh.chosen, by radix select on the key from its most significant byte and the
// lowest indices among the ties with the k-th.  [lo, hi): the slice's tokens.
template <typename T>
__device__ int exact_top(const T* z, int lo, int hi, int k, TopShared& sh) {
  k = min(k, hi - lo);
  uint32_t kth = 0u, mask = 0u;
  int left = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kTopThreads) sh.hist[i] = 0u;
    __syncthreads();
    for (int j = lo + threadIdx.x; j < hi; j += kTopThreads) {
      const uint32_t key = order_key(to_f(z[j]));
      if ((key & mask) == kth) atomicAdd(&sh.hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int above = 0, bin = 255;
      for (; bin > 0 && above + (int)sh.hist[bin] < left; --bin) above += (int)sh.hist[bin];
      sh.bin = bin;
      sh.left = left - above;
    }
    __syncthreads();
    kth |= (uint32_t)sh.bin << shift;
    mask |= 255u << shift;
    left = sh.left;
    __syncthreads();
  }
  if (threadIdx.x == 0) sh.n_chosen = 0;
  __syncthreads();
  for (int j = lo + threadIdx.x; j < hi; j += kTopThreads) {
    const float v = to_f(z[j]);
    if (order_key(v) > kth) sh.chosen[atomicAdd(&sh.n_chosen, 1)] = entry_of(v, j);
  }
  __syncthreads();
  int have = sh.n_chosen;
  for (int j0 = lo; j0 < hi && have < k && kth > kInfKey; j0 += kTopThreads) {
    const int j = j0 + threadIdx.x;
    const float v = j < hi ? to_f(z[j]) : 0.f;
    const bool tie = j < hi && order_key(v) == kth;
    const unsigned ballot = __ballot_sync(0xffffffffu, tie);
    if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = __popc(ballot);
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < kTopWarps; ++w) {
      if (w < (int)(threadIdx.x >> 5)) before += sh.wsum[w];
      total += sh.wsum[w];
    }
    const int at = have + before + __popc(ballot & ((1u << (threadIdx.x & 31)) - 1u));
    if (tie && at < k) sh.chosen[at] = entry_of(v, j);
    have += total;
    __syncthreads();
  }
  return min(have, k);
}

template <typename T>
__global__ void __launch_bounds__(kTopThreads, 4) top_kernel(const T* logits, int64_t ld, int V, int lg, int k,
                                                             const float* temps, float temp, int64_t* out_ids,
                                                             float* out_lp, float* out_lse) {
  extern __shared__ __align__(16) unsigned char top_smem[];
  TopShared& sh = *reinterpret_cast<TopShared*>(top_smem);
  const int n = 1 << lg, row = blockIdx.x >> lg, rank = blockIdx.x & (n - 1), t = threadIdx.x;
  const T* z = logits + (int64_t)row * ld;
  const RowSpan sp = row_span(z, V);
  const Slice sl = row_slice(sp, rank, lg);
  float tm = temps ? temps[row] : temp;
  if (!(tm > 0.f)) tm = 1.f;
  const float c = fminf(kLog2e / tm, FLT_MAX), slack = kSlack / c;  // (a tiny temperature is its limit, one-hot)
  if (t == 0) sh.n_noted = sh.n_chosen = 0;
  constexpr int kU = kClasses;
  const T* body = z + sp.head;
  Oct<T> v[kU];
  float cls[kClasses];
#pragma unroll
  for (int u = 0; u < kU; ++u) cls[u] = -INFINITY;
  int o = sl.o0 + t;
#pragma unroll
  for (int u = 0; u < kU; ++u)
    if (o + u * kTopThreads < sl.o1) {
      v[u].load_once(body + 8 * (int64_t)(o + u * kTopThreads));
      cls[u] = v[u].max();
    }
  const int warps = max(1, min(kTopWarps, (sl.o1 - sl.o0 + 31) >> 5));
  float bound = kth_bound(cls, k, warps, sh);
  MaxSum r = {-FLT_MAX, 0.f};
  float top = -FLT_MAX;
  int round = 0;
  const int rounds = (sl.o1 - sl.o0 + kU * kTopThreads - 1) / (kU * kTopThreads);
  for (; round < rounds; ++round, o += kU * kTopThreads) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (o + u * kTopThreads < sl.o1) {
        const float lm = v[u].max();
        cls[u] = fmaxf(cls[u], lm);
        if (lm >= bound) {
          const int at = atomicAdd(&sh.n_noted, 1);
          if (at < kNoted) sh.noted[at] = o + u * kTopThreads;
        }
        float f[8];
        v[u].get(f);
        add_values(r, top, f, lm, c, slack);
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (o + (u + kU) * kTopThreads < sl.o1) v[u].load_once(body + 8 * (int64_t)(o + (u + kU) * kTopThreads));
    if (round == 2 && rounds > 4) bound = fmaxf(bound, kth_bound(cls, k, warps, sh));
  }
  const int te = sp.head + 8 * sp.octs + t;
  const float ends[2] = {sl.first && t < sp.head ? to_f(z[t]) : -INFINITY,
                         sl.last && t < sp.tail ? to_f(z[te]) : -INFINITY};
  if (sl.first && t < sp.head) add_one(r, ends[0], c);
  if (sl.last && t < sp.tail) add_one(r, ends[1], c);
  put_warp(r, c, sh.red);
  r = join_warps<kTopWarps>(c, sh.red);
  if (t == 0) sh.part = r;
  if (rounds > 1) bound = fmaxf(bound, kth_bound(cls, k, warps, sh));
  const int noted = sh.n_noted;
  if (noted <= kNoted) {
    for (int i = t; i < noted; i += kTopThreads) {
      Oct<T> w;
      const int at = sh.noted[i];
      w.load(body + 8 * (int64_t)at);
      float f[8];
      w.get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (f[e] >= bound) {
          const int p = atomicAdd(&sh.n_chosen, 1);
          if (p < kChosen) sh.chosen[p] = entry_of(f[e], sp.head + 8 * at + e);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (ends[e] >= bound) {
        const int p = atomicAdd(&sh.n_chosen, 1);
        if (p < kChosen) sh.chosen[p] = entry_of(ends[e], e ? te : t);
      }
  }
  __syncthreads();
  int chosen = sh.n_chosen;
  if (noted > kNoted || chosen > kChosen || r.s != r.s) {
    __syncthreads();
    chosen = exact_top(z, sl.first ? 0 : sp.head + 8 * sl.o0, sl.last ? V : sp.head + 8 * sl.o1, k, sh);
    __syncthreads();
  }
  for (int i = t; i < chosen; i += kTopThreads) {
    const unsigned long long me = sh.chosen[i];
    int at = 0;
    for (int j = 0; j < chosen; ++j) at += sh.chosen[j] > me;
    if (at < k) sh.list[at] = me;
  }
  if (t == 0) sh.n_list = min(chosen, k);
  if (n > 1)
    cluster_meet();
  else
    __syncthreads();
  if (n > 1) {
    const int lane = t & 31;
    r = warp_merge(lane < n ? MaxSum{ld_cluster(&sh.part.m, lane), ld_cluster(&sh.part.s, lane)}
                            : MaxSum{-FLT_MAX, 0.f}, c);
  }
  const float log_s = logf(r.s);
  const bool none = r.s == 0.f;  // nothing but -inf
  int total = sh.n_list;
  int len = 0;  // of the list of CTA `lane`
  if (n > 1) {
    len = (t & 31) < n ? ld_cluster(&sh.n_list, t & 31) : 0;
    total = __reduce_add_sync(0xffffffffu, len);
    for (int i0 = 0; i0 < n * k; i0 += kTopThreads) {  // all lists at once: a remote load takes some 500 cycles
      const int q = min((i0 + t) / k, n - 1), i = i0 + t - q * k;
      const int have = __shfl_sync(0xffffffffu, len, q);
      if (i < have) sh.others[q * kTopMax + i] = ld_cluster(&sh.list[i], q);
    }
    __syncthreads();
  }
  for (int i0 = 0; i0 < sh.n_list; i0 += kTopThreads) {
    const int i = i0 + t;
    const unsigned long long me = i < sh.n_list ? sh.list[i] : 0ull;
    int place = i < sh.n_list ? i : k;
    for (int q = 0; q < n && n > 1; ++q) {
      int lo = 0, hi = __shfl_sync(0xffffffffu, len, q);
      if (q == rank) continue;
      while (lo < hi) {  // entries before lo are larger, those from hi on are not
        const int mid = (lo + hi) >> 1;
        if (sh.others[q * kTopMax + mid] > me)
          lo = mid + 1;
        else
          hi = mid;
      }
      place += lo;
    }
    if (place < k) {
      out_ids[(int64_t)row * k + place] = (int64_t)(uint32_t)~(uint32_t)me;
      out_lp[(int64_t)row * k + place] = (key_value((uint32_t)(me >> 32)) - r.m) / tm - log_s;
    }
  }
  if (rank == 0 && t == 0) out_lse[row] = none ? -INFINITY : r.m / tm + log_s;
  if (rank == 0 && total < k) {  // the remaining places go to the first -inf of the row
    for (int j0 = 0; j0 < V && total < k; j0 += kTopThreads) {
      const int j = j0 + t;
      const bool hit = j < V && to_f(z[j]) == -INFINITY;
      const unsigned ballot = __ballot_sync(0xffffffffu, hit);
      if ((t & 31) == 0) sh.wsum[t >> 5] = __popc(ballot);
      __syncthreads();
      int before = 0, sum = 0;
      for (int w = 0; w < kTopWarps; ++w) {
        if (w < (t >> 5)) before += sh.wsum[w];
        sum += sh.wsum[w];
      }
      const int at = total + before + __popc(ballot & ((1u << (t & 31)) - 1u));
      if (hit && at < k) {
        out_ids[(int64_t)row * k + at] = j;
        out_lp[(int64_t)row * k + at] = r.s != r.s ? r.s : -INFINITY;
      }
      total += sum;
      __syncthreads();
    }
  }
  if (n > 1) cluster_meet();  // a CTA's list outlives its readers
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
  // CTAs a row: enough for three on every SM, at most 8, none for fewer than 4096 tokens
  int n = 1;
  while (n < 8 && N * n < 3 * 148 && V / (2 * n) >= 4096) n *= 2;
  auto go = [&](auto kern, auto* p) {
    launch_rows(kern, (int64_t)N * n, kTopThreads, sizeof(TopShared), n, false, st, p, logits.stride(0), V, log2_of(n),
                (int)k, tp, (float)temperature, ids.data_ptr<int64_t>(), lp.data_ptr<float>(),
                lse.data_ptr<float>());
  };
  if (logits.scalar_type() == at::kFloat)
    go(top_kernel<float>, (const float*)logits.data_ptr());
  else
    go(top_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits.data_ptr());
  return {ids, lp, lse};
}

}  // namespace vocab
}  // namespace libra
