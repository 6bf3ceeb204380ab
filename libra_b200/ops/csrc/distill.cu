// Distillation from a teacher's top logprobs, forward and backward.
//
// A row has student logits z (q = softmax(z / T)) and a teacher's table of K
// tokens with logprobs.  Both distributions are taken over buckets: every
// listed token, and one bucket for all others, with q_r = sum of q over them
// and p_r = max(1 - sum p, 2^-24).  (tail = drop: the listed p are divided by
// their sum and p_r = 0.)  A bucket of others that the student gives no mass
// is left out.  With h_b = dL/dq_b the gradient of every divergence is
//
//   dL/dz_j = q_j (h_b(j) - sum_b q_b h_b) / T
//
//   forward  L = sum p (log p - log q)                     h = -p / q
//   reverse  L = sum q (log q - log p)                     h = log q - log p
//   js       L = b KL(p|m) + (1-b) KL(q|m), m = bp+(1-b)q   h = (1-b) log(q / m)
//
// so all tokens outside the table share one coefficient.  q_r is summed over
// the unlisted tokens themselves, not taken as 1 - sum q, which would cancel
// for a confident student; a bitmap of the listed tokens tells them apart.
// The sums of the K buckets are in fp64 (they subtract nearly equal numbers
// where the student is close to the teacher); the long sum over the
// vocabulary is in fp32 relative to its own maximum.
#include "vocab_rows.cuh"

namespace libra {
namespace vocab {

constexpr int kDistThreads = 512;
constexpr int kDistMax = 256;  // slots of a teacher's table
constexpr double kRestFloor = 5.9604644775390625e-08;  // 2^-24, what fp32 logprobs leave open near a sum of one

constexpr int kLossRow = 1, kProbRow = 2;

enum Divergence : int { kForward = 0, kReverse = 1, kJs = 2 };

// What the backward needs of a row: stats [N, 4] fp32.
//   [0] max m of the unlisted logits
//   [1] A: unlisted dL/dx_j = A exp((z_j - m) / T)
//   [2] B: softmax of an unlisted token = B exp((z_j - m) / T)
//   [3] kLossRow if the loss is not identically 0, plus kProbRow if the target's logprob is finite
struct DistArgs {
  const int64_t* ids;  // [N, K]
  const float* lps;    // [N, K]
  int K;
  const int64_t* targets;  // [N] or null
  int div;
  double beta, T;
  bool drop;
  float* loss;   // [N]
  float* logp;   // [N] or null
  float* stats;  // [N, 4]
  int* clean;    // [N, K] token of each slot that counts, else -1
  float* dk;     // [N, K] dL/dx of the slot's token
  float* qk;     // [N, K] its softmax
  int* err;
};

struct DistShared {
  MaxSum red[kDistThreads / 32];
  double sum[kDistThreads / 32];
  int ids[kDistMax];
};

// Sum over the block in a fixed order; every thread gets it.
__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += sh[w];
  __syncthreads();
  return s;
}

// The slots of a row that count: a token inside the vocabulary, a logprob above -inf, the first occurrence of its
// token.  Sets their bits (bit of token j: j - head + 8) and returns this thread's token or -1.
__device__ __forceinline__ int row_slots(const DistArgs& a, int row, int V, int head, uint32_t* bits, DistShared& sh,
                                         float& lp) {
  const int k = threadIdx.x;
  int id = -1;
  lp = 0.f;
  if (k < a.K) {
    const int64_t t = a.ids[(int64_t)row * a.K + k];
    lp = a.lps[(int64_t)row * a.K + k];
    if (t >= 0 && t < V && lp > -INFINITY) id = (int)t;
    sh.ids[k] = id;
  }
  bool twice = false;
  if (id >= 0) {
    const int bit = id - head + 8;
    twice = (atomicOr(&bits[bit >> 5], 1u << (bit & 31)) >> (bit & 31)) & 1u;
  }
  if (__syncthreads_or(twice)) {
    for (int j = 0; j < k && id >= 0; ++j)
      if (j < a.K && sh.ids[j] == id) id = -1;
  }
  return id;
}

// Everything of a row that follows from the unlisted tokens' (m, s): loss, logprob, stats and the slots' gradients.
template <typename T>
__device__ void row_loss(const DistArgs& a, int row, int V, const T* z, int id, float lpf, MaxSum rest,
                         DistShared& sh) {
  const int k = threadIdx.x;
  const double rT = 1.0 / a.T;
  const double zk = id >= 0 ? (double)to_f(z[id]) : 0.0;
  // common maximum of the listed and unlisted logits
  float mk = id >= 0 ? to_f(z[id]) : -FLT_MAX;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mk = fmaxf(mk, __shfl_xor_sync(0xffffffffu, mk, off));
  if ((k & 31) == 0) sh.red[k >> 5].m = mk;
  __syncthreads();
  float mf = rest.m;
  for (int w = 0; w < kDistThreads / 32; ++w) mf = fmaxf(mf, sh.red[w].m);
  const double m = (double)mf;
  const bool any = __syncthreads_or(id >= 0);
  const double s_rest = (double)rest.s;
  const double shift = ((double)rest.m - m) * rT;  // of the unlisted sum to the common maximum
  const double e_rest = s_rest == 0.0 ? 0.0 : s_rest * exp(shift);
  const double ek = id >= 0 ? exp((zk - m) * rT) : 0.0;
  const double s = block_sum(ek, sh.sum) + e_rest;
  const double log_s = log(s);
  const bool has_rest = !(s_rest == 0.0);
  const double q_rest = e_rest / s;
  const double lq_rest = has_rest ? shift + log(s_rest) - log_s : 0.0;
  double lp = (double)lpf;
  double p = id >= 0 ? exp(lp) : 0.0;
  const double mass = block_sum(p, sh.sum);
  const bool valid = any && !(s == 0.0) && !(a.drop && mass == 0.0);
  double p_rest = 0.0;
  if (a.drop) {
    const double by = mass > 0.0 ? mass : 1.0;
    lp -= log(by);
    p /= by;
  } else if (has_rest) {
    p_rest = fmax(1.0 - mass, kRestFloor);
  }
  const double total = a.drop ? 1.0 : mass + p_rest;
  const double lp_rest = p_rest > 0.0 ? log(p_rest) : 0.0;
  const double lq = id >= 0 ? (zk - m) * rT - log_s : 0.0;
  const double q = ek / s;
  double loss = 0.0, dk = 0.0, d_rest = 0.0;  // d_rest: q_r times the unlisted tokens' coefficient
  if (a.div == kForward) {
    const double t = id >= 0 && p > 0.0 ? p * (lp - lq) : 0.0;
    loss = block_sum(t, sh.sum) + (p_rest > 0.0 ? p_rest * (lp_rest - lq_rest) : 0.0);
    dk = q * total - p;
    d_rest = q_rest * total - p_rest;
  } else {
    double h = 0.0, h_rest = 0.0, kp = 0.0, kp_rest = 0.0;
    if (a.div == kReverse) {
      if (id >= 0 && !(q == 0.0)) h = lq - lp;
      if (has_rest) h_rest = lq_rest - lp_rest;
    } else {
      const double b = a.beta;
      if (id >= 0) {
        const double lm = log(b * p + (1.0 - b) * q);
        if (!(q == 0.0)) h = (1.0 - b) * (lq - lm);
        if (p > 0.0) kp = b * p * (lp - lm);
      }
      if (has_rest) {
        const double lm = log(b * p_rest + (1.0 - b) * q_rest);
        h_rest = (1.0 - b) * (lq_rest - lm);
        if (p_rest > 0.0) kp_rest = b * p_rest * (lp_rest - lm);
      }
    }
    const double mean = block_sum(q * h, sh.sum) + q_rest * h_rest;
    loss = mean + block_sum(kp, sh.sum) + kp_rest;
    dk = q * (h - mean);
    d_rest = q_rest * (h_rest - mean);
  }
  if (k < a.K) {
    const int64_t at = (int64_t)row * a.K + k;
    a.clean[at] = id;
    a.dk[at] = id >= 0 && valid ? (float)dk : 0.f;
    a.qk[at] = s == 0.0 ? 0.f : (float)q;
  }
  if (k == 0) {
    a.loss[row] = valid ? (float)loss : 0.f;
    float* st = a.stats + 4 * (int64_t)row;
    st[0] = rest.m;
    st[1] = valid && has_rest ? (float)(d_rest / s_rest) : 0.f;
    st[2] = has_rest ? (float)(q_rest / s_rest) : 0.f;
    int flags = valid ? kLossRow : 0;
    if (a.targets) {
      const int64_t t = a.targets[row];
      const bool in = t >= 0 && t < V;
      if (!in) atomicCAS(a.err, 0, kBadArgument);
      const float lt = in && !(s == 0.0) ? (float)(((double)to_f(z[t]) - m) * rT - log_s) : -INFINITY;
      a.logp[row] = lt;
      if (lt != -INFINITY) flags |= kProbRow;
    }
    st[3] = (float)flags;
  }
}

template <typename T>
__global__ void __launch_bounds__(kDistThreads) distill_fwd_kernel(const T* logits, int64_t ld, int V, DistArgs a) {
  extern __shared__ uint32_t dist_bits[];
  __shared__ DistShared sh;
  const int row = blockIdx.x;
  const T* z = logits + (int64_t)row * ld;
  const RowSpan sp = row_span(z, V);
  const int words = (V + 15 + 31) >> 5;
  for (int i = threadIdx.x; i < words; i += kDistThreads) dist_bits[i] = 0u;
  __syncthreads();
  float lp;
  const int id = row_slots(a, row, V, sp.head, dist_bits, sh, lp);
  const float c = (float)(1.4426950408889634 / a.T);
  MaxSum r = {-FLT_MAX, 0.f};
  for (int j = threadIdx.x; j < V; j += kDistThreads) {
    const int bit = j - sp.head + 8;
    if (!((dist_bits[bit >> 5] >> (bit & 31)) & 1u)) add_one(r, to_f(z[j]), c);
  }
  r = block_merge<kDistThreads>(r, c, sh.red);
  row_loss(a, row, V, z, id, lp, r, sh);
}

// dz = (g dL/dx + g_lp dlogp/dx) / T.  out may be the logits.  A row without gradient is written as zeros.
template <typename T>
__global__ void __launch_bounds__(kDistThreads) distill_bwd_kernel(const T* logits, int64_t ld, T* out, int64_t out_ld,
                                                                   int V, int K, const int64_t* targets, float T_,
                                                                   const float* stats, const int* clean,
                                                                   const float* dk, const float* qk, const float* g,
                                                                   const float* g_lp) {
  const int row = blockIdx.x;
  const T* z = logits + (int64_t)row * ld;
  T* o = out + (int64_t)row * out_ld;
  const float* st = stats + 4 * (int64_t)row;
  const float rT = 1.f / T_, c = kLog2e / T_;
  const int flags = (int)st[3];
  const float gk = flags & kLossRow ? (g ? g[row] : 1.f) : 0.f;
  const float gl = g_lp && (flags & kProbRow) ? g_lp[row] : 0.f;
  const int64_t target = g_lp && (flags & kProbRow) ? targets[row] : -1;
  if (!(flags & kLossRow) && target < 0) {
    for (int j = threadIdx.x; j < V; j += kDistThreads) from_f(o + j, 0.f);
    return;
  }
  const float coef = (gk * st[1] - gl * st[2]) * rT, m = st[0];
  // the table's tokens and the target, whose values replace the common form
  const int k = threadIdx.x;
  int id = -1;
  float val = 0.f;
  if (k < K) {
    const int64_t at = (int64_t)row * K + k;
    id = clean[at];
    val = (gk * dk[at] - gl * qk[at] + (id == target ? gl : 0.f)) * rT;
  }
  const bool listed = __syncthreads_or(id >= 0 && id == target);
  if (k == K && !listed && target >= 0 && target < V) {
    id = (int)target;
    val = coef * ex2((to_f(z[id]) - m) * c) + gl * rT;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < V; j += kDistThreads) from_f(o + j, coef * ex2((to_f(z[j]) - m) * c));
  __syncthreads();
  if (id >= 0) from_f(o + id, val);
}

static void check_distill(const torch::Tensor& logits, const torch::Tensor& ids, const torch::Tensor& lps, int64_t div,
                          double beta, double T, const char* op) {
  check_rows(logits, op);
  const int64_t N = logits.size(0), V = logits.size(1);
  LIBRA_CHECK(ids.dim() == 2 && ids.size(0) == N && ids.size(1) >= 1 && ids.size(1) <= kDistMax &&
                  vec_of(ids, logits, at::kLong, ids.numel()),
              "%s: teacher_ids must be contiguous int64 [N, 1..%d] on the logits' device", op, kDistMax);
  LIBRA_CHECK(lps.sizes() == ids.sizes() && vec_of(lps, logits, at::kFloat, ids.numel()),
              "%s: teacher_logprobs must be contiguous fp32 like teacher_ids", op);
  LIBRA_CHECK(V >= 1 && V <= 1600000, "%s: vocabulary of 1 to 1600000 tokens", op);
  LIBRA_CHECK(div >= 0 && div <= 2 && beta > 0.0 && beta < 1.0 && T > 0.0, "%s: divergence, beta or temperature", op);
}

// -> {loss [N], logp [N] or empty, stats [N, 4], clean [N, K], dk [N, K], qk [N, K]}
std::vector<torch::Tensor> distill_fwd(torch::Tensor logits, torch::Tensor ids, torch::Tensor lps, int64_t div,
                                       double beta, bool drop, double T, c10::optional<torch::Tensor> targets,
                                       torch::Tensor err) {
  check_distill(logits, ids, lps, div, beta, T, "distill_loss");
  const int N = (int)logits.size(0), V = (int)logits.size(1), K = (int)ids.size(1);
  if (targets.has_value())
    LIBRA_CHECK(vec_of(*targets, logits, at::kLong, N), "distill_loss: targets must be contiguous int64 [N] on the "
                "logits' device");
  LIBRA_CHECK(err.device() == logits.device() && err.scalar_type() == at::kInt, "distill_loss: error word");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  auto loss = torch::empty({N}, f32), logp = torch::empty({targets.has_value() ? N : 0}, f32);
  auto stats = torch::empty({N, 4}, f32), dk = torch::empty({N, K}, f32), qk = torch::empty({N, K}, f32);
  auto clean = torch::empty({N, K}, logits.options().dtype(at::kInt));
  if (N == 0) return {loss, logp, stats, clean, dk, qk};
  DistArgs a = {};
  a.ids = ids.data_ptr<int64_t>();
  a.lps = lps.data_ptr<float>();
  a.K = K;
  a.targets = targets.has_value() ? targets->data_ptr<int64_t>() : nullptr;
  a.div = (int)div;
  a.beta = beta;
  a.T = T;
  a.drop = drop;
  a.loss = loss.data_ptr<float>();
  a.logp = logp.data_ptr<float>();
  a.stats = stats.data_ptr<float>();
  a.clean = clean.data_ptr<int>();
  a.dk = dk.data_ptr<float>();
  a.qk = qk.data_ptr<float>();
  a.err = err.data_ptr<int>();
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const size_t smem = (size_t)((V + 15 + 31) >> 5) * 4;
  auto go = [&](auto kern, auto* p) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    LIBRA_CHECK(e == cudaSuccess, "distill_loss: %s", cudaGetErrorString(e));
    kern<<<N, kDistThreads, smem, st>>>(p, logits.stride(0), V, a);
    LIBRA_LAUNCH_CHECK();
  };
  if (logits.scalar_type() == at::kFloat)
    go(distill_fwd_kernel<float>, (const float*)logits.data_ptr());
  else
    go(distill_fwd_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits.data_ptr());
  return {loss, logp, stats, clean, dk, qk};
}

// Gradient with respect to the logits into out (which may be the logits): g [N] or none for ones, g_lp [N] or none.
void distill_bwd(torch::Tensor logits, torch::Tensor out, double T, c10::optional<torch::Tensor> targets,
                 torch::Tensor stats, torch::Tensor clean, torch::Tensor dk, torch::Tensor qk,
                 c10::optional<torch::Tensor> g, c10::optional<torch::Tensor> g_lp) {
  check_rows(logits, "distill_loss");
  const int N = (int)logits.size(0), V = (int)logits.size(1), K = (int)clean.size(1);
  LIBRA_CHECK(out.device() == logits.device() && out.scalar_type() == logits.scalar_type() &&
                  out.sizes() == logits.sizes() && (V <= 1 || out.stride(1) == 1) && (N <= 1 || out.stride(0) >= V),
              "distill_loss: the gradient has the logits' shape and type, unit inner stride");
  check_apart(logits, out, "distill_loss");
  LIBRA_CHECK(vec_of(stats, logits, at::kFloat, 4 * (int64_t)N) && vec_of(clean, logits, at::kInt, (int64_t)N * K) &&
                  vec_of(dk, logits, at::kFloat, (int64_t)N * K) && vec_of(qk, logits, at::kFloat, (int64_t)N * K) &&
                  K >= 1 && K <= kDistMax,
              "distill_loss: saved tensors do not match the logits");
  if (g.has_value()) LIBRA_CHECK(vec_of(*g, logits, at::kFloat, N), "distill_loss: upstream gradient fp32 [N]");
  if (g_lp.has_value())
    LIBRA_CHECK(vec_of(*g_lp, logits, at::kFloat, N) && targets.has_value() &&
                    vec_of(*targets, logits, at::kLong, N),
                "distill_loss: upstream gradient fp32 [N] of the logprobs, with their targets");
  if (N == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto go = [&](auto kern, auto* p, auto* o) {
    kern<<<N, kDistThreads, 0, st>>>(p, logits.stride(0), o, out.stride(0), V, K,
                                     targets.has_value() ? targets->data_ptr<int64_t>() : nullptr, (float)T,
                                     stats.data_ptr<float>(), clean.data_ptr<int>(), dk.data_ptr<float>(),
                                     qk.data_ptr<float>(), g.has_value() ? g->data_ptr<float>() : nullptr,
                                     g_lp.has_value() ? g_lp->data_ptr<float>() : nullptr);
    LIBRA_LAUNCH_CHECK();
  };
  if (logits.scalar_type() == at::kFloat)
    go(distill_bwd_kernel<float>, (const float*)logits.data_ptr(), (float*)out.data_ptr());
  else
    go(distill_bwd_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits.data_ptr(), (__nv_bfloat16*)out.data_ptr());
}

}  // namespace vocab
}  // namespace libra
