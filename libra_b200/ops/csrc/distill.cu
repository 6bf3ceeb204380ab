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

constexpr int kDistThreads = 256;
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
  MaxSum part;  // this CTA's unlisted (m, s)
  int twice;    // one of this CTA's tokens is listed twice
  int ids[kDistMax];
  double e[kDistMax], p[kDistMax], h[kDistMax];
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// Reads the row's slots and sets, in the bitmap of this CTA's slice, the bits of its tokens: bit of token j is
// j - head - 8 o0 + 8.  A slot counts if its token is inside the vocabulary and its logprob above -inf; second
// occurrences of a token are only noticed here (`twice`), since they are rare.
__device__ __forceinline__ void row_slots(const DistArgs& a, int row, int V, const RowSpan& sp, const Slice& sl,
                                          uint32_t* bits, DistShared& sh) {
  const int words = (sl.o1 - sl.o0 + 2 + 3) >> 2;
  for (int i = threadIdx.x; i < words; i += kDistThreads) bits[i] = 0u;
  if (threadIdx.x == 0) sh.twice = 0;
  const int k = threadIdx.x;
  int id = -1;
  if (k < a.K) {
    const int64_t t = a.ids[(int64_t)row * a.K + k];
    if (t >= 0 && t < V && a.lps[(int64_t)row * a.K + k] > -INFINITY) id = (int)t;
    sh.ids[k] = id;
  }
  __syncthreads();
  if (id >= 0) {
    const int rel = id - sp.head, o = rel >> 3;
    if ((rel < 0 && sl.first) || (rel >= 0 && o >= sl.o0 && (o < sl.o1 || sl.last))) {
      const int bit = rel - 8 * sl.o0 + 8;
      if ((atomicOr(&bits[bit >> 5], 1u << (bit & 31)) >> (bit & 31)) & 1u) sh.twice = 1;
    }
  }
  __syncthreads();
}

// One octet into a running (m, s), without the tokens whose bits are set.
__device__ __forceinline__ void add_octet(MaxSum& a, float (&v)[8], uint32_t listed, float c) {
  if (listed) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((listed >> e) & 1u) v[e] = -INFINITY;
  }
  const float lm = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
  if (lm > a.m) {
    a.s *= ex2((a.m - lm) * c);
    a.m = lm;
  }
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = ex2((v[e] - a.m) * c);
  a.s += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
}

// Head and tail of the row, one element a thread.
template <typename T>
__device__ __forceinline__ void add_ends(MaxSum& a, const T* z, const RowSpan& sp, const Slice& sl,
                                         const uint32_t* bits, float c) {
  const int t = threadIdx.x;
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bits);
  if (sl.first && t < sp.head && !((bytes[0] >> (8 - sp.head + t)) & 1)) add_one(a, to_f(z[t]), c);
  if (sl.last && t < sp.tail && !((bytes[sl.o1 - sl.o0 + 1] >> t) & 1))
    add_one(a, to_f(z[sp.head + 8 * (int64_t)sp.octs + t]), c);
}

// Everything of a row that follows from the unlisted tokens' (m, s): loss, logprob, stats and the slots' gradients.
// Run by one warp, a lane for every 32nd slot.
template <typename T>
__device__ void row_loss(const DistArgs& a, int row, int V, const T* z, MaxSum rest, bool twice, DistShared& sh) {
  const int lane = threadIdx.x & 31, K = a.K;
  const double rT = 1.0 / a.T;
  const float* lps = a.lps + (int64_t)row * K;
  if (twice) {  // the first slot of a token counts
    for (int k = lane; k < K; k += 32) {
      int id = sh.ids[k];
      for (int j = 0; j < k && id >= 0; ++j)
        if (a.ids[(int64_t)row * K + j] == id && lps[j] > -INFINITY) id = -1;
      sh.h[k] = (double)id;
    }
    __syncwarp();
    for (int k = lane; k < K; k += 32) sh.ids[k] = (int)sh.h[k];
    __syncwarp();
  }
  // common maximum of the listed and unlisted logits
  float mf = rest.m;
  bool any = false;
  for (int k = lane; k < K; k += 32) {
    const int id = sh.ids[k];
    const float v = id >= 0 ? to_f(z[id]) : -INFINITY;
    any |= id >= 0;
    sh.e[k] = (double)v;
    mf = fmaxf(mf, v);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) mf = fmaxf(mf, __shfl_xor_sync(0xffffffffu, mf, off));
  any = __any_sync(0xffffffffu, any);
  const double m = (double)mf;
  double s = 0.0, mass = 0.0;
  for (int k = lane; k < K; k += 32) {
    const bool on = sh.ids[k] >= 0;
    const double x = on ? (sh.e[k] - m) * rT : 0.0;  // log q + log s
    sh.h[k] = x;
    sh.e[k] = on ? exp(x) : 0.0;
    sh.p[k] = on ? exp((double)lps[k]) : 0.0;
    s += sh.e[k];
    mass += sh.p[k];
  }
  const double s_rest = (double)rest.s;
  const double shift = ((double)rest.m - m) * rT;  // of the unlisted sum to the common maximum
  const double e_rest = s_rest == 0.0 ? 0.0 : s_rest * exp(shift);
  s = warp_sum(s) + e_rest;
  mass = warp_sum(mass);
  const double log_s = log(s);
  const bool has_rest = !(s_rest == 0.0);
  const bool valid = any && !(s == 0.0) && !(a.drop && mass == 0.0);
  const double q_rest = e_rest / s;
  const double lq_rest = has_rest ? shift + log(s_rest) - log_s : 0.0;
  double p_rest = 0.0, by = 1.0, log_by = 0.0;
  if (a.drop) {
    if (mass > 0.0) {
      by = 1.0 / mass;
      log_by = log(mass);
    }
  } else if (has_rest) {
    p_rest = fmax(1.0 - mass, kRestFloor);
  }
  const double total = a.drop ? 1.0 : mass + p_rest;
  const double lp_rest = p_rest > 0.0 ? log(p_rest) : 0.0;
  const double rs = 1.0 / s, b = a.beta;
  double loss = 0.0, mean = 0.0, d_rest, h_rest = 0.0;  // d_rest: q_r times the unlisted tokens' coefficient
  const int64_t base = (int64_t)row * K;
  for (int k = lane; k < K; k += 32) {
    const bool on = sh.ids[k] >= 0;
    const double p = sh.p[k] * by, q = sh.e[k] * rs;
    const double lp = (double)lps[k] - log_by, lq = sh.h[k] - log_s;
    double h = 0.0;
    if (on) {
      if (a.div == kForward) {
        if (p > 0.0) loss += p * (lp - lq);
        h = q * total - p;  // here already the gradient
      } else if (a.div == kReverse) {
        if (!(q == 0.0)) h = lq - lp;
        mean += q * h;
      } else {
        const double lm = log(b * p + (1.0 - b) * q);
        if (!(q == 0.0)) h = (1.0 - b) * (lq - lm);
        if (p > 0.0) loss += b * p * (lp - lm);
        mean += q * h;
      }
    }
    sh.h[k] = h;
    sh.e[k] = q;
  }
  loss = warp_sum(loss);
  if (a.div == kForward) {
    if (p_rest > 0.0) loss += p_rest * (lp_rest - lq_rest);
    d_rest = q_rest * total - p_rest;
  } else {
    if (has_rest) {
      if (a.div == kReverse) {
        h_rest = lq_rest - lp_rest;
      } else {
        const double lm = log(b * p_rest + (1.0 - b) * q_rest);
        h_rest = (1.0 - b) * (lq_rest - lm);
        if (p_rest > 0.0) loss += b * p_rest * (lp_rest - lm);
      }
    }
    mean = warp_sum(mean) + q_rest * h_rest;
    loss += mean;
    d_rest = q_rest * (h_rest - mean);
  }
  for (int k = lane; k < K; k += 32) {
    const bool on = sh.ids[k] >= 0 && valid;
    const double d = a.div == kForward ? sh.h[k] : sh.e[k] * (sh.h[k] - mean);
    a.clean[base + k] = sh.ids[k];
    a.dk[base + k] = on ? (float)d : 0.f;
    a.qk[base + k] = s == 0.0 ? 0.f : (float)sh.e[k];
  }
  if (lane == 0) {
    a.loss[row] = valid ? (float)loss : 0.f;
    int flags = valid ? kLossRow : 0;
    if (a.targets) {
      const int64_t t = a.targets[row];
      const bool in = t >= 0 && t < V;
      if (!in) atomicCAS(a.err, 0, kBadArgument);
      const float lt = in && !(s == 0.0) ? (float)(((double)to_f(z[t]) - m) * rT - log_s) : -INFINITY;
      a.logp[row] = lt;
      if (lt != -INFINITY) flags |= kProbRow;
    }
    *reinterpret_cast<float4*>(a.stats + 4 * (int64_t)row) =
        make_float4(rest.m, valid && has_rest ? (float)(d_rest / s_rest) : 0.f,
                    has_rest ? (float)(q_rest / s_rest) : 0.f, (float)flags);
  }
}

// One cluster of `n` CTAs a row: each CTA sums its slice, rank 0 joins the parts and finishes the row.
template <typename T>
__global__ void __launch_bounds__(kDistThreads, 4) distill_fwd_kernel(const T* logits, int64_t ld, int V, int n,
                                                                      DistArgs a) {
  extern __shared__ uint32_t dist_bits[];
  __shared__ DistShared sh;
  const int row = blockIdx.x / n, rank = blockIdx.x % n;
  const T* z = logits + (int64_t)row * ld;
  const RowSpan sp = row_span(z, V);
  const Slice sl = row_slice(sp, rank, n);
  row_slots(a, row, V, sp, sl, dist_bits, sh);
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(dist_bits) + 1 - sl.o0;
  const float c = (float)(1.4426950408889634 / a.T);
  MaxSum r = {-FLT_MAX, 0.f};
  add_ends(r, z, sp, sl, dist_bits, c);
  constexpr int kU = sizeof(T) == 2 ? 4 : 2;  // 64 bytes in flight a thread
  const T* body = z + sp.head;
  int o = sl.o0 + threadIdx.x;
  for (; o + (kU - 1) * kDistThreads < sl.o1; o += kU * kDistThreads) {
    Oct<T> v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) v[u].load_once(body + 8 * (int64_t)(o + u * kDistThreads));
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float f[8];
      v[u].get(f);
      add_octet(r, f, bytes[o + u * kDistThreads], c);
    }
  }
  for (; o < sl.o1; o += kDistThreads) {
    Oct<T> v;
    v.load_once(body + 8 * (int64_t)o);
    float f[8];
    v.get(f);
    add_octet(r, f, bytes[o], c);
  }
  r = block_merge<kDistThreads>(r, c, sh.red);
  if (threadIdx.x == 0) sh.part = r;
  if (n > 1) cluster_sync_all();
  if (rank == 0 && threadIdx.x < 32) {
    int twice = sh.twice;
    for (int i = 1; i < n; ++i) {
      r = merge(r, MaxSum{ld_cluster(&sh.part.m, i), ld_cluster(&sh.part.s, i)}, c);
      twice |= ld_cluster(&sh.twice, i);
    }
    row_loss(a, row, V, z, r, twice != 0, sh);
  }
  if (n > 1) cluster_sync_all();  // a CTA's shared memory outlives its readers
}

// dz = (g dL/dx + g_lp dlogp/dx) / T over one of gridDim.y slices of a row.  out may be the logits.  A row without
// gradient is written as zeros.
template <typename T>
__global__ void __launch_bounds__(kDistThreads) distill_bwd_kernel(const T* logits, int64_t ld, T* out, int64_t out_ld,
                                                                   int V, int K, const int64_t* targets, double Td,
                                                                   const float* stats, const int* clean,
                                                                   const float* dk, const float* qk, const float* g,
                                                                   const float* g_lp) {
  const int row = blockIdx.x;
  const T* z = logits + (int64_t)row * ld;
  T* out_row = out + (int64_t)row * out_ld;
  const float4 st = *reinterpret_cast<const float4*>(stats + 4 * (int64_t)row);
  const float rT = (float)(1.0 / Td), c = (float)(1.4426950408889634 / Td);
  const int flags = (int)st.w;
  const bool lp = g_lp && (flags & kProbRow);
  const float gk = flags & kLossRow ? (g ? g[row] : 1.f) : 0.f, gl = lp ? g_lp[row] : 0.f;
  const int64_t target = lp ? targets[row] : -1;
  const bool zero = !(flags & kLossRow) && !lp;
  const float coef = (gk * st.y - gl * st.z) * rT, m = st.x;
  const RowSpan sp = row_span(z, V);
  const Slice sl = row_slice(sp, blockIdx.y, gridDim.y);
  const int lo = sl.first ? 0 : sp.head + 8 * sl.o0, hi = sl.last ? V : sp.head + 8 * sl.o1;
  // the listed tokens and the target, whose values replace the common form
  const int k = threadIdx.x;
  int id = -1;
  float val = 0.f, t_val = 0.f;
  if (k < K) {
    const int64_t at = (int64_t)row * K + k;
    id = clean[at];
    val = (gk * dk[at] - gl * qk[at] + (id == target ? gl : 0.f)) * rT;
  }
  const bool in_slice = target >= lo && target < hi;
  if (k == 0 && in_slice) t_val = coef * ex2((to_f(z[target]) - m) * c) + gl * rT;
  const bool listed = __syncthreads_or(id >= 0 && id == target);  // (and every read of a special precedes the writes)
  const bool vec = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(out_row)) & 15u) == 0;
  if (zero) {
    for (int j = lo + k; j < hi; j += kDistThreads) from_f(out_row + j, 0.f);
    return;
  }
  if (vec) {
    if (sl.first && k < sp.head) from_f(out_row + k, coef * ex2((to_f(z[k]) - m) * c));
    const int te = sp.head + 8 * sp.octs + k;
    if (sl.last && k < sp.tail) from_f(out_row + te, coef * ex2((to_f(z[te]) - m) * c));
    constexpr int kU = sizeof(T) == 2 ? 4 : 2;
    const T* body = z + sp.head;
    T* dst = out_row + sp.head;
    int o = sl.o0 + k;
    for (; o < sl.o1; o += kU * kDistThreads) {
      Oct<T> v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (o + u * kDistThreads < sl.o1) v[u].load_once(body + 8 * (int64_t)(o + u * kDistThreads));
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (o + u * kDistThreads < sl.o1) {
          float f[8];
          v[u].get(f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = coef * ex2((f[e] - m) * c);
          store_oct(dst + 8 * (int64_t)(o + u * kDistThreads), f);
        }
      }
    }
  } else {  // the two rows are not aligned alike
    for (int j = lo + k; j < hi; j += kDistThreads) from_f(out_row + j, coef * ex2((to_f(z[j]) - m) * c));
  }
  __syncthreads();
  if (id >= lo && id < hi) from_f(out_row + id, val);
  if (k == 0 && in_slice && !listed) from_f(out_row + target, t_val);
}

// CTAs a row: enough for three on every SM, at most 8 (a portable cluster), none below 2048 octets' worth of row.
static int row_split(int N, int V) {
  static const int want = 3 * 148;
  int n = 1;
  while (n < 8 && N * n < want && V / (2 * n) >= 4096) n *= 2;
  return n;
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
  const int n = row_split(N, V);
  const size_t smem = (size_t)((V / 8 / n + 1 + 2 + 3) / 4) * 4;
  auto go = [&](auto kern, auto* p) {
    launch_cluster(kern, dim3((unsigned)(N * (int64_t)n)), kDistThreads, smem, n, st, p, logits.stride(0), V, n, a);
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
    kern<<<dim3(N, row_split(N, V)), kDistThreads, 0, st>>>(
        p, logits.stride(0), o, out.stride(0), V, K, targets.has_value() ? targets->data_ptr<int64_t>() : nullptr, T,
        stats.data_ptr<float>(), clean.data_ptr<int>(), dk.data_ptr<float>(), qk.data_ptr<float>(),
        g.has_value() ? g->data_ptr<float>() : nullptr, g_lp.has_value() ? g_lp->data_ptr<float>() : nullptr);
    LIBRA_LAUNCH_CHECK();
  };
  if (logits.scalar_type() == at::kFloat)
    go(distill_bwd_kernel<float>, (const float*)logits.data_ptr(), (float*)out.data_ptr());
  else
    go(distill_bwd_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits.data_ptr(), (__nv_bfloat16*)out.data_ptr());
}

}  // namespace vocab
}  // namespace libra
