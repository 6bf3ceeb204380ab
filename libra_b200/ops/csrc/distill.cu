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

constexpr int kFwdThreads = 256, kOneThreads = 192, kOneCtas = 5, kTableWarps = 4;
constexpr int kBwdThreads = 256;
constexpr int kDistMax = 256;  // slots of a teacher's table
constexpr int kHash = 512;
constexpr double kRestFloor = 5.9604644775390625e-08;  // 2^-24, what fp32 logprobs leave open near a sum of one

constexpr int kLossRow = 1, kProbRow = 2;

enum Divergence : int { kForward = 0, kReverse = 1, kJs = 2 };

// What the backward needs of a row: stats [N, 4] fp32.
//   [0] reference m of the unlisted logits
//   [1] A: unlisted dL/dx_j = A exp((z_j - m) / T)
//   [2] B: softmax of an unlisted token = B exp((z_j - m) / T)
//   [3] kLossRow if the loss is not identically 0, plus kProbRow if the target's logprob has a gradient

// Sums over a row's table.  With mk the largest listed logit and x_k = (z_k - mk) / T:
struct __align__(16) TableSums {
  double s, mass, dot;  // sum of exp(x), of p, of p (log p - x); tail = drop: of p relative to the row's largest
  double p_rest;        // the teacher's mass outside the table
  float sf, massf, p_restf, lp_rest, by, log_by;  // p is scaled by `by` (tail = drop)
  float mk;
  int any;
};
struct DistArgs {
  const int64_t* ids;  // [N, K]
  const float* lps;    // [N, K]
  int N, K;
  const int64_t* targets;  // [N] or null
  int div;
  double beta, T;
  bool drop;
  float* loss;   // [N]
  float* logp;   // [N] or null
  float* stats;  // [N, 4] or null
  float* dk;     // [N, K] or null: dL/dx of the slot's token
  float* qk;     // [N, K] or null: its softmax
  int* err;
  // the rows' tables, per slot: token (-1: the slot does not count), exp(x_k), p_k and x_k - log p_k (in fp64 until
  // here, since the two nearly cancel)
  int* clean;
  float *ex, *p, *xl;  // [N, K]
  TableSums* sums;     // [N]
  MaxSum* parts;       // [N, splits] of the unlisted tokens
};

// What a row's gradients need: log q - log p = xl + off, q = exp(x) w, p = p_k by.
struct RowFin {
  float off, w, by, total, mean;
  float m, A, B;  // as in stats
  int flags;
};

// A slot counts if its token is inside the vocabulary and its logprob above -inf.
__device__ __forceinline__ int slot_token(const DistArgs& a, int64_t at, int V, float& lp) {
  const int64_t t = a.ids[at];
  lp = a.lps[at];
  return t >= 0 && t < V && lp > -INFINITY ? (int)t : -1;
}

// Sets the bits of the row's tokens in the bitmap of this CTA's slice: bit of token j is j - head - 8 o0 + 8.
template <int kThreads>
__device__ __forceinline__ void row_bits(const DistArgs& a, int row, const RowSpan& sp, const Slice& sl,
                                         uint32_t* bits) {
  const int words = (sl.o1 - sl.o0 + 2 + 3) >> 2;
  constexpr int kMine = (kDistMax + kThreads - 1) / kThreads;
  int id[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int k = threadIdx.x + i * kThreads;
    id[i] = k < a.K ? a.clean[(int64_t)row * a.K + k] : -1;
  }
  for (int w = threadIdx.x; w < words; w += kThreads) bits[w] = 0u;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int rel = id[i] - sp.head, o = rel >> 3;
    if (id[i] >= 0 && ((rel < 0 && sl.first) || (rel >= 0 && o >= sl.o0 && (o < sl.o1 || sl.last)))) {
      const int bit = rel - 8 * sl.o0 + 8;
      atomicOr(&bits[bit >> 5], 1u << (bit & 31));
    }
  }
  __syncthreads();
}

// One octet into a thread's running (m, s), without the tokens whose bits are set; `top` is m + kSlack / c.
template <typename T>
__device__ __forceinline__ void add_octet(MaxSum& a, float& top, const Oct<T>& raw, uint32_t listed, float c,
                                          float slack) {
  float v[8];
  raw.get(v);
  float lm = raw.max();
  if (listed) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((listed >> e) & 1u) v[e] = -INFINITY;
    lm = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
  }
  add_values(a, top, v, lm, c, slack);
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

// One warp a row fills its table and sums.  A kernel of its own, since one row's chain of gathers and fp64 functions
// takes about 5 us: inside the streaming kernels it set the pace (4096 x 151936 bf16 in one pass: 0.70 ms).
template <typename T>
__global__ void __launch_bounds__(kTableWarps * 32) distill_table_kernel(const T* logits, int64_t ld, int V,
                                                                         DistArgs a) {
  __shared__ int hashes[kTableWarps][kHash];
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, row = blockIdx.x * kTableWarps + (threadIdx.x >> 5), K = a.K;
  if (row >= a.N) return;
  const T* z = logits + (int64_t)row * ld;
  int* hash = hashes[threadIdx.x >> 5];
  const int64_t base = (int64_t)row * K;
  int* ids = a.clean + base;
  const double rT = 1.0 / a.T;
  for (int i = lane; i < kHash; i += 32) hash[i] = -1;
  __syncwarp();
  bool twice = false, any = false;
  float mk = -FLT_MAX, most = -INFINITY;  // of the listed logits and of their logprobs
  for (int k = lane; k < K; k += 32) {
    float lp;
    const int id = slot_token(a, base + k, V, lp);
    ids[k] = id;
    const float v = id >= 0 ? to_f(z[id]) : -INFINITY;
    a.ex[base + k] = v;
    if (id < 0) continue;
    any = true;
    mk = fmaxf(mk, v);
    most = fmaxf(most, lp);
    unsigned h = ((unsigned)id * 2654435761u) >> 23;
    while (true) {  // at most 256 of the 512 places are taken
      const int old = atomicCAS(&hash[h], -1, id);
      twice |= old == id;
      if (old == -1 || old == id) break;
      h = (h + 1) & (kHash - 1);
    }
  }
  __syncwarp();
  if (__any_sync(0xffffffffu, twice)) {  // the first slot of a token counts
    for (int k0 = (K - 1) / 32 * 32; k0 >= 0; k0 -= 32) {  // from behind: earlier slots are still as they were
      const int k = k0 + lane;
      int id = k < K ? ids[k] : -1;
      for (int j = 0; j < k && id >= 0; ++j)
        if (ids[j] == id) id = -1;
      __syncwarp();
      if (k < K) ids[k] = id;
      __syncwarp();
    }
    most = -INFINITY;
    for (int k = lane; k < K; k += 32)
      if (ids[k] >= 0) most = fmaxf(most, a.lps[base + k]);
  }
  mk = warp_max(mk);
  any = __any_sync(0xffffffffu, any);
  // tail = drop: relative to the row's largest, since only the ratios of the p count and none of them may underflow
  most = warp_max(most);
  const double lp_max = a.drop && any ? (double)most : 0.0;
  double s = 0.0, mass = 0.0, dot = 0.0;
  for (int k = lane; k < K; k += 32) {
    const bool on = ids[k] >= 0;
    const double lp = on ? (double)a.lps[base + k] - lp_max : 0.0;
    const double x = on ? ((double)a.ex[base + k] - (double)mk) * rT : 0.0;
    const double ex = on ? exp(x) : 0.0, p = on ? exp(lp) : 0.0;
    a.ex[base + k] = (float)ex;
    a.p[base + k] = (float)p;
    a.xl[base + k] = (float)(x - lp);
    s += ex;
    mass += p;
    if (p > 0.0) dot += p * (lp - x);
  }
  s = warp_sum(s);
  mass = warp_sum(mass);
  dot = warp_sum(dot);
  if (lane == 0) {
    const double p_rest = a.drop ? 0.0 : fmax(1.0 - mass, kRestFloor);
    const bool scale = a.drop && any;  // mass lies in [1, K] then
    a.sums[row] = TableSums{s, mass, dot, p_rest, (float)s, (float)mass, (float)p_rest,
                            a.drop ? 0.f : (float)log(p_rest), scale ? (float)(1.0 / mass) : 1.f,
                            scale ? (float)log(mass) : 0.f, mk, any};
  }
}

// h of a bucket from d = log q - log p (see the top of the file), q > 0.
__device__ __forceinline__ float bucket_h(const DistArgs& a, float d) {
  if (a.div == kReverse) return d;
  const float b = (float)a.beta;
  // (1-b) log(q / m), and p / q = exp(-d), which stays finite for a q that fp32 still holds
  return -(1.f - b) * logf(b * ex2(fminf(-d * kLog2e, 126.f)) + (1.f - b));
}
__device__ __forceinline__ float slot_grad(const DistArgs& a, const RowFin& f, float ex, float p, float xl) {
  const float q = ex * f.w;
  if (a.div == kForward) return q * f.total - p * f.by;
  return q == 0.f ? 0.f : q * (bucket_h(a, xl + f.off) - f.mean);
}

// What the gradients of a row need, by one warp in fp32: a listed gradient is a difference of two probabilities, each
// right to a few 2^-24, and the row waits for this chain (in fp64 it takes some 5 us, see distill_table_kernel).
__device__ __forceinline__ RowFin finish_grads(const DistArgs& a, int row, const TableSums& u, MaxSum rest, float c) {
  const float mk = u.mk, s_list = u.sf, mass = u.massf, lp_rest = u.lp_rest, log_by = u.log_by;
  const int64_t base = (int64_t)row * a.K;
  float p_rest = u.p_restf;
  const bool any = u.any != 0;
  const float rT = (float)(1.0 / a.T), m = fmaxf(rest.m, mk);
  const float fl = ex2((mk - m) * c), fr = ex2((rest.m - m) * c);
  const float e_rest = rest.s * fr, s = s_list * fl + e_rest, rs = 1.f / s;
  const bool has_rest = !(rest.s == 0.f);
  if (!has_rest) p_rest = 0.f;
  const float q_rest = e_rest * rs;
  RowFin f;
  f.by = u.by;
  f.w = fl * rs;
  f.total = a.drop ? 1.f : mass + p_rest;
  f.off = 0.f;
  f.mean = 0.f;
  float d_rest;  // q_r times the unlisted tokens' coefficient
  if (a.div == kForward) {
    d_rest = q_rest * f.total - p_rest;
  } else {
    const float log_s = logf(s);
    f.off = (mk - m) * rT - log_s + log_by;
    float mean = 0.f, h_rest = 0.f;
    for (int k = threadIdx.x & 31; k < a.K; k += 32) {
      const float q = a.clean[base + k] < 0 ? 0.f : a.ex[base + k] * f.w;
      if (!(q == 0.f)) mean += q * bucket_h(a, a.xl[base + k] + f.off);
    }
    if (has_rest && q_rest > 0.f)
      h_rest = a.drop ? -(1.f - (float)a.beta) * logf(1.f - (float)a.beta)
                      : bucket_h(a, (rest.m - m) * rT + logf(rest.s) - log_s - lp_rest);
    f.mean = warp_sum(mean) + q_rest * h_rest;
    d_rest = q_rest * (h_rest - f.mean);
  }
  const bool valid = any && !(s == 0.f);
  f.m = rest.m;
  f.A = valid && has_rest ? d_rest / rest.s : 0.f;
  f.B = has_rest ? q_rest / rest.s : 0.f;
  f.flags = valid ? kLossRow : 0;
  return f;
}

// Loss of a row in fp64, by one warp; also log s and the common maximum it refers to.
__device__ __forceinline__ double finish_loss(const DistArgs& a, int row, const TableSums& u, MaxSum rest,
                                              double& log_s, double& m) {
  const int64_t base = (int64_t)row * a.K;
  const double rT = 1.0 / a.T, b = a.beta, s_rest = (double)rest.s;
  m = (double)fmaxf(rest.m, u.mk);
  const double al = ((double)u.mk - m) * rT, ar = ((double)rest.m - m) * rT;
  const bool has_rest = !(s_rest == 0.0);
  const double e_rest = !has_rest ? 0.0 : ar == 0.0 ? s_rest : s_rest * exp(ar);
  const double fl = al == 0.0 ? 1.0 : exp(al), s = u.s * fl + e_rest;
  log_s = log(s);
  const double lq_rest = has_rest ? ar + log(s_rest) - log_s : 0.0;
  const double p_rest = has_rest ? u.p_rest : 0.0, lp_rest = p_rest > 0.0 ? log(p_rest) : 0.0;
  const bool scale = a.drop && u.any;
  const double by = scale ? 1.0 / u.mass : 1.0, log_by = scale ? log(u.mass) : 0.0;
  double loss;
  if (a.div == kForward) {
    loss = by * u.dot + by * u.mass * (log_s - al - log_by);
    if (p_rest > 0.0) loss += p_rest * (lp_rest - lq_rest);
  } else {
    const double off = al - log_s + log_by, w = fl / s, q_rest = e_rest / s;
    double sum = 0.0;
    for (int k = threadIdx.x & 31; k < a.K; k += 32) {
      if (a.clean[base + k] < 0) continue;
      const double q = (double)a.ex[base + k] * w, p = (double)a.p[base + k] * by, d = (double)a.xl[base + k] + off;
      if (a.div == kReverse) {
        if (!(q == 0.0)) sum += q * d;
      } else {
        // log(m / p) = log(b + (1-b) e^d) and log(m / q) = log(b e^-d + (1-b)), with the larger power taken out of both:
        // a q far below p is a subnormal whose e^-d is infinite
        const double e = exp(-fabs(d)), l = log(d > 0.0 ? b * e + (1.0 - b) : b + (1.0 - b) * e);
        if (p > 0.0) sum -= b * p * (l + fmax(d, 0.0));
        if (!(q == 0.0)) sum -= (1.0 - b) * q * (l + fmax(-d, 0.0));
      }
    }
    loss = warp_sum(sum);
    if (has_rest && a.div == kReverse) loss += q_rest * (lq_rest - lp_rest);
    if (has_rest && a.div == kJs) {
      const double mix = b * p_rest + (1.0 - b) * q_rest;
      if (p_rest > 0.0) loss += b * p_rest * (lp_rest - log(mix));
      if (!(q_rest == 0.0)) loss += (1.0 - b) * q_rest * (lq_rest - log(mix));
    }
  }
  return u.any && !(s == 0.0) ? loss : 0.0;
}

// The unlisted tokens' (m, s) of one of 2^lg slices of a row.
template <typename T>
__global__ void __launch_bounds__(kFwdThreads, 4) distill_sum_kernel(const T* logits, int64_t ld, int V, int lg,
                                                                     DistArgs a) {
  extern __shared__ uint32_t dist_bits[];
  __shared__ MaxSum red[kFwdThreads / 32];
  pdl_launch_dependents();
  const int row = blockIdx.x >> lg, rank = blockIdx.x & ((1 << lg) - 1), t = threadIdx.x;
  const T* z = logits + (int64_t)row * ld;
  const RowSpan sp = row_span(z, V);
  const Slice sl = row_slice(sp, rank, lg);
  const float c = (float)(1.4426950408889634 / a.T), slack = kSlack / c;
  constexpr int kU = sizeof(T) == 2 ? 4 : 2;  // 64 bytes in flight a thread
  const T* body = z + sp.head;
  Oct<T> v[kU];
  int o = sl.o0 + t;
  // the first loads are under way before the tables are there
#pragma unroll
  for (int u = 0; u < kU; ++u)
    if (o + u * kFwdThreads < sl.o1) v[u].load_once(body + 8 * (int64_t)(o + u * kFwdThreads));
  pdl_wait();
  row_bits<kFwdThreads>(a, row, sp, sl, dist_bits);
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(dist_bits) + 1 - sl.o0;
  MaxSum r = {-FLT_MAX, 0.f};
  float top = -FLT_MAX;
  const int step = kU * kFwdThreads;
  for (; o + step - kFwdThreads < sl.o1; o += step) {
    Oct<T> w[kU];  // the next round's loads fly while this one is summed
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (o + step + u * kFwdThreads < sl.o1) w[u].load_once(body + 8 * (int64_t)(o + step + u * kFwdThreads));
#pragma unroll
    for (int u = 0; u < kU; ++u) add_octet(r, top, v[u], bytes[o + u * kFwdThreads], c, slack);
#pragma unroll
    for (int u = 0; u < kU; ++u) v[u] = w[u];
  }
#pragma unroll
  for (int u = 0; u < kU; ++u)
    if (o + u * kFwdThreads < sl.o1) add_octet(r, top, v[u], bytes[o + u * kFwdThreads], c, slack);
  add_ends(r, z, sp, sl, dist_bits, c);
  put_warp(r, c, red);
  if (t < 32) {
    r = join_warps<kFwdThreads / 32>(c, red);
    if (t == 0) a.parts[blockIdx.x] = r;
  }
}

// One warp a row: loss, logprob, and what the backward needs, from the table and the slices' sums.
template <typename T>
__global__ void __launch_bounds__(kTableWarps * 32) distill_row_kernel(const T* logits, int64_t ld, int V, int lg,
                                                                       DistArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31, row = blockIdx.x * kTableWarps + (threadIdx.x >> 5);
  if (row >= a.N) return;
  const float c = (float)(1.4426950408889634 / a.T);
  const TableSums u = a.sums[row];
  const MaxSum rest = warp_merge(lane < (1 << lg) ? a.parts[((int64_t)row << lg) + lane] : MaxSum{-FLT_MAX, 0.f}, c);
  double log_s, m;
  const double loss = finish_loss(a, row, u, rest, log_s, m);
  if (lane == 0) a.loss[row] = (float)loss;
  if (!a.stats) return;
  const RowFin f = finish_grads(a, row, u, rest, c);
  const int64_t base = (int64_t)row * a.K;
  for (int k = lane; k < a.K; k += 32) {
    const float ex = a.ex[base + k];
    const bool on = a.clean[base + k] >= 0;
    a.dk[base + k] = on && f.flags ? slot_grad(a, f, ex, a.p[base + k], a.xl[base + k]) : 0.f;
    a.qk[base + k] = on && ex != 0.f ? ex * f.w : 0.f;
  }
  if (lane == 0) {
    int flags = f.flags;
    if (a.targets) {
      const int64_t g = a.targets[row];
      const bool in = g >= 0 && g < V;
      if (!in) atomicCAS(a.err, 0, kBadArgument);
      const bool defined = in && log_s != -INFINITY;  // the row has a distribution
      a.logp[row] = defined ? (float)(((double)to_f(logits[(int64_t)row * ld + g]) - m) / a.T - log_s) : -INFINITY;
      if (defined) flags |= kProbRow;
    }
    *reinterpret_cast<float4*>(a.stats + 4 * (int64_t)row) = make_float4(f.m, f.A, f.B, (float)flags);
  }
}

// coef exp((z - m) / T) of an octet.
template <typename T>
__device__ __forceinline__ void grad_oct(const Oct<T>& raw, float (&f)[8], float m, float c, float coef) {
  raw.get(f);
  exp_oct(f, m, c);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const F2 x = mul2(F2{f[2 * i], f[2 * i + 1]}, F2{coef, coef});
    f[2 * i] = x.x;
    f[2 * i + 1] = x.y;
  }
}

// dz = (g dL/dx + g_lp dlogp/dx) / T over one of 2^lg slices of a row.  out may be the logits.  A row without
// gradient is written as zeros.
template <typename T>
__global__ void __launch_bounds__(kBwdThreads) distill_bwd_kernel(const T* logits, int64_t ld, T* out, int64_t out_ld,
                                                                   int V, int lg, int K, const int64_t* targets, double Td,
                                                                   const float* stats, const int* clean,
                                                                   const float* dk, const float* qk, const float* g,
                                                                   const float* g_lp) {
  const int row = blockIdx.x >> lg, rank = blockIdx.x & ((1 << lg) - 1);
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
  const Slice sl = row_slice(sp, rank, lg);
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
    for (int j = lo + k; j < hi; j += kBwdThreads) from_f(out_row + j, 0.f);
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
    for (; o < sl.o1; o += kU * kBwdThreads) {
      Oct<T> v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (o + u * kBwdThreads < sl.o1) v[u].load_once(body + 8 * (int64_t)(o + u * kBwdThreads));
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (o + u * kBwdThreads < sl.o1) {
          float f[8];
          grad_oct(v[u], f, m, c, coef);
          store_oct(dst + 8 * (int64_t)(o + u * kBwdThreads), f);
        }
      }
    }
  } else {  // the two rows are not aligned alike
    for (int j = lo + k; j < hi; j += kBwdThreads) from_f(out_row + j, coef * ex2((to_f(z[j]) - m) * c));
  }
  __syncthreads();
  if (id >= lo && id < hi) from_f(out_row + id, val);
  if (k == 0 && in_slice && !listed) from_f(out_row + target, t_val);
}

// Unit gradient in one pass: a cluster holds the whole row in shared memory, each CTA its slice, so the logits are read
// once.  A thread copies, sums and rewrites the same octets, which needs no barrier.  Behind the one cluster barrier
// that the slices' sums wait for, every CTA finishes the row for itself (a few scalars by the first warp).  out may be
// the logits: the tables were read before.
template <typename T>
__global__ void __launch_bounds__(kOneThreads, kOneCtas) distill_onepass_kernel(const T* logits, int64_t ld, T* out,
                                                                                int64_t out_ld, int V, int lg,
                                                                                int bits_at, DistArgs a) {
  extern __shared__ __align__(16) unsigned char dist_smem[];
  __shared__ MaxSum red[kOneThreads / 32];
  __shared__ MaxSum part;
  __shared__ RowFin fin;
  pdl_launch_dependents();
  T* held = reinterpret_cast<T*>(dist_smem);
  uint32_t* bits = reinterpret_cast<uint32_t*>(dist_smem + bits_at);
  const int n = 1 << lg, row = blockIdx.x >> lg, rank = blockIdx.x & (n - 1), t = threadIdx.x;
  const T* z = logits + (int64_t)row * ld;
  const RowSpan sp = row_span(z, V);
  const Slice sl = row_slice(sp, rank, lg);
  const int octs = sl.o1 - sl.o0, half = octs / 2 / kOneThreads * kOneThreads;
  const T* body = z + sp.head + 8 * (int64_t)sl.o0;
  constexpr int kPer = 16 / sizeof(T);  // elements a copy
  for (int o = t; o < half; o += kOneThreads)
#pragma unroll
    for (int e = 0; e < 8; e += kPer) copy16_async(held + 8 * o + e, body + 8 * (int64_t)o + e);
  copy_commit();
  for (int o = half + t; o < octs; o += kOneThreads)
#pragma unroll
    for (int e = 0; e < 8; e += kPer) copy16_async(held + 8 * o + e, body + 8 * (int64_t)o + e);
  copy_commit();
  const bool has_head = sl.first && t < sp.head, has_tail = sl.last && t < sp.tail;
  const int tail_at = sp.head + 8 * sp.octs + t;
  const float z_head = has_head ? to_f(z[t]) : 0.f, z_tail = has_tail ? to_f(z[tail_at]) : 0.f;
  pdl_wait();
  const TableSums u = a.sums[row];
  row_bits<kOneThreads>(a, row, sp, sl, bits);
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bits) + 1;
  const float rT = (float)(1.0 / a.T), c = (float)(1.4426950408889634 / a.T), slack = kSlack / c;
  MaxSum r = {-FLT_MAX, 0.f};
  float top = -FLT_MAX;
  copy_wait<1>();
  int o = t;
#pragma unroll 2
  for (; o < half; o += kOneThreads) {
    Oct<T> v;
    v.load(held + 8 * o);
    add_octet(r, top, v, bytes[o], c, slack);
  }
  copy_wait<0>();
#pragma unroll 2
  for (; o < octs; o += kOneThreads) {
    Oct<T> v;
    v.load(held + 8 * o);
    add_octet(r, top, v, bytes[o], c, slack);
  }
  add_ends(r, z, sp, sl, bits, c);
  put_warp(r, c, red);
  if (t < 32) {
    r = join_warps<kOneThreads / 32>(c, red);
    if (t == 0) part = r;
  }
  cluster_meet();
  if (t < 32) {
    r = warp_merge(t < n ? MaxSum{ld_cluster(&part.m, t), ld_cluster(&part.s, t)} : MaxSum{-FLT_MAX, 0.f}, c);
    const RowFin f = finish_grads(a, row, u, r, c);
    if (t == 0) {
      fin = f;
      if (rank == 0) a.parts[row] = r;
    }
  }
  cluster_arrive();
  __syncthreads();
  const float m = fin.m, coef = fin.A * rT;
  const int lo = sl.first ? 0 : sp.head + 8 * sl.o0, hi = sl.last ? V : sp.head + 8 * sl.o1;
  T* out_row = out + (int64_t)row * out_ld;
  T* dst = out_row + sp.head + 8 * (int64_t)sl.o0;
  if (!fin.flags) {  // whatever the logits are
    for (int j = lo + t; j < hi; j += kOneThreads) from_f(out_row + j, 0.f);
    cluster_wait();
    return;
  }
  if (has_head) from_f(out_row + t, coef * ex2((z_head - m) * c));
  if (has_tail) from_f(out_row + tail_at, coef * ex2((z_tail - m) * c));
  if (aligned16(dst)) {
#pragma unroll 2
    for (o = t; o < octs; o += kOneThreads) {
      Oct<T> v;
      v.load(held + 8 * o);
      float f[8];
      grad_oct(v, f, m, c, coef);
      store_oct(dst + 8 * (int64_t)o, f);
    }
  } else {  // the two rows are not aligned alike
    for (o = t; o < octs; o += kOneThreads) {
      Oct<T> v;
      v.load(held + 8 * o);
      float f[8];
      grad_oct(v, f, m, c, coef);
#pragma unroll
      for (int e = 0; e < 8; ++e) from_f(dst + 8 * (int64_t)o + e, f[e]);
    }
  }
  __syncthreads();
  for (int k = t; k < a.K; k += kOneThreads) {
    const int64_t at = (int64_t)row * a.K + k;
    const int id = a.clean[at];
    if (id >= lo && id < hi) from_f(out_row + id, rT * slot_grad(a, fin, a.ex[at], a.p[at], a.xl[at]));
  }
  cluster_wait();  // a CTA's part outlives its readers
}

// CTAs a row: enough for two waves of four on every SM (777 x 50257 fp32, forward and backward: 119 us with one CTA a
// row, which leaves the second wave a third full, 103 us with four), at most `most`, none for fewer than 4096 tokens.
static int row_split(int N, int V, int most) {
  int n = 1;
  while (n < most && N * n < 8 * 148 && V / (2 * n) >= 4096) n *= 2;
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
  LIBRA_CHECK(div >= 0 && div <= 2 && beta > 0.0 && beta < 1.0 && T >= 1e-6 && T <= 1e6,
              "%s: divergence, beta or temperature", op);
}

// The tables' memory in one allocation: sums, slices' parts, exp(x), p, x - log p, and the tokens unless a.clean has a
// place for them.
static torch::Tensor alloc_tables(DistArgs& a, const torch::Tensor& logits, int64_t splits) {
  const int64_t NK = (int64_t)a.N * a.K, per = sizeof(TableSums) / 4;
  auto buf = torch::empty({a.N * (per + 2 * splits) + (a.clean ? 3 : 4) * NK}, logits.options().dtype(at::kFloat));
  float* p = buf.data_ptr<float>();
  a.sums = reinterpret_cast<TableSums*>(p);
  p += a.N * per;
  a.parts = reinterpret_cast<MaxSum*>(p);
  p += a.N * 2 * splits;
  a.ex = p;
  a.p = p + NK;
  a.xl = p + 2 * NK;
  if (!a.clean) a.clean = reinterpret_cast<int*>(p + 3 * NK);
  return buf;
}

static DistArgs make_args(const torch::Tensor& logits, const torch::Tensor& ids, const torch::Tensor& lps, int64_t div,
                          double beta, bool drop, double T, torch::Tensor& loss, const torch::Tensor& err) {
  LIBRA_CHECK(err.device() == logits.device() && err.scalar_type() == at::kInt, "distill_loss: error word");
  DistArgs a = {};
  a.ids = ids.data_ptr<int64_t>();
  a.lps = lps.data_ptr<float>();
  a.N = (int)logits.size(0);
  a.K = (int)ids.size(1);
  a.div = (int)div;
  a.beta = beta;
  a.T = T;
  a.drop = drop;
  a.loss = loss.data_ptr<float>();
  a.err = err.data_ptr<int>();
  return a;
}

// -> {loss [N], logp [N] or empty, saved}: saved is one fp32 buffer with stats [N, 4], dk [N, K], qk [N, K] and the
// slots' tokens [N, K] (int32) at its front.
std::vector<torch::Tensor> distill_fwd(torch::Tensor logits, torch::Tensor ids, torch::Tensor lps, int64_t div,
                                       double beta, bool drop, double T, c10::optional<torch::Tensor> targets,
                                       torch::Tensor err) {
  check_distill(logits, ids, lps, div, beta, T, "distill_loss");
  const int N = (int)logits.size(0), V = (int)logits.size(1), K = (int)ids.size(1);
  if (targets.has_value())
    LIBRA_CHECK(vec_of(*targets, logits, at::kLong, N), "distill_loss: targets must be contiguous int64 [N] on the "
                "logits' device");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  auto loss = torch::empty({N}, f32), logp = torch::empty({targets.has_value() ? N : 0}, f32);
  DistArgs a = make_args(logits, ids, lps, div, beta, drop, T, loss, err);
  const int n = row_split(N, V, 32), lg = log2_of(n);
  const int64_t NK = (int64_t)N * K;
  auto saved = torch::empty({4 * (int64_t)N + 3 * NK}, f32);
  if (N == 0) return {loss, logp, saved};
  a.stats = saved.data_ptr<float>();
  a.dk = a.stats + 4 * (int64_t)N;
  a.qk = a.dk + NK;
  a.clean = reinterpret_cast<int*>(a.qk + NK);
  auto work = alloc_tables(a, logits, n);
  a.targets = targets.has_value() ? targets->data_ptr<int64_t>() : nullptr;
  a.logp = logp.data_ptr<float>();
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const int rows = (N + kTableWarps - 1) / kTableWarps;
  const size_t smem = (slice_octs(V, n) + 2 + 3) / 4 * 4;
  auto go = [&](auto* p) {
    using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    const int64_t ld = logits.stride(0);
    launch_rows(distill_table_kernel<E>, rows, kTableWarps * 32, 0, 1, false, st, p, ld, V, a);
    launch_rows(distill_sum_kernel<E>, (int64_t)N * n, kFwdThreads, smem, 1, true, st, p, ld, V, lg, a);
    launch_rows(distill_row_kernel<E>, rows, kTableWarps * 32, 0, 1, true, st, p, ld, V, lg, a);
  };
  if (logits.scalar_type() == at::kFloat)
    go((const float*)logits.data_ptr());
  else
    go((const __nv_bfloat16*)logits.data_ptr());
  return {loss, logp, saved};
}

void distill_bwd(torch::Tensor logits, torch::Tensor out, double T, int64_t K, c10::optional<torch::Tensor> targets,
                 torch::Tensor saved, c10::optional<torch::Tensor> g, c10::optional<torch::Tensor> g_lp);

constexpr int64_t kHeldBytes = 40 << 10;   // of a row in one CTA: five such CTAs fill an SM
constexpr int64_t kHeldMost = 190 << 10;

// Loss [N], and the gradient for an upstream gradient of one into out (which may be the logits).
torch::Tensor distill_onepass(torch::Tensor logits, torch::Tensor ids, torch::Tensor lps, int64_t div, double beta,
                              bool drop, double T, torch::Tensor out, torch::Tensor err) {
  check_distill(logits, ids, lps, div, beta, T, "distill_loss_grad");
  const int N = (int)logits.size(0), V = (int)logits.size(1);
  LIBRA_CHECK(out.device() == logits.device() && out.scalar_type() == logits.scalar_type() &&
                  out.sizes() == logits.sizes() && (V <= 1 || out.stride(1) == 1) && (N <= 1 || out.stride(0) >= V),
              "distill_loss_grad: the gradient has the logits' shape and type, unit inner stride");
  check_apart(logits, out, "distill_loss_grad");
  const int size = (int)logits.element_size();
  int n = row_split(N, V, 8);
  while (n < 16 && (int64_t)V * size / n > kHeldBytes) n *= 2;
  if ((int64_t)V * size / n > kHeldMost) {  // a row that 16 CTAs cannot hold: two passes
    auto f = distill_fwd(logits, ids, lps, div, beta, drop, T, c10::nullopt, err);
    distill_bwd(logits, out, T, ids.size(1), c10::nullopt, f[2], c10::nullopt, c10::nullopt);
    return f[0];
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  auto loss = torch::empty({N}, logits.options().dtype(at::kFloat));
  if (N == 0) return loss;
  DistArgs a = make_args(logits, ids, lps, div, beta, drop, T, loss, err);
  auto work = alloc_tables(a, logits, 1);
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const int octs = slice_octs(V, n), bits_at = octs * 8 * size, rows = (N + kTableWarps - 1) / kTableWarps;
  const size_t smem = bits_at + (octs + 2 + 3) / 4 * 4;
  auto go = [&](auto* p) {
    using E = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    const int64_t ld = logits.stride(0);
    launch_rows(distill_table_kernel<E>, rows, kTableWarps * 32, 0, 1, false, st, p, ld, V, a);
    launch_rows(distill_onepass_kernel<E>, (int64_t)N * n, kOneThreads, smem, n, true, st, p, ld, (E*)out.data_ptr(),
                out.stride(0), V, log2_of(n), bits_at, a);
    launch_rows(distill_row_kernel<E>, rows, kTableWarps * 32, 0, 1, true, st, p, ld, V, 0, a);
  };
  if (logits.scalar_type() == at::kFloat)
    go((const float*)logits.data_ptr());
  else
    go((const __nv_bfloat16*)logits.data_ptr());
  return loss;
}

// Gradient with respect to the logits into out (which may be the logits): g [N] or none for ones, g_lp [N] or none.
void distill_bwd(torch::Tensor logits, torch::Tensor out, double T, int64_t K, c10::optional<torch::Tensor> targets,
                 torch::Tensor saved, c10::optional<torch::Tensor> g, c10::optional<torch::Tensor> g_lp) {
  check_rows(logits, "distill_loss");
  const int N = (int)logits.size(0), V = (int)logits.size(1);
  LIBRA_CHECK(out.device() == logits.device() && out.scalar_type() == logits.scalar_type() &&
                  out.sizes() == logits.sizes() && (V <= 1 || out.stride(1) == 1) && (N <= 1 || out.stride(0) >= V),
              "distill_loss: the gradient has the logits' shape and type, unit inner stride");
  check_apart(logits, out, "distill_loss");
  LIBRA_CHECK(K >= 1 && K <= kDistMax && vec_of(saved, logits, at::kFloat, (4 + 3 * K) * (int64_t)N),
              "distill_loss: saved tensor does not match the logits");
  if (g.has_value()) LIBRA_CHECK(vec_of(*g, logits, at::kFloat, N), "distill_loss: upstream gradient fp32 [N]");
  if (g_lp.has_value())
    LIBRA_CHECK(vec_of(*g_lp, logits, at::kFloat, N) && targets.has_value() &&
                    vec_of(*targets, logits, at::kLong, N),
                "distill_loss: upstream gradient fp32 [N] of the logprobs, with their targets");
  if (N == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const int n = row_split(N, V, 32);
  const float* stats = saved.data_ptr<float>();
  const float *dk = stats + 4 * (int64_t)N, *qk = dk + K * (int64_t)N;
  const int* clean = reinterpret_cast<const int*>(qk + K * (int64_t)N);
  auto go = [&](auto kern, auto* p, auto* o) {
    launch_rows(kern, (int64_t)N * n, kBwdThreads, 0, 1, false, st, p, logits.stride(0), o, out.stride(0), V,
                log2_of(n), (int)K, targets.has_value() ? (const int64_t*)targets->data_ptr<int64_t>() : nullptr, T,
                stats, clean, dk, qk, g.has_value() ? (const float*)g->data_ptr<float>() : nullptr,
                g_lp.has_value() ? (const float*)g_lp->data_ptr<float>() : nullptr);
  };
  if (logits.scalar_type() == at::kFloat)
    go(distill_bwd_kernel<float>, (const float*)logits.data_ptr(), (float*)out.data_ptr());
  else
    go(distill_bwd_kernel<__nv_bfloat16>, (const __nv_bfloat16*)logits.data_ptr(), (__nv_bfloat16*)out.data_ptr());
}

// distill_fwd and distill_bwd as one differentiable function of the logits.  In C++, since a Python function's two trips
// through the interpreter cost a small batch more than its kernels (64 x 151936 bf16, forward and backward: 102 us).
struct DistillLoss : public torch::autograd::Function<DistillLoss> {
  using List = torch::autograd::variable_list;
  static List forward(torch::autograd::AutogradContext* ctx, torch::Tensor logits, torch::Tensor ids,
                      torch::Tensor lps, int64_t div, double beta, bool drop, double T,
                      c10::optional<torch::Tensor> targets, torch::Tensor err) {
    auto r = distill_fwd(logits, ids, lps, div, beta, drop, T, targets, err);
    ctx->save_for_backward({logits, targets.has_value() ? *targets : torch::Tensor(), r[2]});
    ctx->saved_data["T"] = T;
    ctx->saved_data["K"] = ids.size(1);
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }
  static List backward(torch::autograd::AutogradContext* ctx, List up) {
    LIBRA_CHECK(!at::GradMode::is_enabled(), "distill_loss: its gradient is not differentiable");
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor &logits = saved[0], &targets = saved[1];
    List out(9);
    if (!up[0].defined() && !(targets.defined() && up[1].defined())) return out;
    out[0] = torch::empty(logits.sizes(), logits.options());
    const auto g = up[0].defined() ? up[0].contiguous() : torch::zeros({logits.size(0)}, saved[2].options());
    c10::optional<torch::Tensor> t, g_lp;
    if (targets.defined() && up[1].defined()) {
      t = targets;
      g_lp = up[1].contiguous();
    }
    distill_bwd(logits, out[0], ctx->saved_data["T"].toDouble(), ctx->saved_data["K"].toInt(), t, saved[2], g, g_lp);
    return out;
  }
};

// -> {loss [N], logp [N] or empty}, differentiable
std::vector<torch::Tensor> distill_loss(torch::Tensor logits, torch::Tensor ids, torch::Tensor lps, int64_t div,
                                        double beta, bool drop, double T, c10::optional<torch::Tensor> targets,
                                        torch::Tensor err) {
  return DistillLoss::apply(logits, ids, lps, div, beta, drop, T, targets, err);
}

}  // namespace vocab
}  // namespace libra
