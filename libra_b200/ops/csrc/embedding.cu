// Embedding lookup with scaling, and its gradient by sorted tokens.
//
// dW[v] = scale * sum over the positions i with token v of g[i].  The (token, position) pairs are sorted by token
// (stable, so a token's positions stay in order) and cut into chunks of equally many pairs, whatever the tokens are.  A
// CTA sums the runs of equal tokens that start in its chunk, in fp32, and writes each to its row once.  A run that goes
// on through the whole next chunk is shared: every chunk leaves its part of it, and a second kernel joins the parts
// from left to right.  Each row is written by one thread a column, so the same inputs give the same bits, and a token
// that fills half the batch is spread over as many CTAs as any other half.
//
// A forward pass whose table wants a gradient sorts its tokens in the first CTAs of the lookup's own launch: the sort
// is a chain of barriers on a few SMs that moves next to nothing, and the lookup has the others meanwhile (8192 tokens of
// 2560 bf16: 16.4 us without the sort, 20.5 with it; of 8, where next to nothing is moved: 4.2 and 18).
#include "row_moves.cuh"
#include "sorted_keys.cuh"

namespace libra {
namespace embed {

using namespace rows;
using vocab::launch_rows;

struct Tokens {
  const void* p;
  bool wide;  // int64
  int64_t first;
  int rows;   // of the table
  // Row of the table, or `rows` for a token outside it.
  __device__ __forceinline__ uint32_t row(int i) const {
    const int64_t r = (wide ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int*>(p)[i]) - first;
    return r >= 0 && r < rows ? (uint32_t)r : (uint32_t)rows;
  }
};

// ------------------------------------------------------------------ sort

struct Digit {
  int shift;
  uint32_t mask;
  __device__ __forceinline__ int of(uint32_t key) const { return (int)((key >> shift) & mask); }
};

struct FirstPass {  // from the tokens themselves; notes which rows occur
  struct Item {
    uint32_t key;
  };
  Tokens tk;
  Digit d;
  uint32_t *key_out, *pos_out, *seen;
  __device__ __forceinline__ Item load(int i) const { return {tk.row(i)}; }
  __device__ __forceinline__ int bin(const Item& a) const { return d.of(a.key); }
  __device__ __forceinline__ void put(int i, const Item& a, uint32_t at) {
    key_out[at] = a.key;
    pos_out[at] = (uint32_t)i;
    if (a.key < (uint32_t)tk.rows) atomicOr(seen + (a.key >> 5), 1u << (a.key & 31));
  }
  __device__ __forceinline__ void group(int, uint32_t, uint32_t) {}
};
struct NextPass {
  struct Item {
    uint32_t key, pos;
  };
  const uint32_t *key_in, *pos_in;
  Digit d;
  uint32_t *key_out, *pos_out;
  __device__ __forceinline__ Item load(int i) const { return {__ldcg(key_in + i), __ldcg(pos_in + i)}; }
  __device__ __forceinline__ int bin(const Item& a) const { return d.of(a.key); }
  __device__ __forceinline__ void put(int, const Item& a, uint32_t at) {
    key_out[at] = a.key;
    pos_out[at] = a.pos;
  }
  __device__ __forceinline__ void group(int, uint32_t, uint32_t) {}
};

// What a sort leaves: keys [n], positions [n], and a bit for every row of the table that occurs.
struct Order {
  uint32_t *key, *pos, *seen, *scratch;  // scratch: 2 n
  int n, passes, bits, ctas;
};
// Warps of a sorting CTA.  Few are quicker while a warp's 512 counters outnumber its tokens (2048 tokens: 12 us of the
// device with 8, 16 with 32), many for longer batches, whose lookup they also leave alone on their SMs (131072 x 2560:
// 232 us with 8, 204 with 32, 184 for the lookup alone).
constexpr int kFewWarps = 8, kManyWarps = 32, kFewTokens = 4096;
constexpr int kDigit = 9;  // at most sorted::kWordBins bins a pass

template <int kWarps>
__device__ __forceinline__ void sort_tokens(const Tokens& tk, const Order& o, uint32_t* sm) {
  const uint32_t mask = (1u << o.bits) - 1;
  const int words = (tk.rows + 31) / 32;
  // cleared before the first put: a pass's barriers lie between
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < words; i += o.ctas * blockDim.x) o.seen[i] = 0;
  auto key = [&](int p) { return ((o.passes - 1 - p) & 1) ? o.scratch : o.key; };
  auto pos = [&](int p) { return ((o.passes - 1 - p) & 1) ? o.scratch + o.n : o.pos; };
  FirstPass p0{tk, {0, mask}, key(0), pos(0), o.seen};
  sorted::counting_pass<kWarps>(o.n, 1 << o.bits, 1u, sm, o.ctas, p0);
  for (int p = 1; p < o.passes; ++p) {
    NextPass q{key(p - 1), pos(p - 1), {p * o.bits, mask}, key(p), pos(p)};
    sorted::counting_pass<kWarps>(o.n, 1 << o.bits, 1u, sm, o.ctas, q);
  }
}

// ------------------------------------------------------------------ lookup

// A warp takes an equal part of a row, at most eight loads a lane: part p of item i is unit i * parts + p.  Bound by DRAM
// and L2: 8192 text-like tokens x 2560 bf16 in 16.4 us with the launch (76 MB), 131072 in 184 us (1.34 GB through L2).
constexpr int kLookLoads = 8;
struct Parts {
  int parts, per;  // per: lanes of a part, a multiple of 32
};
template <class B>
static Parts parts_of(int H) {
  const int lanes = B::lanes(H), parts = std::max(1, (lanes + 32 * kLookLoads - 1) / (32 * kLookLoads));
  return {parts, ((lanes + parts - 1) / parts + 31) / 32 * 32};
}

template <class B>
__device__ __forceinline__ void look_up(const Tokens& tk, int64_t unit, const Parts& pt, const typename B::T* w, int64_t ld,
                                        bool whole, float scale, int H, typename B::T* out, int* err) {
  const int i = (int)(unit / pt.parts), p = (int)(unit - (int64_t)i * pt.parts);
  const int lane = threadIdx.x & 31, c = p * pt.per + lane, stop = min(B::lanes(H), (p + 1) * pt.per);
  const uint32_t r = tk.row(i);
  const bool here = r < (uint32_t)tk.rows;
  if (!here && whole && lane == 0) atomicCAS(err, 0, kBadArgument);
  const typename B::T* src = w + (int64_t)r * ld;
  typename B::T* dst = out + (int64_t)i * H;
  B b[kLookLoads];
#pragma unroll
  for (int u = 0; u < kLookLoads; ++u) {
    if (here && c + 32 * u < stop) b[u].load(src, c + 32 * u, H);
    else b[u].zero();
  }
#pragma unroll
  for (int u = 0; u < kLookLoads; ++u) {
    if (c + 32 * u >= stop) break;
    if (scale != 1.f) {
      float v[B::V];
      b[u].get(v);
#pragma unroll
      for (int q = 0; q < B::V; ++q) v[q] *= scale;
      b[u].set(v);
    }
    b[u].store(dst, c + 32 * u, H);
  }
}

constexpr int kLookWarps = 4;
template <class B>
__global__ void __launch_bounds__(kLookWarps * 32)
    lookup_kernel(Tokens tk, int64_t units, Parts pt, const typename B::T* __restrict__ w, int64_t ld, bool whole,
                  float scale, int H, typename B::T* __restrict__ out, int* err) {
  const int64_t u = (int64_t)blockIdx.x * kLookWarps + (threadIdx.x >> 5);
  if (u < units) look_up<B>(tk, u, pt, w, ld, whole, scale, H, out, err);
}

// The first cluster sorts, the CTAs behind it look up.
template <class B, int kWarps>
__global__ void __launch_bounds__(kWarps * 32)
    lookup_sort_kernel(Tokens tk, Order o, int64_t units, Parts pt, const typename B::T* __restrict__ w, int64_t ld,
                       bool whole, float scale, int H, typename B::T* __restrict__ out, int* err) {
  extern __shared__ uint32_t sm[];
  if ((int)blockIdx.x < o.ctas) {
    sort_tokens<kWarps>(tk, o, sm);
    return;
  }
  const int64_t warps = (int64_t)(gridDim.x - o.ctas) * kWarps;
  for (int64_t u = (int64_t)(blockIdx.x - o.ctas) * kWarps + (threadIdx.x >> 5); u < units; u += warps)
    look_up<B>(tk, u, pt, w, ld, whole, scale, H, out, err);
}

// ------------------------------------------------------------------ sums of runs

constexpr uint32_t kNoKey = 0xffffffffu;

struct Target {  // where a row's gradient goes
  void* out;     // dense: the gradient, of the table's type
  float* main;   // or an fp32 buffer that it is added to
  float scale;
};

template <class B>
__device__ __forceinline__ void write_row(const Target& to, uint32_t row, int i, int H, float (&acc)[B::V]) {
#pragma unroll
  for (int q = 0; q < B::V; ++q) acc[q] *= to.scale;
  if (to.main) {
    float* m = to.main + (int64_t)row * H;
    B::sum_f(m, i, H, acc);
    B::put_f(m, i, H, acc);
  } else {
    B b;
    b.set(acc);
    b.store((typename B::T*)to.out + (int64_t)row * H, i, H);
  }
}

// A chunk has L pairs, the last one fewer; the grid's first `chunks * slices` CTAs take one each, for a slice of the rows'
// lanes.  parts holds two fp32 rows a chunk: its part of a shared run that came in from the left, and of one that starts
// here.  The CTAs behind clear the rows of a dense gradient that no token names.
//
// Loads run ahead of the sums by U pairs, those of main's rows too (kMain): a run is one or two pairs long as a rule,
// and what a row's sum is added to would else be waited for at every run.  Bound by DRAM: 8192 text-like tokens x 2560
// into main take 40 us with the join (178 MB, 0.68 of the copy rate), into a dense gradient of 151936 rows 136 us (0.92).
// Tried without gain: reductions at L2 instead of loads and stores of main (43 us for this kernel against 33), pairs
// copied ahead into shared memory (50), four elements a lane (34), chunks of 8 and 32 (32 and 37).
constexpr int kRunThreads = 192;  // at most
template <class B, int L, bool kMain>
__global__ void __launch_bounds__(kRunThreads)
    run_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos, const uint32_t* __restrict__ seen,
               int n, uint32_t R, const typename B::T* __restrict__ g, int64_t ldg, int H, int chunks, int slices,
               Target to, float* __restrict__ parts) {
  static_assert(L <= 32, "a warp looks at a chunk");
  pdl_launch_dependents();  // join_kernel may look for its runs; it waits for this kernel's end before it reads parts
  const int lane = threadIdx.x & 31, lanes = B::lanes(H);
  if ((int)blockIdx.x >= chunks * slices) {
    const int warp = (blockIdx.x - chunks * slices) * (blockDim.x / 32) + (threadIdx.x >> 5);
    const int warps = (gridDim.x - chunks * slices) * (blockDim.x / 32);
    B z;
    z.zero();
    for (uint32_t r = warp; r < R; r += warps) {
      if (seen[r >> 5] >> (r & 31) & 1) continue;
      for (int c = lane; c < lanes; c += 32) z.store((typename B::T*)to.out + (int64_t)r * H, c, H);
    }
    return;
  }
  __shared__ uint32_t sk[3 * L + 2];
  __shared__ int2 pair[2 * L];  // {position, row of the table | what follows << 30} of this CTA's pairs
  const int chunk = blockIdx.x / slices, i = (blockIdx.x - chunk * slices) * blockDim.x + threadIdx.x;
  const int lo = chunk * L, hi = min(n, lo + L);
  for (int t = threadIdx.x; t < 3 * L + 2; t += blockDim.x) {
    const int at = lo - L - 1 + t;
    sk[t] = at >= 0 && at < n ? key[at] : kNoKey;
  }
  __syncthreads();
  auto K = [&](int at) { return sk[at - (lo - L - 1)]; };

  // pairs [beg, end) are this CTA's
  int beg = lo, end = hi;
  const uint32_t k0 = K(lo), k1 = K(hi - 1);
  const bool from_left = K(lo - 1) == k0;
  if (from_left && K(lo - L - 1) != k0) {  // it starts in the chunk before ...
    const int same = __ffs(~__ballot_sync(0xffffffffu, lane < hi - lo && K(lo + lane) == k0)) - 1;
    const int stop = lo + (same < 0 ? 32 : same);
    if (stop < hi || K(hi) != k0) beg = stop;  // ... and ends in this one: that chunk sums it
  }
  const bool from_far = from_left && beg == lo;
  if (K(hi) == k1) {
    const int same = __ffs(~__ballot_sync(0xffffffffu, lane < L && K(hi + lane) == k1)) - 1;
    const int stop = hi + (same < 0 ? 32 : same);
    const bool here = !(from_far && k1 == k0) && beg < hi;  // the run starts in this chunk
    if (here && K(stop) != k1) end = stop;                  // (stop <= hi + L) and ends in the next
  }
  // what becomes of the sum behind a pair: it goes on, is a part from the left or to the right, or a row
  enum { kOn, kLeft, kRight, kRow };
  for (int t = threadIdx.x; t < end - beg; t += blockDim.x) {
    const int at = beg + t;
    const uint32_t k = K(at);
    const bool more = K(at + 1) == k;
    const uint32_t what = more && at + 1 < end ? kOn : from_far && k == k0 ? kLeft : more ? kRight : kRow;
    pair[t] = k < R ? make_int2((int)pos[at], (int)(k | what << 30)) : make_int2(-1, 0);
  }
  __syncthreads();
  if (i >= lanes) return;
  float* part = parts + 2 * (int64_t)chunk * H;
  float acc[B::V] = {};
  constexpr int U = kMain ? 4 : 8;
  for (int s = 0; s < end - beg; s += U) {
    B b[U];
    float m[kMain ? U : 1][B::V];
    int2 p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[u] = s + u < end - beg ? pair[s + u] : make_int2(-1, 0);
      if (p[u].x >= 0) b[u].load_once(g + p[u].x * ldg, i, H);
      if constexpr (kMain) {
        if ((uint32_t)p[u].y >> 30 == kRow) B::get_f(to.main + (int64_t)(p[u].y & 0x3fffffff) * H, i, H, m[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p[u].x < 0) return;  // the end, or tokens outside the table, behind all others
      float v[B::V];
      b[u].get(v);
#pragma unroll
      for (int q = 0; q < B::V; ++q) acc[q] += v[q];
      const uint32_t what = (uint32_t)p[u].y >> 30, k = p[u].y & 0x3fffffff;
      if (what == kOn) continue;
      if (what == kRow) {
        if constexpr (kMain) {
#pragma unroll
          for (int q = 0; q < B::V; ++q) acc[q] = fmaf(acc[q], to.scale, m[u][q]);
          B::put_f(to.main + (int64_t)k * H, i, H, acc);
        } else {
          write_row<B>(to, k, i, H, acc);
        }
      } else {
        B::put_f(what == kLeft ? part : part + H, i, H, acc);
      }
#pragma unroll
      for (int q = 0; q < B::V; ++q) acc[q] = 0.f;
    }
  }
}

// Joins the shared runs.  A CTA looks at eight chunks for runs that start there and go on through the whole next chunk,
// by the order alone and so ahead of run_kernel's end, and sums their parts for 32 lanes of the row: warp w those of
// chunks w, w + 8, ... behind the first, and the warps' sums in their order.
constexpr int kJoinChunks = 8, kJoinWarps = 8;
template <class B, int L>
__global__ void __launch_bounds__(kJoinWarps * 32)
    join_kernel(const uint32_t* __restrict__ key, int n, uint32_t R, int H, int slices, Target to,
                const float* __restrict__ parts) {
  __shared__ float sums[kJoinWarps][B::V][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int block = blockIdx.x / slices, i = (blockIdx.x - block * slices) * 32 + lane;
  const int64_t lo = (int64_t)(block * kJoinChunks + lane) * L, hi = lo + L;
  uint32_t k = kNoKey;
  bool starts = false;
  if (lane < kJoinChunks && hi + L < n) {
    k = key[hi - 1];
    const uint32_t far = key[hi + L], before = lo ? key[lo - 1] : kNoKey;
    starts = k < R && far == k && before != k;
  }
  uint32_t todo = __ballot_sync(0xffffffffu, starts);
  if (todo == 0) {
    pdl_wait();
    return;
  }
  int last = 0;  // of the run that starts in this lane's chunk
  for (uint32_t left = todo; left; left &= left - 1) {
    const int j = __ffs(left) - 1;
    const uint32_t kj = __shfl_sync(0xffffffffu, k, j);
    // the first pair behind the run lies in [a, b]; the lanes look at 32 places between them at a time
    int a = (block * kJoinChunks + j + 2) * L, b = n;
    while (a < b) {
      const int at = a + (int)((int64_t)(b - a) * lane / 32);
      const uint32_t same = __ballot_sync(0xffffffffu, key[at] <= kj);
      if (same == 0) break;  // a itself
      const int top = 31 - __clz(same), from = a;
      a = from + (int)((int64_t)(b - from) * top / 32) + 1;
      if (top < 31) b = from + (int)((int64_t)(b - from) * (top + 1) / 32);
    }
    if (lane == j) last = (a - 1) / L;
  }
  pdl_wait();
  const bool here = i < B::lanes(H);
  for (; todo; todo &= todo - 1) {
    const int j = __ffs(todo) - 1, chunk = block * kJoinChunks + j;
    const int end = __shfl_sync(0xffffffffu, last, j);
    float acc[B::V] = {};
    if (here) {
#pragma unroll 8
      for (int c = chunk + warp; c <= end; c += kJoinWarps)
        B::sum_f(parts + (2 * (int64_t)c + (c == chunk ? 1 : 0)) * H, i, H, acc);
    }
#pragma unroll
    for (int q = 0; q < B::V; ++q) sums[warp][q][lane] = acc[q];
    __syncthreads();
    const uint32_t kj = __shfl_sync(0xffffffffu, k, j);
    if (warp == 0 && here) {
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w) {
#pragma unroll
        for (int q = 0; q < B::V; ++q) acc[q] += sums[w][q][lane];
      }
      write_row<B>(to, kj, i, H, acc);
    }
    __syncthreads();
  }
}

static void check_tokens(const torch::Tensor& tokens, const torch::Tensor& w) {
  ROWS_CHECK(w.is_cuda() && w.dim() == 2 && row_type(w), "embedding: weight must be [V, H], bf16 or fp32");
  ROWS_CHECK(w.size(1) <= 1 || w.stride(1) == 1, "embedding: the weight's rows must be contiguous");
  ROWS_CHECK(tokens.device() == w.device() && (tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt),
             "embedding: tokens must be int64 or int32 on the weight's device");
  ROWS_CHECK(tokens.numel() < (1ll << 30) && w.size(0) < (1ll << 30) && w.size(1) < (1ll << 30),
             "embedding: too many tokens, or too large a table");
}

// -> {rows [*tokens, H], order or nothing}; whole: a token outside the table is an error, else it is another shard's;
// want_order: the tokens' order too, which embedding_bwd takes.
std::vector<torch::Tensor> embedding_fwd(torch::Tensor tokens, torch::Tensor w, double scale, int64_t first, bool whole,
                                         bool want_order, torch::Tensor err) {
  check_tokens(tokens, w);
  tokens = tokens.contiguous();
  LIBRA_CHECK(err.device() == w.device() && err.scalar_type() == at::kInt, "embedding: error word");
  const int64_t n = tokens.numel(), H = w.size(1), R = w.size(0);
  const c10::cuda::CUDAGuard guard(w.device());
  auto sizes = tokens.sizes().vec();
  sizes.push_back(H);
  auto out = torch::empty(sizes, w.options());
  torch::Tensor order;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const Tokens tk{tokens.data_ptr(), tokens.scalar_type() == at::kLong, first, (int)R};
  if (want_order) order = torch::empty({4 * n + (R + 31) / 32}, w.options().dtype(at::kInt));  // 2 n of it scratch
  if (n == 0 || H == 0) return {out, order};
  by_lanes(w, row_vectors(w), [&](auto lanes) {
    using B = decltype(lanes);
    using T = typename B::T;
    const T* table = (const T*)w.data_ptr();
    T* to = (T*)out.data_ptr();
    const Parts pt = parts_of<B>((int)H);
    const int64_t units = n * pt.parts;
    if (!want_order) {
      launch_rows(lookup_kernel<B>, (units + kLookWarps - 1) / kLookWarps, kLookWarps * 32, 0, 1, false, st, tk, units, pt,
                  table, w.stride(0), whole, (float)scale, (int)H, to, err.data_ptr<int>());
      return;
    }
    int total = 1;
    while ((R >> total) != 0) ++total;  // bits of the largest key, R itself
    Order o;
    o.n = (int)n;
    o.passes = (total + kDigit - 1) / kDigit;
    o.bits = (total + o.passes - 1) / o.passes;
    o.ctas = n <= 1024 ? 1 : 8;
    o.key = (uint32_t*)order.data_ptr<int>();
    o.pos = o.key + n;
    o.scratch = o.key + 2 * n;
    o.seen = o.key + 4 * n;
    auto go = [&](auto warps) {
      constexpr int kWarps = decltype(warps)::value;
      // four rounds of 32-warp CTAs (131072 x 2560: 204 us, with one round 235)
      const int64_t look = std::min<int64_t>((units + kWarps - 1) / kWarps, 148 * 4);
      launch_rows(lookup_sort_kernel<B, kWarps>, o.ctas * (1 + (look + o.ctas - 1) / o.ctas), kWarps * 32,
                  sorted::pass_smem(kWarps, 1 << o.bits), o.ctas, false, st, tk, o, units, pt, table, w.stride(0), whole,
                  (float)scale, (int)H, to, err.data_ptr<int>());
    };
    if (n <= kFewTokens)
      go(std::integral_constant<int, kFewWarps>());
    else
      go(std::integral_constant<int, kManyWarps>());
  });
  return {out, order};
}

// Gradient of the table w [rows, H] from g [n, H] and the tokens' order: added to main (fp32, contiguous) or returned,
// of w's type.
torch::Tensor embedding_bwd(torch::Tensor order, torch::Tensor g, torch::Tensor w, double scale,
                            c10::optional<torch::Tensor> main) {
  const int64_t H = w.size(1), R = w.size(0);
  LIBRA_CHECK(g.device() == w.device() && g.dim() >= 1 && g.size(-1) == H && g.scalar_type() == w.scalar_type(),
              "embedding: the gradient must be [*, H] of the table's type");
  if (g.dim() != 2) g = g.reshape({H ? g.numel() / H : 0, H});
  const int64_t n = g.size(0);
  LIBRA_CHECK(order.device() == w.device() && order.scalar_type() == at::kInt && order.is_contiguous() &&
                  (H == 0 || order.numel() == 4 * n + (R + 31) / 32),
              "embedding: the order is not that of these tokens");
  if (main.has_value())
    ROWS_CHECK(main->device() == w.device() && main->scalar_type() == at::kFloat && main->is_contiguous() &&
                    main->numel() == R * H,
                "embedding: main_grad must be contiguous fp32 of the table's shape");
  const c10::cuda::CUDAGuard guard(w.device());
  g = unit_inner(g);
  torch::Tensor out;
  if (n == 0 || H == 0 || R == 0) {
    if (!main.has_value()) out = torch::zeros({R, H}, w.options());
    return out;
  }
  if (!main.has_value()) out = torch::empty({R, H}, w.options());
  const uint32_t *key = (const uint32_t*)order.data_ptr<int>(), *pos = key + n, *seen = key + 4 * n;
  const Target to{main.has_value() ? nullptr : out.data_ptr(), main.has_value() ? main->data_ptr<float>() : nullptr,
                  (float)scale};
  const bool wide = row_vectors(g) && (main.has_value() ? reinterpret_cast<uintptr_t>(to.main) % 16 == 0
                                                         : row_vectors(out));
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  auto sums = [&](auto lanes_type, auto to_main) {
    using B = decltype(lanes_type);
    using T = typename B::T;
    constexpr bool kMain = decltype(to_main)::value;
    auto go = [&](auto len) {
      constexpr int L = decltype(len)::value;
      const int64_t chunks = (n + L - 1) / L;
      const int lanes = B::lanes((int)H), slices = (lanes + kRunThreads - 1) / kRunThreads;
      const int threads = ((lanes + slices - 1) / slices + 31) / 32 * 32;
      const bool shared = n > 2 * L;  // a run can only then go on through a whole chunk
      torch::Tensor parts;
      if (shared) parts = torch::empty({chunks, 2, H}, w.options().dtype(at::kFloat));
      float* const part = shared ? parts.data_ptr<float>() : nullptr;
      const int64_t clear = kMain ? 0 : std::min<int64_t>((R + 3) / 4, 148 * 8);
      LIBRA_CHECK(chunks * slices + clear < (1ll << 31), "embedding: too many tokens");
      launch_rows(run_kernel<B, L, kMain>, chunks * slices + clear, threads, 0, 1, false, st, key, pos, seen, (int)n,
                  (uint32_t)R, (const T*)g.data_ptr(), g.stride(0), (int)H, (int)chunks, slices, to, part);
      if (!shared) return;
      const int wide32 = (lanes + 31) / 32;
      launch_rows(join_kernel<B, L>, (chunks + kJoinChunks - 1) / kJoinChunks * wide32, kJoinWarps * 32, 0, 1, true, st,
                  key, (int)n, (uint32_t)R, (int)H, wide32, to, (const float*)part);
    };
    if (n <= 16384)
      go(std::integral_constant<int, 16>());
    else
      go(std::integral_constant<int, 32>());
  };
  by_lanes(w, wide, [&](auto b) {
    if (main.has_value())
      sums(b, std::true_type());
    else
      sums(b, std::false_type());
  });
  return out;
}

// The fp32 buffer that a parameter's gradients accumulate into, where it has one.
static c10::optional<torch::Tensor> main_grad_of(const torch::Tensor& w) {
  py::gil_scoped_acquire gil;
  const py::object p = py::cast(w);
  const py::object m = py::getattr(p, "main_grad", py::none());
  if (m.is_none()) return c10::nullopt;
  return m.cast<torch::Tensor>();
}

// embedding_fwd and embedding_bwd as one differentiable function of the table.  In C++, since a Python function's trips
// through the interpreter cost a small batch more than its kernels.
struct Embedding : public torch::autograd::Function<Embedding> {
  using List = torch::autograd::variable_list;
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, torch::Tensor tokens, torch::Tensor w,
                               double scale, int64_t first, bool whole, torch::Tensor err) {
    auto r = embedding_fwd(tokens, w, scale, first, whole, true, err);
    ctx->saved_data["w"] = w;  // its shape and main_grad; the values may change before the backward pass
    ctx->saved_data["order"] = r[1];
    ctx->saved_data["scale"] = scale;
    return r[0];
  }
  static List backward(torch::autograd::AutogradContext* ctx, List up) {
    LIBRA_CHECK(!at::GradMode::is_enabled(), "embedding: its gradient is not differentiable");
    const auto w = ctx->saved_data["w"].toTensor();
    auto main = main_grad_of(w);
    List out(6);
    out[1] = embedding_bwd(ctx->saved_data["order"].toTensor(), up[0], w, ctx->saved_data["scale"].toDouble(), main);
    if (main.has_value() && !main->is_inference()) main->unsafeGetTensorImpl()->bump_version();
    return out;
  }
};

torch::Tensor embedding(torch::Tensor tokens, torch::Tensor w, double scale, int64_t first, bool whole,
                        torch::Tensor err) {
  if (at::GradMode::is_enabled() && w.requires_grad()) return Embedding::apply(tokens, w, scale, first, whole, err);
  return embedding_fwd(tokens, w, scale, first, whole, false, err)[0];
}

}  // namespace embed
}  // namespace libra
