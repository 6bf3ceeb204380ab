// Embedding lookup with scaling, and its gradient by sorted tokens.
//
// dW[v] = scale * sum over the positions i with token v of g[i].  The (token, position) pairs are sorted by token
// (stable, so a token's positions stay in order), cut into chunks of equally many pairs whatever the tokens are, and
// every chunk sums its runs of equal tokens in fp32.  A run inside one chunk goes straight to its row; a run that
// crosses a border leaves one partial sum a chunk, which a second kernel joins from left to right.  No atomics: the
// same inputs give the same bits, and a token that fills half the batch is spread over as many CTAs as any other half.
#include "row_moves.cuh"
#include "sorted_keys.cuh"

namespace libra {
namespace embed {

using namespace rows;
using vocab::launch_rows;

// ------------------------------------------------------------------ lookup

template <typename T, int V, typename I>
__global__ void __launch_bounds__(256)
    lookup_kernel(const I* __restrict__ tokens, const T* __restrict__ w, int64_t ld, int64_t rows_w, int64_t first,
                  bool whole, float scale, int H, T* __restrict__ out, int* err) {
  const int64_t i = blockIdx.x;
  const int64_t r = (int64_t)tokens[i] - first;
  const bool here = r >= 0 && r < rows_w;
  if (!here && whole && threadIdx.x == 0) atomicCAS(err, 0, kBadArgument);
  for (int c = threadIdx.x * V; c < H; c += blockDim.x * V) {
    Bits<T, V> b;
    b.zero();
    if (here) {
      b.load(w + r * ld + c);
      if (scale != 1.f) {
        float v[V];
        b.get(v);
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] *= scale;
        b.set(v);
      }
    }
    b.store(out + i * H + c);
  }
}

// ------------------------------------------------------------------ sort

template <typename I>
struct FirstPass {  // from the tokens themselves; what is not in the table sorts behind it
  struct Item {
    uint32_t key;
  };
  const I* tokens;
  int64_t first, rows_w;
  int shift;
  uint32_t mask;
  uint32_t *key_out, *pos_out;
  __device__ __forceinline__ Item load(int i) const {
    const int64_t r = (int64_t)tokens[i] - first;
    return {r >= 0 && r < rows_w ? (uint32_t)r : (uint32_t)rows_w};
  }
  __device__ __forceinline__ int bin(const Item& a) const { return (int)(a.key & mask); }
  __device__ __forceinline__ void put(int i, const Item& a, uint32_t at) {
    key_out[at] = a.key;
    pos_out[at] = (uint32_t)i;
  }
  __device__ __forceinline__ void group(int, uint32_t, uint32_t) {}
};
struct NextPass {
  struct Item {
    uint32_t key, pos;
  };
  const uint32_t *key_in, *pos_in;
  int shift;
  uint32_t mask;
  uint32_t *key_out, *pos_out;
  __device__ __forceinline__ Item load(int i) const { return {__ldcg(key_in + i), __ldcg(pos_in + i)}; }
  __device__ __forceinline__ int bin(const Item& a) const { return (int)((a.key >> shift) & mask); }
  __device__ __forceinline__ void put(int, const Item& a, uint32_t at) {
    key_out[at] = a.key;
    pos_out[at] = a.pos;
  }
  __device__ __forceinline__ void group(int, uint32_t, uint32_t) {}
};

// Radix sort of the tokens by `passes` digits of `bits` bits; the sorted pairs end in buffer (passes - 1) % 2.
template <typename I>
__global__ void __launch_bounds__(sorted::kThreads)
    sort_kernel(const I* __restrict__ tokens, int n, int64_t first, int64_t rows_w, int passes, int bits, int ctas,
                uint32_t* buf) {
  extern __shared__ uint32_t sm[];
  const uint32_t mask = (1u << bits) - 1;
  uint32_t* at[2] = {buf, buf + 2 * (int64_t)n};
  FirstPass<I> p0{tokens, first, rows_w, 0, mask, at[0], at[0] + n};
  sorted::counting_pass(n, 1 << bits, 1u, sm, ctas, p0);
  for (int p = 1; p < passes; ++p) {
    NextPass q{at[(p - 1) & 1], at[(p - 1) & 1] + n, p * bits, mask, at[p & 1], at[p & 1] + n};
    sorted::counting_pass(n, 1 << bits, 1u, sm, ctas, q);
  }
}

// ------------------------------------------------------------------ sums of runs

struct Target {  // where a row's gradient goes
  void* out;     // dense: the gradient, of the table's type
  float* main;   // or an fp32 buffer that it is added to
  float scale;
};

template <typename T, int V>
__device__ __forceinline__ void write_row(const Target& to, uint32_t row, int H, int c, const float (&acc)[V]) {
  const int64_t o = (int64_t)row * H + c;
  if (to.main) {
    if constexpr (V == 1) {
      to.main[o] = fmaf(to.scale, acc[0], to.main[o]);
    } else {
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        float4* p = reinterpret_cast<float4*>(to.main + o + q);
        float4 m = *p;
        m.x = fmaf(to.scale, acc[q], m.x);
        m.y = fmaf(to.scale, acc[q + 1], m.y);
        m.z = fmaf(to.scale, acc[q + 2], m.z);
        m.w = fmaf(to.scale, acc[q + 3], m.w);
        *p = m;
      }
    }
  } else {
    float v[V];
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] = acc[q] * to.scale;
    Bits<T, V> b;
    b.set(v);
    b.store((T*)to.out + o);
  }
}

template <int V>
__device__ __forceinline__ void write_part(float* p, const float (&acc)[V]) {
#pragma unroll
  for (int q = 0; q < V; ++q) p[q] = acc[q];
}

// CTA (chunk, column slice): sorted pairs [chunk * L, chunk * L + L).  parts holds two fp32 rows a chunk: the sum of a
// run that came in from the chunk before, and that of one that starts here and goes on into the next.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    run_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ pos, int n, int L, uint32_t rows_w,
               const T* __restrict__ g, int64_t ldg, int H, Target to, float* __restrict__ parts) {
  const int lo = blockIdx.x * L, hi = min(n, lo + L);
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (c >= H) return;
  const uint32_t before = lo > 0 ? key[lo - 1] : 0xffffffffu, after = hi < n ? key[hi] : 0xffffffffu;
  float* part = parts + 2 * (int64_t)blockIdx.x * H + c;
  float acc[V] = {};
  uint32_t now = key[lo];
  bool from_left = now == before;
  for (int i = lo; i < hi; ++i) {
    if (now >= rows_w) return;  // tokens outside the table, behind all others
    Bits<T, V> b;
    b.load_once(g + (int64_t)pos[i] * ldg + c);
    float v[V];
    b.get(v);
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] += v[q];
    const uint32_t next = i + 1 < hi ? key[i + 1] : after;
    if (next != now || i + 1 == hi) {
      if (from_left)
        write_part<V>(part, acc);
      else if (next == now)
        write_part<V>(part + H, acc);
      else
        write_row<T, V>(to, now, H, c, acc);
#pragma unroll
      for (int q = 0; q < V; ++q) acc[q] = 0.f;
      now = next;
      from_left = false;
    }
  }
}

// CTA (chunk, column slice): joins the run that starts in this chunk and goes on into the next ones, if there is one.
template <typename T, int V>
__global__ void __launch_bounds__(256)
    join_kernel(const uint32_t* __restrict__ key, int n, int L, uint32_t rows_w, int H, Target to,
                const float* __restrict__ parts) {
  const int64_t hi = (int64_t)(blockIdx.x + 1) * L;
  if (hi >= n) return;
  const uint32_t k = key[hi - 1];
  if (k >= rows_w || key[hi] != k) return;
  const int lo = blockIdx.x * L;
  if (lo > 0 && key[lo - 1] == k) return;  // it came in from the left: that chunk joins it
  int a = (int)hi, b = n;                  // the run's end: the first pair behind hi with another token
  while (a < b) {
    const int mid = a + (b - a) / 2;
    if (key[mid] > k) b = mid; else a = mid + 1;
  }
  const int last = (a - 1) / L;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
  if (c >= H) return;
  float acc[V];
  const float* p = parts + (2 * (int64_t)blockIdx.x + 1) * H + c;
#pragma unroll
  for (int q = 0; q < V; ++q) acc[q] = p[q];
#pragma unroll 4
  for (int j = blockIdx.x + 1; j <= last; ++j) {
    p = parts + 2 * (int64_t)j * H + c;
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] += p[q];
  }
  write_row<T, V>(to, k, H, c, acc);
}

static void check_tokens(const torch::Tensor& tokens, const torch::Tensor& w, const char* op) {
  LIBRA_CHECK(w.is_cuda() && w.dim() == 2 && row_type(w) && (w.size(1) <= 1 || w.stride(1) == 1),
              "%s: the table must be a 2-D bf16 or fp32 CUDA tensor with a unit inner stride", op);
  LIBRA_CHECK(tokens.device() == w.device() && tokens.is_contiguous() &&
                  (tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt),
              "%s: tokens must be int64 or int32 on the table's device", op);
  LIBRA_CHECK(tokens.numel() < (1ll << 30) && w.size(0) < (1ll << 30) && w.size(1) < (1ll << 30),
              "%s: too many tokens, or too large a table", op);
}

template <typename F>
static void by_token(const torch::Tensor& t, F&& go) {
  if (t.scalar_type() == at::kLong)
    go((const int64_t*)t.data_ptr<int64_t>());
  else
    go((const int*)t.data_ptr<int>());
}
template <typename F>
static void by_row(const torch::Tensor& t, bool vec, F&& go) {
  if (t.scalar_type() == at::kFloat) {
    if (vec) go((float*)nullptr, std::integral_constant<int, 4>());
    else go((float*)nullptr, std::integral_constant<int, 1>());
  } else {
    if (vec) go((__nv_bfloat16*)nullptr, std::integral_constant<int, 8>());
    else go((__nv_bfloat16*)nullptr, std::integral_constant<int, 1>());
  }
}

// out [n, H]; whole: a token outside the table is an error, else it is another shard's.
torch::Tensor embedding_fwd(torch::Tensor tokens, torch::Tensor w, double scale, int64_t first, bool whole,
                            torch::Tensor err) {
  check_tokens(tokens, w, "embedding");
  LIBRA_CHECK(err.device() == w.device() && err.scalar_type() == at::kInt, "embedding: error word");
  const int64_t n = tokens.numel(), H = w.size(1);
  const c10::cuda::CUDAGuard guard(w.device());
  auto sizes = tokens.sizes().vec();
  sizes.push_back(H);
  auto out = torch::empty(sizes, w.options());
  if (n == 0 || H == 0) return out;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  by_row(w, row_vectors(w), [&](auto* p, auto v) {
    using T = std::remove_pointer_t<decltype(p)>;
    constexpr int V = decltype(v)::value;
    const int threads = (int)std::min<int64_t>(256, ((H + V - 1) / V + 31) / 32 * 32);
    by_token(tokens, [&](auto* tk) {
      using I = std::remove_const_t<std::remove_pointer_t<decltype(tk)>>;
      launch_rows(lookup_kernel<T, V, I>, n, threads, 0, 1, false, st, tk, (const T*)w.data_ptr(), w.stride(0),
                  w.size(0), first, whole, (float)scale, (int)H, (T*)out.data_ptr(), err.data_ptr<int>());
    });
  });
  return out;
}

// Gradient of the table w [rows, H] from g [n, H]: added to main (fp32, contiguous) or returned, of w's type.
torch::Tensor embedding_bwd(torch::Tensor tokens, torch::Tensor g, torch::Tensor w, double scale, int64_t first,
                            c10::optional<torch::Tensor> main) {
  check_tokens(tokens, w, "embedding");
  const int64_t n = tokens.numel(), H = w.size(1), R = w.size(0);
  LIBRA_CHECK(g.device() == w.device() && g.dim() == 2 && g.size(0) == n && g.size(1) == H &&
                  g.scalar_type() == w.scalar_type(),
              "embedding: the gradient must be [tokens, H] of the table's type");
  if (main.has_value())
    LIBRA_CHECK(main->device() == w.device() && main->scalar_type() == at::kFloat && main->is_contiguous() &&
                    main->numel() == R * H,
                "embedding: main_grad must be contiguous fp32 of the table's shape");
  const c10::cuda::CUDAGuard guard(w.device());
  g = unit_inner(g);
  torch::Tensor out;
  if (!main.has_value()) out = torch::zeros({R, H}, w.options());
  if (n == 0 || H == 0 || R == 0) return out;
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  int total = 1;
  while ((R >> total) != 0) ++total;  // bits of the largest key, R itself
  const int passes = (total + 9) / 10, bits = (total + passes - 1) / passes;
  const int ctas = sorted::sort_ctas(n);
  const int L = n <= 16384 ? 16 : 64;
  const int64_t chunks = (n + L - 1) / L;
  auto buf = torch::empty({4 * n}, w.options().dtype(at::kInt));
  auto parts = torch::empty({chunks, 2, H}, w.options().dtype(at::kFloat));
  uint32_t* b = (uint32_t*)buf.data_ptr<int>();
  by_token(tokens, [&](auto* tk) {
    using I = std::remove_const_t<std::remove_pointer_t<decltype(tk)>>;
    launch_rows(sort_kernel<I>, ctas, sorted::kThreads, sorted::pass_smem(1 << bits), ctas, false, st, tk, (int)n,
                first, R, passes, bits, ctas, b);
  });
  const uint32_t *key = b + ((passes - 1) & 1) * 2 * n, *pos = key + n;
  const Target to{main.has_value() ? nullptr : out.data_ptr(), main.has_value() ? main->data_ptr<float>() : nullptr,
                  (float)scale};
  const bool vec = row_vectors(g) && H % 8 == 0 && (main.has_value() ? reinterpret_cast<uintptr_t>(to.main) % 16 == 0
                                                                      : row_vectors(out));
  by_row(g, vec, [&](auto* p, auto v) {
    using T = std::remove_pointer_t<decltype(p)>;
    constexpr int V = decltype(v)::value;
    const int64_t lanes = (H + V - 1) / V;
    const int threads = (int)std::min<int64_t>(128, (lanes + 31) / 32 * 32);
    const dim3 grid((unsigned)chunks, (unsigned)((lanes + threads - 1) / threads));
    run_kernel<T, V><<<grid, threads, 0, st>>>(key, pos, (int)n, L, (uint32_t)R, (const T*)g.data_ptr(), g.stride(0),
                                               (int)H, to, parts.data_ptr<float>());
    LIBRA_LAUNCH_CHECK();
    join_kernel<T, V><<<grid, threads, 0, st>>>(key, (int)n, L, (uint32_t)R, (int)H, to, parts.data_ptr<float>());
    LIBRA_LAUNCH_CHECK();
  });
  return out;
}

}  // namespace embed
}  // namespace libra
