// Rows of a mixture-of-experts layer: the router's choice, the plan that sorts (token, slot) pairs by expert, and the
// moves of rows there (dispatch) and back (combine), with their gradients.
//
// Pair j = t * k + i is token t's i-th expert.  The experts' layout gives every expert a group of rows that starts on a
// multiple of `align`; a group's rows behind its pairs, and the rows behind the last group, are padding.
#include "row_moves.cuh"
#include "sorted_keys.cuh"

namespace libra {
namespace experts {

using namespace rows;
using vocab::launch_rows;
using vocab::order_key;
using vocab::key_value;

// ------------------------------------------------------------------ router
//
// A warp takes a row, lane l the experts l, l + 32, ...  Up to 256 experts every lane first sorts its own (key, expert)
// pairs by a fixed network; the largest left over the warp is then the maximum of 32 heads, one redux, and the lane that
// had it moves up one.  Wider rows look through all that a lane has left, k times.  -inf ranks lowest, NaN highest; equal
// logits are taken from the lowest index, which a second redux finds where two lanes tie.  A row of nothing but -inf has
// weights 0.  Slot j belongs to lane j % 32.  Bound by issue slots: 16384 rows of 128 fp32 logits, k = 8: 10 us (2 of them
// the launch; 12 with every lane's four looked through in each of the k rounds), of 512: 47 us.

constexpr int kRouteMax = 1024;  // experts
constexpr int kRouteWarps = 8;

template <int V>
__device__ __forceinline__ void order_pair(uint32_t (&key)[V], uint32_t (&id)[V], int i, int j) {
  // larger keys first, equal ones by the lower expert
  const bool swap = key[j] > key[i] || (key[j] == key[i] && id[j] < id[i]);
  const uint32_t k = key[i], e = id[i];
  key[i] = swap ? key[j] : k;
  id[i] = swap ? id[j] : e;
  key[j] = swap ? k : key[j];
  id[j] = swap ? e : id[j];
}
// Odd-even merge sort (Batcher), V a power of two.
template <int V>
__device__ __forceinline__ void sort_lane(uint32_t (&key)[V], uint32_t (&id)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2) {
#pragma unroll
    for (int k = p; k >= 1; k /= 2) {
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k) {
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) order_pair<V>(key, id, i + j, i + j + k);
      }
    }
  }
}

template <typename T, int V, bool kWide>  // kWide: more than 32 slots
__global__ void __launch_bounds__(kRouteWarps * 32)
    route_fwd_kernel(const T* __restrict__ z, int64_t ld, int N, int E, int k, bool normalize, float* __restrict__ w,
                     int64_t* __restrict__ ids, float2* __restrict__ stats) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (row >= N) return;
  const T* p = z + row * ld;
  float v[V];
  uint32_t key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = 32 * i + lane;
    v[i] = e < E ? to_f(p[e]) : -INFINITY;
    key[i] = e < E ? order_key(v[i]) : 0u;  // no float has key 0
  }
  constexpr bool kSorted = V <= 8;
  uint32_t id[V];
  if constexpr (kSorted) {
#pragma unroll
    for (int i = 0; i < V; ++i) id[i] = 32 * i + lane;
    sort_lane<V>(key, id);
  }
  float top = 0.f, picked = 0.f, sum = 0.f;
  uint32_t mine = 0;
  int at = 0;
  for (int j = 0; j < k; ++j) {
    uint32_t best, first;
    if constexpr (kSorted) {
      best = __reduce_max_sync(0xffffffffu, key[0]);
      const uint32_t have = __ballot_sync(0xffffffffu, key[0] == best);
      if (have & (have - 1))
        first = __reduce_min_sync(0xffffffffu, key[0] == best ? id[0] : 0xffffffffu);
      else
        first = __shfl_sync(0xffffffffu, id[0], __ffs(have) - 1);
      if (id[0] == first) {
#pragma unroll
        for (int i = 0; i + 1 < V; ++i) {
          key[i] = key[i + 1];
          id[i] = id[i + 1];
        }
        key[V - 1] = 0;
      }
    } else {
      best = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) best = max(best, key[i]);
      best = __reduce_max_sync(0xffffffffu, best);
      first = 0xffffffffu;
#pragma unroll
      for (int i = V - 1; i >= 0; --i)
        if (key[i] == best) first = 32 * i + lane;
      first = __reduce_min_sync(0xffffffffu, first);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (first == 32u * i + lane) key[i] = 0;
    }
    if (j == 0) top = key_value(best);
    if (lane == (j & 31)) {
      if (kWide) {
        const float ex = top == -INFINITY ? 0.f : expf(key_value(best) - top);
        w[(int64_t)row * k + j] = ex;
        ids[(int64_t)row * k + j] = first;
        sum += ex;
      } else {
        mine = best;
        at = (int)first;
      }
    }
  }
  if (!kWide && lane < k && top != -INFINITY) sum = picked = expf(key_value(mine) - top);
  if (!normalize) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (32 * i + lane < E && top != -INFINITY) sum += expf(v[i] - top);
  }
  sum = warp_sum(sum);
  const int64_t o = (int64_t)row * k;
  if (kWide) {
    for (int j = lane; j < k; j += 32) w[o + j] = sum == 0.f ? 0.f : w[o + j] / sum;
  } else if (lane < k) {
    w[o + lane] = sum == 0.f ? 0.f : picked / sum;
    ids[o + lane] = at;
  }
  if (stats && lane == 0) stats[row] = make_float2(top, sum);
}

// Gradient of the weights with respect to the logits.  Renormalised weights are a softmax of the chosen logits alone:
// dz_i = w_i (g_i - sum_j w_j g_j), nothing elsewhere.  Otherwise w_i = p_i, and dz_e = p_e ([e chosen] g_e - sum_j w_j
// g_j) with p from the logits and the row's statistics.
template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32)
    route_bwd_kernel(const T* __restrict__ z, int64_t ld, int N, int E, int k, const float* __restrict__ w,
                     const int64_t* __restrict__ ids, const float2* __restrict__ stats, const float* __restrict__ g,
                     T* __restrict__ dz) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (row >= N) return;
  const int64_t o = (int64_t)row * k;
  float inner = 0.f;
  for (int j = lane; j < k; j += 32) inner = fmaf(w[o + j], g[o + j], inner);
  inner = warp_sum(inner);
  float d[V];
  const float2 s = stats ? stats[row] : make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = 32 * i + lane;
    d[i] = s.y != 0.f && e < E ? -expf(to_f(z[row * ld + e]) - s.x) / s.y * inner : 0.f;
  }
  for (int j0 = 0; j0 < k; j0 += 32) {
    float mine = 0.f;
    int at = -1;
    if (j0 + lane < k) {
      const int64_t j = o + j0 + lane;
      mine = w[j] * (stats ? g[j] : g[j] - inner);
      at = (int)ids[j];
    }
    for (int j = 0; j < min(32, k - j0); ++j) {
      const float val = __shfl_sync(0xffffffffu, mine, j);
      const int e = __shfl_sync(0xffffffffu, at, j);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e == 32 * i + lane) d[i] += val;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (32 * i + lane < E) from_f(dz + (int64_t)row * E + 32 * i + lane, d[i]);
}

template <typename F>
static void by_width(int E, F&& go) {
  if (E <= 32) go(std::integral_constant<int, 1>());
  else if (E <= 64) go(std::integral_constant<int, 2>());
  else if (E <= 128) go(std::integral_constant<int, 4>());
  else if (E <= 256) go(std::integral_constant<int, 8>());
  else if (E <= 512) go(std::integral_constant<int, 16>());
  else go(std::integral_constant<int, 32>());
}

// -> {weights fp32 [N, k], experts int64 [N, k], stats fp32 [N, 2] or empty}
static std::vector<torch::Tensor> route_fwd(const torch::Tensor& z, int64_t k, bool normalize, bool want_stats) {
  ROWS_CHECK(z.is_cuda() && z.dim() == 2 && row_type(z), "route_topk: logits must be [T, E], bf16 or fp32");
  const int64_t N = z.size(0), E = z.size(1);
  ROWS_CHECK(E >= 1 && E <= kRouteMax && k >= 1 && k <= E, "route_topk: 1 to %d experts and k in [1, %lld], got %lld and "
             "%lld", kRouteMax, (long long)E, (long long)E, (long long)k);
  ROWS_CHECK(N < (1ll << 31), "route_topk: too many rows");
  const c10::cuda::CUDAGuard guard(z.device());
  auto w = torch::empty({N, k}, z.options().dtype(at::kFloat));
  auto ids = torch::empty({N, k}, z.options().dtype(at::kLong));
  torch::Tensor stats;
  if (want_stats) stats = torch::empty({N, 2}, z.options().dtype(at::kFloat));
  if (N == 0) return {w, ids, stats};
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  by_width((int)E, [&](auto v) {
    auto go = [&](auto* p) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
      constexpr int V = decltype(v)::value;
      launch_rows(k > 32 ? route_fwd_kernel<T, V, true> : route_fwd_kernel<T, V, false>, (N + kRouteWarps - 1) / kRouteWarps, kRouteWarps * 32, 0, 1,
                  false, st, p, z.stride(0), (int)N, (int)E, (int)k, normalize, w.data_ptr<float>(),
                  ids.data_ptr<int64_t>(), want_stats ? (float2*)stats.data_ptr<float>() : (float2*)nullptr);
    };
    if (z.scalar_type() == at::kFloat)
      go((const float*)z.data_ptr());
    else
      go((const __nv_bfloat16*)z.data_ptr());
  });
  return {w, ids, stats};
}

// z: the logits where the weights were not renormalised (stats is then defined); else only E and their type are needed.
static torch::Tensor route_bwd(const torch::Tensor& z, int64_t E, at::ScalarType type, const torch::Tensor& w,
                               const torch::Tensor& ids, const torch::Tensor& stats, const torch::Tensor& g) {
  const int64_t N = w.size(0), k = w.size(1);
  const c10::cuda::CUDAGuard guard(w.device());
  auto dz = torch::empty({N, E}, w.options().dtype(type));
  if (N == 0) return dz;
  by_width((int)E, [&](auto v) {
    auto go = [&](auto* p) {
      using T = std::remove_pointer_t<decltype(p)>;
      launch_rows(route_bwd_kernel<T, decltype(v)::value>, (N + kRouteWarps - 1) / kRouteWarps, kRouteWarps * 32, 0, 1,
                  false, at::cuda::getCurrentCUDAStream(), z.defined() ? (const T*)z.data_ptr() : (const T*)nullptr,
                  z.defined() ? z.stride(0) : 0, (int)N, (int)E, (int)k, (const float*)w.data_ptr<float>(),
                  (const int64_t*)ids.data_ptr<int64_t>(),
                  stats.defined() ? (const float2*)stats.data_ptr<float>() : (const float2*)nullptr,
                  (const float*)g.data_ptr<float>(), (T*)dz.data_ptr());
    };
    if (type == at::kFloat)
      go((float*)nullptr);
    else
      go((__nv_bfloat16*)nullptr);
  });
  return dz;
}

struct RouteTopk : public torch::autograd::Function<RouteTopk> {
  using List = torch::autograd::variable_list;
  static List forward(torch::autograd::AutogradContext* ctx, torch::Tensor z, int64_t k, bool normalize) {
    auto r = route_fwd(z, k, normalize, !normalize);
    ctx->save_for_backward({normalize ? torch::Tensor() : z, r[0], r[1], r[2]});
    ctx->saved_data["E"] = z.size(1);
    ctx->saved_data["type"] = (int64_t)z.scalar_type();
    ctx->mark_non_differentiable({r[1]});
    ctx->set_materialize_grads(false);
    return {r[0], r[1]};
  }
  static List backward(torch::autograd::AutogradContext* ctx, List up) {
    LIBRA_CHECK(!at::GradMode::is_enabled(), "route_topk: its gradient is not differentiable");
    List out(3);
    if (!up[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    out[0] = route_bwd(s[0], ctx->saved_data["E"].toInt(), (at::ScalarType)ctx->saved_data["type"].toInt(), s[1], s[2],
                       s[3], up[0].contiguous());
    return out;
  }
};

// -> weights fp32 [N, k], experts int64 [N, k], differentiable
std::tuple<torch::Tensor, torch::Tensor> route_topk(torch::Tensor z, int64_t k, bool normalize) {
  if (z.dim() == 2) z = unit_inner(z);
  const auto r = at::GradMode::is_enabled() && z.requires_grad() ? RouteTopk::apply(z, k, normalize)
                                                                  : route_fwd(z, k, normalize, false);
  return {r[0], r[1]};
}

// ------------------------------------------------------------------ plan

struct PlanItems {
  using Item = int;
  const void* ids;
  bool wide;  // int64
  int* rows;
  int *offs, *counts;
  int E;
  uint32_t align;
  int* err;
  __device__ __forceinline__ Item load(int i) const {
    const int64_t e = wide ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int*>(ids)[i];
    if (e >= E) {
      atomicCAS(err, 0, kBadArgument);
      return -1;
    }
    return e < 0 ? -1 : (int)e;
  }
  __device__ __forceinline__ int bin(Item e) const { return e; }
  __device__ __forceinline__ void put(int i, Item, uint32_t place) { rows[i] = (int)place; }
  __device__ __forceinline__ void group(int e, uint32_t start, uint32_t count) {
    offs[e] = (int)start;
    counts[e] = (int)count;
    if (e == E - 1) offs[E] = (int)(start + (count + align - 1) / align * align);
  }
};

// CTAs of the cluster: as many as leave a warp the eight items a lane that it keeps in registers (131072 pairs of 128
// experts: 26 us with 8 CTAs that load them twice).
constexpr int kPlanWarps = 32;
static int plan_ctas(int64_t n) {
  int ctas = 1;
  while (ctas < sorted::kMaxCtas && ctas * kPlanWarps * 32 * sorted::kBatch < n) ctas *= 2;
  return ctas;
}

__global__ void __launch_bounds__(kPlanWarps * 32) plan_kernel(int n, int ctas, PlanItems items) {
  extern __shared__ uint32_t sm[];
  sorted::counting_pass<kPlanWarps>(n, items.E, items.align, sm, ctas, items);
}

// experts [T, k] -> rows int32 [T * k], offs int32 [E + 1], counts int32 [E], and the layout's capacity
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, int64_t> expert_plan(torch::Tensor ids, int64_t E, int64_t align,
                                                                             torch::Tensor err) {
  ROWS_CHECK(ids.is_cuda() && ids.dim() == 2 && ids.size(1) >= 1 &&
                 (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
             "expert_plan: experts must be int64 or int32 [T, k]");
  ROWS_CHECK(E >= 1 && E <= sorted::kMaxBins && align >= 1, "expert_plan: 1 to %d experts and align >= 1, got %lld and "
             "%lld", sorted::kMaxBins, (long long)E, (long long)align);
  ids = ids.contiguous();
  const int64_t n = ids.numel();
  // no pairs still leave one group's rows, so that the grouped products have something to stand on
  const int64_t cap = n == 0 && align > 1 ? align : n + (align - 1) * std::min(E, n);
  ROWS_CHECK(n < (1ll << 31) && align < (1ll << 31) && cap < (1ll << 31),
             "expert_plan: %lld pairs with align %lld do not fit 31 bits", (long long)n, (long long)align);
  LIBRA_CHECK(err.device() == ids.device() && err.scalar_type() == at::kInt, "expert_plan: error word");
  const c10::cuda::CUDAGuard guard(ids.device());
  const auto i32 = ids.options().dtype(at::kInt);
  auto rows_t = torch::empty({n}, i32), offs = torch::empty({E + 1}, i32), counts = torch::empty({E}, i32);
  const int ctas = plan_ctas(n);
  PlanItems it{ids.data_ptr(), ids.scalar_type() == at::kLong, rows_t.data_ptr<int>(), offs.data_ptr<int>(),
               counts.data_ptr<int>(), (int)E, (uint32_t)align, err.data_ptr<int>()};
  launch_rows(plan_kernel, ctas, kPlanWarps * 32, sorted::pass_smem(kPlanWarps, (int)E), ctas, false,
              at::cuda::getCurrentCUDAStream(), (int)n, ctas, it);
  return {rows_t, offs, counts, cap};
}

// ------------------------------------------------------------------ moves

struct Plan {
  const int *rows, *offs, *counts;
  int E, k, cap;
  int64_t align;
};

// Zeros into the layout's padding rows by warps [warp, warps): a slot for every row that a group may have as padding,
// then one for every row behind the last group.
template <class B>
__device__ __forceinline__ void clear_padding(const Plan& pl, typename B::T* out, int H, int64_t warp, int64_t warps) {
  const int lane = threadIdx.x & 31, lanes = B::lanes(H);
  const int64_t slots = pl.E * (pl.align - 1), behind = pl.offs[pl.E];
  B z;
  z.zero();
  for (int64_t s = warp; s < slots + (pl.cap - behind); s += warps) {
    int64_t r;
    if (s < slots) {
      const int e = (int)(s / (pl.align - 1));
      r = (int64_t)pl.offs[e] + pl.counts[e] + (s - e * (pl.align - 1));
      if (r >= pl.offs[e + 1]) continue;
    } else {
      r = behind + (s - slots);
    }
    if (r < 0 || r >= pl.cap) continue;
    for (int c = lane; c < lanes; c += 32) z.store(out + r * H, c, H);
  }
}

// A warp copies row t of x to its pairs' rows, eight loads a lane ahead of their k stores; the grid's first `clear` CTAs
// zero the padding, so that it does not trail behind.  Bound by DRAM writes: 16384 x 2048 bf16, top-8 of 128, 112 us for
// 671 MB (0.92 of the copy rate; 101 us against 111 with bulk copies through shared memory where there is no padding).
constexpr int kMoveWarps = 8;
template <class B>
__global__ void __launch_bounds__(kMoveWarps * 32)
    dispatch_kernel(const typename B::T* __restrict__ x, int64_t ld, int N, int H, Plan pl, int clear,
                    typename B::T* __restrict__ out) {
  constexpr int U = 8;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lanes = B::lanes(H);
  if ((int)blockIdx.x < clear) {
    clear_padding<B>(pl, out, H, blockIdx.x * kMoveWarps + warp, (int64_t)clear * kMoveWarps);
    return;
  }
  const int t = (blockIdx.x - clear) * kMoveWarps + warp;
  if (t >= N) return;
  const typename B::T* src = x + t * ld;
  const int* r = pl.rows + (int64_t)t * pl.k;
  const int mine = lane < pl.k ? r[lane] : -1;
  for (int c = lane; c - lane < lanes; c += 32 * U) {
    B b[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c + 32 * u < lanes) b[u].load(src, c + 32 * u, H);
    for (int i = 0; i < pl.k; ++i) {
      const int to = i < 32 ? __shfl_sync(0xffffffffu, mine, i) : r[i];
      if ((unsigned)to >= (unsigned)pl.cap) continue;
      typename B::T* dst = out + (int64_t)to * H;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + 32 * u < lanes) b[u].store(dst, c + 32 * u, H);
    }
  }
}

// CTA t sums its pairs' rows: out[t] = residual[t] + sum_i w[t, i] y[rows[t, i]], in fp32 with one rounding.  A thread has
// the loads of eight pairs in flight; four such CTAs on an SM keep DRAM busy (16384 x 2048 bf16, top-8: 107 us with the
// residual, 0.96 of the copy rate; a persistent warp a token 6 to 12 % longer).
template <class B>
__global__ void __launch_bounds__(256, 4)
    combine_kernel(const typename B::T* __restrict__ y, int64_t ldy, const float* __restrict__ w,
                   const typename B::T* __restrict__ res, int64_t ldr, int H, Plan pl, typename B::T* __restrict__ out) {
  constexpr int U = 8;
  const int64_t t = blockIdx.x;
  const int lanes = B::lanes(H);
  for (int c = threadIdx.x; c < lanes; c += blockDim.x) {
    float acc[B::V] = {};
    B r;
    if (res) r.load_once(res + t * ldr, c, H);
    for (int i0 = 0; i0 < pl.k; i0 += U) {
      B b[U];
      float wi[U];
      bool here[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = i0 + u < pl.k ? pl.rows[t * pl.k + i0 + u] : -1;
        here[u] = (unsigned)at < (unsigned)pl.cap;
        if (here[u]) {
          b[u].load_once(y + at * ldy, c, H);
          wi[u] = w ? w[t * pl.k + i0 + u] : 1.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!here[u]) continue;
        float v[B::V];
        b[u].get(v);
#pragma unroll
        for (int q = 0; q < B::V; ++q) acc[q] = fmaf(wi[u], v[q], acc[q]);
      }
    }
    if (res) {
      float v[B::V];
      r.get(v);
#pragma unroll
      for (int q = 0; q < B::V; ++q) acc[q] += v[q];
    }
    B o;
    o.set(acc);
    o.store(out + t * H, c, H);
  }
}

// A warp takes pair j: dy[rows[j]] = w[j] g[j / k], dw[j] = <g[j / k], y[rows[j]]>; the grid's first `clear` CTAs zero
// dy's padding.  The eight warps of a CTA share their tokens' rows of g through L1, so y is read and dy written once:
// 16384 x 2048 bf16, top-8: 185 us for 1.21 GB, the copy rate (a CTA's loads without batches of four: 229).
template <class B>
__global__ void __launch_bounds__(kMoveWarps * 32)
    combine_bwd_kernel(const typename B::T* __restrict__ g, int64_t ldg, const typename B::T* __restrict__ y, int64_t ldy,
                       const float* __restrict__ w, int pairs, int clear, int H, Plan pl, typename B::T* __restrict__ dy,
                       float* __restrict__ dw) {
  constexpr int U = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, lanes = B::lanes(H);
  if ((int)blockIdx.x < clear) {
    clear_padding<B>(pl, dy, H, blockIdx.x * kMoveWarps + warp, (int64_t)clear * kMoveWarps);
    return;
  }
  const int64_t j = (int64_t)(blockIdx.x - clear) * kMoveWarps + warp;
  if (j >= pairs) return;
  const int at = pl.rows[j];
  if ((unsigned)at >= (unsigned)pl.cap) {
    if (dw && lane == 0) dw[j] = 0.f;
    return;
  }
  const typename B::T *gr = g + j / pl.k * ldg, *yr = y + at * ldy;
  const float wj = w[j];
  float dot = 0.f;
  for (int c = lane; c < lanes; c += 32 * U) {
    B b[U], a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u].zero();
      b[u].zero();
      if (c + 32 * u < lanes) {
        if (dw) a[u].load_once(yr, c + 32 * u, H);
        b[u].load(gr, c + 32 * u, H);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c + 32 * u >= lanes) break;
      float v[B::V], x[B::V];
      b[u].get(v);
      a[u].get(x);
#pragma unroll
      for (int q = 0; q < B::V; ++q) dot = fmaf(v[q], x[q], dot);
      if (dy) {
#pragma unroll
        for (int q = 0; q < B::V; ++q) v[q] *= wj;
        b[u].set(v);
        b[u].store(dy + (int64_t)at * H, c + 32 * u, H);
      }
    }
  }
  dot = warp_sum(dot);
  if (dw && lane == 0) dw[j] = dot;
}

// CTAs that clear: as many as the padding rows could keep busy, at most four on every SM.
static int clear_ctas(const Plan& pl) { return (int)std::max<int64_t>(1, std::min<int64_t>(pl.cap / kMoveWarps, 592)); }

static Plan plan_of(const torch::Tensor& rows_t, const torch::Tensor& offs, const torch::Tensor& counts, int64_t k,
                    int64_t align, int64_t cap, int64_t N, const torch::Tensor& like, const char* op) {
  const int64_t E = counts.numel();
  auto ints = [&](const torch::Tensor& t) {
    return t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous();
  };
  ROWS_CHECK(ints(rows_t) && ints(offs) && ints(counts) && offs.numel() == E + 1, "%s: not a plan on the rows' device",
             op);
  ROWS_CHECK(k >= 1 && rows_t.numel() == N * k, "%s: %lld tokens for a plan of %lld pairs, %lld a token", op,
             (long long)N, (long long)rows_t.numel(), (long long)k);
  ROWS_CHECK(cap >= 0 && cap < (1ll << 31) && align >= 1 && align < (1ll << 31), "%s: capacity or alignment", op);
  return {rows_t.data_ptr<int>(), offs.data_ptr<int>(), counts.data_ptr<int>(), (int)E, (int)k, (int)cap, align};
}

static void check_move(const torch::Tensor& x, const char* op, const char* what) {
  ROWS_CHECK(x.is_cuda() && x.dim() == 2 && row_type(x), "%s: %s must be 2-D, bf16 or fp32", op, what);
  ROWS_CHECK(x.size(0) < (1ll << 31) && x.size(1) < (1ll << 30), "%s: %s is too large", op, what);
}

// The plan's tensors and numbers, as the three entries hand them on.
struct PlanArgs {
  torch::Tensor rows, offs, counts;
  int64_t k, align;
  Plan of(int64_t cap, int64_t N, const torch::Tensor& like, const char* op) const {
    return plan_of(rows, offs, counts, k, align, cap, N, like, op);
  }
};

static torch::Tensor spread(torch::Tensor x, const PlanArgs& pa, int64_t cap) {
  check_move(x, "moe_dispatch", "x");
  const int64_t N = x.size(0), H = x.size(1);
  const Plan pl = pa.of(cap, N, x, "moe_dispatch");
  const c10::cuda::CUDAGuard guard(x.device());
  x = unit_inner(x);
  auto out = torch::empty({cap, H}, x.options());
  if (cap == 0 || H == 0) return out;
  const int clear = clear_ctas(pl);
  by_lanes(x, row_vectors(x) && row_vectors(out), [&](auto lanes) {
    using B = decltype(lanes);
    using T = typename B::T;
    launch_rows(dispatch_kernel<B>, clear + (N + kMoveWarps - 1) / kMoveWarps, kMoveWarps * 32, 0, 1, false,
                at::cuda::getCurrentCUDAStream(), (const T*)x.data_ptr(), x.stride(0), (int)N, (int)H, pl, clear,
                (T*)out.data_ptr());
  });
  return out;
}

static torch::Tensor sum_back(torch::Tensor y, const c10::optional<torch::Tensor>& w,
                              const c10::optional<torch::Tensor>& res, const PlanArgs& pa, int64_t N) {
  check_move(y, "moe_combine", "y");
  const int64_t cap = y.size(0), H = y.size(1);
  const Plan pl = pa.of(cap, N, y, "moe_combine");
  if (w.has_value())
    ROWS_CHECK(w->dim() == 2 && w->size(0) == N && w->size(1) == pa.k && vocab::vec_of(*w, y, at::kFloat, N * pa.k),
               "moe_combine: weights must be [%lld, %lld] on y's device", (long long)N, (long long)pa.k);
  const c10::cuda::CUDAGuard guard(y.device());
  y = unit_inner(y);
  torch::Tensor r;
  if (res.has_value()) {
    ROWS_CHECK(res->device() == y.device() && res->scalar_type() == y.scalar_type() && res->dim() == 2 &&
                   res->size(0) == N && res->size(1) == H,
               "moe_combine: the residual must be [%lld, %lld] of y's type and device", (long long)N, (long long)H);
    r = unit_inner(*res);
  }
  auto out = torch::empty({N, H}, y.options());
  if (N == 0 || H == 0) return out;
  by_lanes(y, row_vectors(y) && row_vectors(out) && (!r.defined() || row_vectors(r)), [&](auto lanes) {
    using B = decltype(lanes);
    using T = typename B::T;
    const int threads = std::min(256, (B::lanes((int)H) + 31) / 32 * 32);
    launch_rows(combine_kernel<B>, N, threads, 0, 1, false, at::cuda::getCurrentCUDAStream(), (const T*)y.data_ptr(),
                y.stride(0), w.has_value() ? (const float*)w->data_ptr<float>() : (const float*)nullptr,
                r.defined() ? (const T*)r.data_ptr() : (const T*)nullptr, r.defined() ? r.stride(0) : 0, (int)H, pl,
                (T*)out.data_ptr());
  });
  return out;
}

// -> {dy or nothing, dw or nothing}
static std::vector<torch::Tensor> combine_bwd(torch::Tensor g, torch::Tensor y, const torch::Tensor& w,
                                              const PlanArgs& pa, bool want_y, bool want_w) {
  const int64_t N = g.size(0), cap = y.size(0), H = y.size(1), pairs = N * pa.k;
  const Plan pl = pa.of(cap, N, y, "moe_combine");
  const c10::cuda::CUDAGuard guard(y.device());
  g = unit_inner(g);
  y = unit_inner(y);
  torch::Tensor dy, dw;
  if (want_y) dy = pairs == 0 ? torch::zeros({cap, H}, y.options()) : torch::empty({cap, H}, y.options());
  if (want_w) dw = H == 0 ? torch::zeros_like(w) : torch::empty_like(w);
  if (H == 0 || pairs == 0) return {dy, dw};
  const int clear = want_y ? clear_ctas(pl) : 0;
  by_lanes(y, row_vectors(y) && row_vectors(g) && (!want_y || row_vectors(dy)), [&](auto lanes) {
    using B = decltype(lanes);
    using T = typename B::T;
    launch_rows(combine_bwd_kernel<B>, clear + (pairs + kMoveWarps - 1) / kMoveWarps, kMoveWarps * 32, 0, 1, false,
                at::cuda::getCurrentCUDAStream(), (const T*)g.data_ptr(), g.stride(0), (const T*)y.data_ptr(),
                y.stride(0), (const float*)w.data_ptr<float>(), (int)pairs, clear, (int)H, pl,
                want_y ? (T*)dy.data_ptr() : (T*)nullptr, want_w ? dw.data_ptr<float>() : (float*)nullptr);
  });
  return {dy, dw};
}

struct Dispatch : public torch::autograd::Function<Dispatch> {
  using List = torch::autograd::variable_list;
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, torch::Tensor x, torch::Tensor rows_t,
                               torch::Tensor offs, torch::Tensor counts, int64_t k, int64_t align, int64_t cap) {
    ctx->save_for_backward({rows_t, offs, counts});
    ctx->saved_data["k"] = k;
    ctx->saved_data["N"] = x.size(0);
    return spread(x, {rows_t, offs, counts, k, align}, cap);
  }
  static List backward(torch::autograd::AutogradContext* ctx, List up) {
    LIBRA_CHECK(!at::GradMode::is_enabled(), "moe_dispatch: its gradient is not differentiable");
    const auto s = ctx->get_saved_variables();
    List out(7);
    out[0] = sum_back(up[0], c10::nullopt, c10::nullopt, {s[0], s[1], s[2], ctx->saved_data["k"].toInt(), 1},
                      ctx->saved_data["N"].toInt());
    return out;
  }
};

torch::Tensor moe_dispatch(torch::Tensor x, torch::Tensor rows_t, torch::Tensor offs, torch::Tensor counts, int64_t k,
                           int64_t align, int64_t cap) {
  if (at::GradMode::is_enabled() && x.requires_grad()) return Dispatch::apply(x, rows_t, offs, counts, k, align, cap);
  return spread(x, {rows_t, offs, counts, k, align}, cap);
}

struct Combine : public torch::autograd::Function<Combine> {
  using List = torch::autograd::variable_list;
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, torch::Tensor y, torch::Tensor w,
                               c10::optional<torch::Tensor> res, torch::Tensor rows_t, torch::Tensor offs,
                               torch::Tensor counts, int64_t k, int64_t align, int64_t N) {
    ctx->save_for_backward({y, w, rows_t, offs, counts});
    ctx->saved_data["k"] = k;
    ctx->saved_data["align"] = align;
    return sum_back(y, w, res, {rows_t, offs, counts, k, align}, N);
  }
  static List backward(torch::autograd::AutogradContext* ctx, List up) {
    LIBRA_CHECK(!at::GradMode::is_enabled(), "moe_combine: its gradient is not differentiable");
    const auto s = ctx->get_saved_variables();
    List out(9);
    const bool want_y = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1);
    if (want_y || want_w) {
      auto r = combine_bwd(up[0], s[0], s[1],
                           {s[2], s[3], s[4], ctx->saved_data["k"].toInt(), ctx->saved_data["align"].toInt()}, want_y,
                           want_w);
      out[0] = r[0];
      out[1] = r[1];
    }
    if (ctx->needs_input_grad(2)) out[2] = up[0];
    return out;
  }
};

torch::Tensor moe_combine(torch::Tensor y, torch::Tensor w, c10::optional<torch::Tensor> res, torch::Tensor rows_t,
                          torch::Tensor offs, torch::Tensor counts, int64_t k, int64_t align, int64_t cap, int64_t N) {
  ROWS_CHECK(y.dim() == 2 && y.size(0) == cap, "moe_combine: y must be [%lld, H], bf16 or fp32", (long long)cap);
  if (w.scalar_type() != at::kFloat) w = w.to(at::kFloat);
  if (!w.is_contiguous()) w = w.contiguous();
  if (at::GradMode::is_enabled() &&
      (y.requires_grad() || w.requires_grad() || (res.has_value() && res->requires_grad())))
    return Combine::apply(y, w, res, rows_t, offs, counts, k, align, N);
  return sum_back(y, w, res, {rows_t, offs, counts, k, align}, N);
}

}  // namespace experts
}  // namespace libra
