// control_logits — penalties for repeated tokens, biases and grammar masks on
// rows of logits, ahead of the samplers of rollout.cu.  For token v of row b:
//
//   z1 = z > 0 ? z / r : z * r      if v occurs in the row's history
//   z2 = z1 - f * n - p * [n > 0]   n = occurrences of v behind the prompt
//   z3 = z2 + sum of v's biases
//   out = z3, or -inf where the grammar's bit of v is 0
//
// in fp32, rounded once to the output's type.
//
// A CTA owns a tile of a row's tokens and keeps their occurrences in shared
// memory: it scans the row's whole history (from L2, where the row's other
// tiles find it too) and counts what falls into its tile, then streams the
// tile once.  An octet without occurrences, biases or masked tokens is only
// converted.  Tokens with biases are left out of the stream and written
// afterwards from their own logit, so the call can work in place and still
// round once.
#include <algorithm>
#include <type_traits>

#include "vocab_rows.cuh"

namespace libra {
namespace vocab {

constexpr int kCtlThreads = 512;

struct CtlArgs {
  bool has_hist, has_mask;  // (a table without rows has no address)
  const int* hist;          // [H, hist_w] or null
  int64_t hist_ld;
  int hist_rows_n, hist_w;
  const int* hist_rows;     // [B] or null: row b
  const int* hist_lens;     // [B]
  const int* prompt_lens;   // [B] or null: 0
  const float *rep, *pres, *freq;  // [B] or null
  const int* bias_offs;     // [B + 1] or null
  const int* bias_ids;
  const float* bias_vals;
  int bias_n;
  const int* mask;          // [M, mask_w] or null
  int64_t mask_ld;
  int mask_n;
  const int* mask_rows;     // [B] or null: row b
  int* err;
};

// Counters of a tile's tokens: occurrences behind the prompt, and a bit for tokens of the prompt.  16 bits a token while
// the history cannot overflow them (64 KB for 32768 tokens: three CTAs on an SM), else 32.
template <int kBits>
struct Counts {
  static constexpr uint32_t kSeen = 1u << (kBits - 1), kCount = kSeen - 1;
  static constexpr int kPer = 32 / kBits;
  uint32_t* w;
  __device__ __forceinline__ int shift(int i) const { return kBits == 32 ? 0 : (i & 1) * 16; }
  __device__ __forceinline__ uint32_t& word(int i) const { return w[i / kPer]; }
  __device__ __forceinline__ void add(int i) const { atomicAdd(&word(i), 1u << shift(i)); }
  __device__ __forceinline__ void see(int i) const { atomicOr(&word(i), kSeen << shift(i)); }
  __device__ __forceinline__ uint32_t get(int i) const {
    return kBits == 32 ? word(i) : (word(i) >> shift(i)) & 0xffffu;
  }
  // of an octet that starts at a multiple of 8; false if all are zero
  __device__ __forceinline__ bool octet(int i, uint32_t (&c)[8]) const {
    uint4 a = *reinterpret_cast<const uint4*>(&word(i));
    if (kBits == 32) {
      const uint4 b = *reinterpret_cast<const uint4*>(&word(i + 4));
      c[0] = a.x; c[1] = a.y; c[2] = a.z; c[3] = a.w;
      c[4] = b.x; c[5] = b.y; c[6] = b.z; c[7] = b.w;
      return (a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) != 0u;
    }
    const uint32_t v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = (v[e >> 1] >> (16 * (e & 1))) & 0xffffu;
    return (a.x | a.y | a.z | a.w) != 0u;
  }
};

struct Penalty {
  float rep, inv, pres, freq;  // inv = 1 / rep
};

// Without branches: some lane of a warp has an occurrence in almost every octet of the frequent tokens.  A product with
// 1 / r instead of the quotient adds one rounding (2^-24), and takes a fifth of a division's instructions.
template <int kBits>
__device__ __forceinline__ float penalize(float x, uint32_t c, const Penalty& p) {
  const uint32_t k = c & Counts<kBits>::kCount;
  // 2^23 + k is a float whose low bits are k
  const float n = kBits == 16 ? __uint_as_float(0x4b000000u | k) - 8388608.f : (float)k;
  const float s = x > 0.f ? p.inv : p.rep;
  x *= c ? s : 1.f;
  const float less = fmaf(p.freq, n, p.pres);
  return x - (k ? less : 0.f);
}

// Bits of tokens j .. j + 7.
__device__ __forceinline__ uint32_t mask_bits(const int* mask, int j, int V) {
  const int w = j >> 5;
  const uint32_t lo = (uint32_t)__ldg(mask + w);
  const int s = j & 31;
  if (s <= 24) return (lo >> s) & 0xffu;
  const uint32_t hi = (w + 1) * 32 < V ? (uint32_t)__ldg(mask + w + 1) : 0u;
  return __funnelshift_r(lo, hi, s) & 0xffu;
}

template <typename TI, typename TO, int kBits>
__global__ void __launch_bounds__(kCtlThreads, 3) control_kernel(const TI* logits, int64_t ld, TO* out, int64_t out_ld,
                                                              int V, int tiles, int tile_octs, CtlArgs a) {
  using C = Counts<kBits>;
  extern __shared__ __align__(16) uint32_t ctl_smem[];
  __shared__ int twice;
  const C cnt{ctl_smem};
  uint32_t* biases = ctl_smem + (8 * tile_octs + 32) / C::kPer;  // a bit a token
  const int b = blockIdx.x / tiles, tile = blockIdx.x % tiles, t = threadIdx.x;
  const TI* z = logits + (int64_t)b * ld;
  TO* dst = out + (int64_t)b * out_ld;
  const RowSpan sp = row_span(z, V);
  const int o0 = tile * tile_octs, o1 = min(sp.octs, o0 + tile_octs);
  const bool first = tile == 0, last = tile == tiles - 1;
  // tokens [lo, hi) of the row; token j has counter j - base, and octets start at multiples of 8 of it
  const int base = sp.head + 8 * o0 - 8;
  const int lo = first ? 0 : sp.head + 8 * o0, hi = last ? V : sp.head + 8 * o1;
  const float rep = a.rep ? a.rep[b] : 1.f;
  const Penalty pen = {rep, 1.f / rep, a.pres ? a.pres[b] : 0.f, a.freq ? a.freq[b] : 0.f};
  bool bad = false;
  int len = 0, prompt = 0;
  const int* h = nullptr;
  if (a.has_hist && (rep != 1.f || pen.pres != 0.f || pen.freq != 0.f)) {
    const int hr = a.hist_rows ? a.hist_rows[b] : b;
    len = a.hist_lens[b];
    const bool in = hr >= 0 && hr < a.hist_rows_n;
    bad = !in || len < 0 || len > a.hist_w;
    len = in ? min(len, a.hist_w) : 0;
    prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
    h = a.hist + (int64_t)(in ? hr : 0) * a.hist_ld;
  }
  int b0 = 0, b1 = 0;
  if (a.bias_offs) {
    b0 = a.bias_offs[b];
    b1 = a.bias_offs[b + 1];
    if (b0 < 0 || b1 < b0 || b1 > a.bias_n) {
      bad = true;
      b0 = b1 = 0;
    }
  }
  const int* mask = nullptr;
  if (a.has_mask) {
    const int mr = a.mask_rows ? a.mask_rows[b] : b;
    bad = bad || mr >= a.mask_n;
    if (mr >= 0 && mr < a.mask_n) mask = a.mask + (int64_t)mr * a.mask_ld;
  }
  if (bad && t == 0) atomicCAS(a.err, 0, kBadArgument);
  const bool counted = len > 0, biased = b1 > b0;
  if (counted || biased) {
    const int quads = counted ? (hi - base + C::kPer * 4 - 1) / (C::kPer * 4) : 0;
    for (int i = t; i < quads; i += kCtlThreads) reinterpret_cast<uint4*>(ctl_smem)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = t; i < (hi - base + 31) / 32 && biased; i += kCtlThreads) biases[i] = 0u;
    if (t == 0) twice = 0;
    __syncthreads();
    const auto count = [&](int i, int id) {
      if (id >= lo && id < hi) {
        if (i < prompt)
          cnt.see(id - base);
        else
          cnt.add(id - base);
      }
    };
    const int quads_in = aligned16(h) ? len / 4 : 0;  // four tokens a load
#pragma unroll 4
    for (int i = t; i < quads_in; i += kCtlThreads) {
      const int4 q = __ldg(reinterpret_cast<const int4*>(h) + i);
      count(4 * i, q.x);
      count(4 * i + 1, q.y);
      count(4 * i + 2, q.z);
      count(4 * i + 3, q.w);
    }
#pragma unroll 4
    for (int i = 4 * quads_in + t; i < len; i += kCtlThreads) count(i, h[i]);
    for (int e = b0 + t; e < b1; e += kCtlThreads) {
      const int id = a.bias_ids[e];
      if (id < lo || id >= hi) continue;
      const int i = id - base;
      if ((atomicOr(&biases[i >> 5], 1u << (i & 31)) >> (i & 31)) & 1u) twice = 1;
    }
    __syncthreads();
  } else if (!mask && (const void*)z == (const void*)dst) {
    return;  // in place, and nothing to do
  }
  // head and tail of the row: a token a thread
  if ((first && t < sp.head) || (last && t >= 32 && t - 32 < sp.tail)) {
    const int j = t < 32 ? t : sp.head + 8 * sp.octs + t - 32;
    const uint32_t c = counted ? cnt.get(j - base) : 0u;
    float x = penalize<kBits>(to_f(z[j]), c, pen);
    if (mask && !((mask[j >> 5] >> (j & 31)) & 1)) x = -INFINITY;
    if (!biased || !((biases[(j - base) >> 5] >> ((j - base) & 31)) & 1)) from_f(dst + j, x);
  }
  const uint8_t* bias_bytes = reinterpret_cast<const uint8_t*>(biases) + 1;
  const TI* body = z + sp.head;
  TO* obody = dst + sp.head;
  const bool vec = aligned16(obody);
  constexpr int kU = sizeof(TI) == 2 ? 4 : 2;
  for (int o = o0 + t; o < o1; o += kU * kCtlThreads) {
    Oct<TI> v[kU];
    uint32_t allow[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int p = o + u * kCtlThreads;
      allow[u] = 0xffu;
      if (p < o1) {
        if (mask) allow[u] = mask_bits(mask, sp.head + 8 * p, V);
        if (allow[u]) v[u].load_once(body + 8 * (int64_t)p);
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int p = o + u * kCtlThreads;
      if (p >= o1) continue;
      float f[8];
      v[u].get(f);
      uint32_t c[8];
      if (counted && cnt.octet(8 * (p - o0) + 8, c)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = penalize<kBits>(f[e], c[e], pen);
      }
      const uint32_t skip = biased ? bias_bytes[p - o0] : 0u;
      if (allow[u] != 0xffu) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!((allow[u] >> e) & 1u)) f[e] = -INFINITY;
      }
      TO* at = obody + 8 * (int64_t)p;
      if (vec && !skip) {
        store_oct(at, f);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!((skip >> e) & 1u)) from_f(at + e, f[e]);
      }
    }
  }
  // biased tokens, from their own logits; one listed twice is written by its first entry, the sum in list order
  for (int e = b0 + t; e < b1; e += kCtlThreads) {
    const int id = a.bias_ids[e];
    if (id < lo || id >= hi) continue;
    float s = a.bias_vals[e];
    if (twice) {
      bool again = false;
      for (int i = b0; i < e && !again; ++i) again = a.bias_ids[i] == id;
      if (again) continue;
      for (int i = e + 1; i < b1; ++i)
        if (a.bias_ids[i] == id) s += a.bias_vals[i];
    }
    float x = penalize<kBits>(to_f(z[id]), counted ? cnt.get(id - base) : 0u, pen) + s;
    if (mask && !((mask[id >> 5] >> (id & 31)) & 1)) x = -INFINITY;
    from_f(dst + id, x);
  }
}

// logits [B, V] bf16 / fp32; history [H, L] int32 with lengths [B] int32 (and optional row numbers and prompt
// lengths [B] int32); repetition / presence / frequency fp32 [B]; biases as int32 offsets [B + 1], int32 ids,
// fp32 values; mask int32 [M, >= ceil(V / 32)] with optional row numbers [B] int32 (negative: no mask);
// out [B, V] fp32 / bf16, which may be the logits themselves.  Row numbers, lengths and offsets outside their
// tables are not followed; they set the error word.
void control_logits(torch::Tensor logits, c10::optional<torch::Tensor> history,
                    c10::optional<torch::Tensor> history_rows, c10::optional<torch::Tensor> history_lens,
                    c10::optional<torch::Tensor> prompt_lens, c10::optional<torch::Tensor> repetition,
                    c10::optional<torch::Tensor> presence, c10::optional<torch::Tensor> frequency,
                    c10::optional<torch::Tensor> bias_offsets, c10::optional<torch::Tensor> bias_ids,
                    c10::optional<torch::Tensor> bias_values, c10::optional<torch::Tensor> mask,
                    c10::optional<torch::Tensor> mask_rows, torch::Tensor out, torch::Tensor err) {
  check_rows(logits, "control_logits");
  const int B = (int)logits.size(0), V = (int)logits.size(1);
  LIBRA_CHECK(out.device() == logits.device() && out.dim() == 2 && out.size(0) == B && out.size(1) == V &&
                  (out.scalar_type() == at::kBFloat16 || out.scalar_type() == at::kFloat) &&
                  (V <= 1 || out.stride(1) == 1) && (B <= 1 || out.stride(0) >= V),
              "control_logits: out must be bf16 or fp32 [B, V] on the logits' device, unit inner stride");
  check_apart(logits, out, "control_logits");
  auto opt = [&](const c10::optional<torch::Tensor>& t, at::ScalarType ty, int64_t n, const char* name) -> const void* {
    if (!t.has_value()) return nullptr;
    LIBRA_CHECK(vec_of(*t, logits, ty, n), "control_logits: %s must be a contiguous [%lld] tensor of its type on the "
                "logits' device", name, (long long)n);
    return t->data_ptr();
  };
  CtlArgs a = {};
  if (history.has_value()) {
    LIBRA_CHECK(history->device() == logits.device() && history->dim() == 2 && history->scalar_type() == at::kInt &&
                    (history->size(1) <= 1 || history->stride(1) == 1) && history->size(0) < (1ll << 31) &&
                    history->size(1) < (1ll << 31),
                "control_logits: history must be int32 [H, L] on the logits' device, unit inner stride");
    LIBRA_CHECK(history_lens.has_value(), "control_logits: history needs history_lens");
    LIBRA_CHECK(history_rows.has_value() || history->size(0) >= B, "control_logits: history has fewer rows than logits");
    a.has_hist = true;
    a.hist = history->data_ptr<int>();
    a.hist_ld = history->stride(0);
    a.hist_rows_n = (int)history->size(0);
    a.hist_w = (int)history->size(1);
    a.hist_rows = (const int*)opt(history_rows, at::kInt, B, "history_rows");
    a.hist_lens = (const int*)opt(history_lens, at::kInt, B, "history_lens");
    a.prompt_lens = (const int*)opt(prompt_lens, at::kInt, B, "prompt_lens");
  }
  a.rep = (const float*)opt(repetition, at::kFloat, B, "repetition");
  a.pres = (const float*)opt(presence, at::kFloat, B, "presence");
  a.freq = (const float*)opt(frequency, at::kFloat, B, "frequency");
  if (bias_offsets.has_value()) {
    LIBRA_CHECK(bias_ids.has_value() && bias_values.has_value() && bias_ids->numel() == bias_values->numel() &&
                    bias_ids->numel() < (1ll << 31),
                "control_logits: biases need offsets, ids and as many values");
    a.bias_offs = (const int*)opt(bias_offsets, at::kInt, B + 1, "bias_offsets");
    a.bias_n = (int)bias_ids->numel();
    a.bias_ids = (const int*)opt(bias_ids, at::kInt, a.bias_n, "bias_ids");
    a.bias_vals = (const float*)opt(bias_values, at::kFloat, a.bias_n, "bias_values");
  }
  if (mask.has_value()) {
    LIBRA_CHECK(mask->device() == logits.device() && mask->dim() == 2 && mask->scalar_type() == at::kInt &&
                    (mask->size(1) <= 1 || mask->stride(1) == 1) && mask->size(1) >= (V + 31) / 32 &&
                    mask->size(0) < (1ll << 31),
                "control_logits: mask must be int32 [M, ceil(V / 32)] on the logits' device, unit inner stride");
    LIBRA_CHECK(mask_rows.has_value() || mask->size(0) >= B, "control_logits: mask has fewer rows than logits");
    a.has_mask = true;
    a.mask = mask->data_ptr<int>();
    a.mask_ld = mask->stride(0);
    a.mask_n = (int)mask->size(0);
    a.mask_rows = (const int*)opt(mask_rows, at::kInt, B, "mask_rows");
  }
  LIBRA_CHECK(err.device() == logits.device() && err.scalar_type() == at::kInt, "control_logits: error word");
  if (B == 0 || V == 0) return;
  a.err = err.data_ptr<int>();
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  // Tiles of 32768 tokens, since every tile scans the history once (256 x 151936 fp32 with 16384 tokens of history:
  // 75 us, 0.65 of the floor; with the history read one token a load 81 us, and 84 us with tiles of 16384), smaller
  // ones while that leaves SMs without three CTAs.
  int tile = 32768;
  while (tile > 2048 && (int64_t)B * ((V + tile - 1) / tile) < 3 * 148) tile /= 2;
  const int tiles = std::max(1, (V / 8 + tile / 8 - 1) / (tile / 8));
  // 16-bit counters hold 2^15 - 1 occurrences (256 rows bf16, histories up to 4096 in a 65520-wide table: 96 us with
  // 32-bit ones, one CTA an SM; 65.5 us with 16-bit ones for the same rows as a 4096-wide table)
  const bool wide = a.has_hist && a.hist_w >= (1 << 15);
  const size_t smem = (size_t)(tile + 32) * (wide ? 4 : 2) + (tile + 32) / 8;
  auto go = [&](auto* in, auto* o) {
    using I = std::remove_const_t<std::remove_pointer_t<decltype(in)>>;
    using O = std::remove_pointer_t<decltype(o)>;
    if (wide)
      launch_rows(control_kernel<I, O, 32>, (int64_t)B * tiles, kCtlThreads, smem, 1, false, st, in, logits.stride(0),
                  o, out.stride(0), V, tiles, tile / 8, a);
    else
      launch_rows(control_kernel<I, O, 16>, (int64_t)B * tiles, kCtlThreads, smem, 1, false, st, in, logits.stride(0),
                  o, out.stride(0), V, tiles, tile / 8, a);
  };
  using bf = __nv_bfloat16;
  const bool fi = logits.scalar_type() == at::kFloat, fo = out.scalar_type() == at::kFloat;
  void *pi = logits.data_ptr(), *po = out.data_ptr();
  if (fi && fo) go((const float*)pi, (float*)po);
  if (fi && !fo) go((const float*)pi, (bf*)po);
  if (!fi && fo) go((const bf*)pi, (float*)po);
  if (!fi && !fo) go((const bf*)pi, (bf*)po);
}

}  // namespace vocab
}  // namespace libra
