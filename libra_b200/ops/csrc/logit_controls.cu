// control_logits — penalties for repeated tokens, biases and grammar masks on
// rows of logits, ahead of the samplers of rollout.cu.  For token v of row b:
//
//   z1 = z > 0 ? z / r : z * r      if v occurs in the row's history
//   z2 = z1 - f * n - p * [n > 0]   n = occurrences of v behind the prompt
//   z3 = z2 + sum of v's biases
//   out = z3, or -inf where the grammar's bit of v is 0
//
// in fp32, rounded once to the output's type.
#include "vocab_rows.cuh"

namespace libra {
namespace vocab {

constexpr int kCtlThreads = 256;
constexpr int kCtlTile = 8192;  // tokens of one CTA
constexpr uint32_t kSeen = 0x80000000u;

struct CtlArgs {
  const int* hist;          // [H, hist_w]
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

template <typename TI, typename TO>
__global__ void __launch_bounds__(kCtlThreads) control_kernel(const TI* logits, int64_t ld, TO* out, int64_t out_ld,
                                                              int V, CtlArgs a) {
  extern __shared__ uint32_t ctl_smem[];
  uint32_t* cnt = ctl_smem;                                    // [kCtlTile]
  float* bias = reinterpret_cast<float*>(ctl_smem + kCtlTile);  // [kCtlTile]
  const int b = blockIdx.y;
  const int v0 = blockIdx.x * kCtlTile;
  const int n = min(kCtlTile, V - v0);
  const float rep = a.rep ? a.rep[b] : 1.f, pres = a.pres ? a.pres[b] : 0.f, freq = a.freq ? a.freq[b] : 0.f;
  bool bad = false;
  for (int i = threadIdx.x; i < kCtlTile; i += kCtlThreads) {
    cnt[i] = 0u;
    bias[i] = 0.f;
  }
  __syncthreads();
  if (a.hist && (rep != 1.f || pres != 0.f || freq != 0.f)) {
    const int hr = a.hist_rows ? a.hist_rows[b] : b;
    int len = a.hist_lens[b];
    if (hr < 0 || hr >= a.hist_rows_n || len < 0 || len > a.hist_w) bad = true;
    if (hr < 0 || hr >= a.hist_rows_n) len = 0;
    len = min(len, a.hist_w);
    const int prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
    const int* h = a.hist + (int64_t)max(hr, 0) * a.hist_ld;
    for (int i = threadIdx.x; i < len; i += kCtlThreads) {
      const unsigned t = (unsigned)(h[i] - v0);
      if (h[i] >= 0 && t < (unsigned)n) {
        if (i < prompt)
          atomicOr(&cnt[t], kSeen);
        else
          atomicAdd(&cnt[t], 1u);
      }
    }
  }
  if (a.bias_offs) {
    int lo = a.bias_offs[b], hi = a.bias_offs[b + 1];
    if (lo < 0 || hi < lo || hi > a.bias_n) {
      bad = true;
      lo = hi = 0;
    }
    // a token's entries are summed in list order by the thread of its first entry
    for (int e = lo + threadIdx.x; e < hi; e += kCtlThreads) {
      const int id = a.bias_ids[e];
      if (id < v0 || id >= v0 + n) continue;
      bool first = true;
      for (int j = lo; j < e && first; ++j) first = a.bias_ids[j] != id;
      if (!first) continue;
      float s = 0.f;
      for (int j = e; j < hi; ++j)
        if (a.bias_ids[j] == id) s += a.bias_vals[j];
      bias[id - v0] = s;
    }
  }
  const int* mask = nullptr;
  if (a.mask) {
    const int mr = a.mask_rows ? a.mask_rows[b] : b;
    if (mr >= a.mask_n) bad = true;
    if (mr >= 0 && mr < a.mask_n) mask = a.mask + (int64_t)mr * a.mask_ld;
  }
  if (bad && a.err && threadIdx.x == 0) atomicCAS(a.err, 0, kBadArgument);
  __syncthreads();
  const TI* z = logits + (int64_t)b * ld + v0;
  TO* o = out + (int64_t)b * out_ld + v0;
  for (int i = threadIdx.x; i < n; i += kCtlThreads) {
    float x = to_f(z[i]);
    const uint32_t c = cnt[i];
    if (c) {
      x = x > 0.f ? x / rep : x * rep;
      const uint32_t k = c & ~kSeen;
      if (k) x = x - freq * (float)k - pres;
    }
    x += bias[i];
    if (mask && !((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1)) x = -INFINITY;
    from_f(o + i, x);
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
    a.mask = mask->data_ptr<int>();
    a.mask_ld = mask->stride(0);
    a.mask_n = (int)mask->size(0);
    a.mask_rows = (const int*)opt(mask_rows, at::kInt, B, "mask_rows");
  }
  LIBRA_CHECK(err.device() == logits.device() && err.scalar_type() == at::kInt, "control_logits: error word");
  LIBRA_CHECK(B < 65536, "control_logits: at most 65535 rows");
  if (B == 0 || V == 0) return;
  a.err = err.data_ptr<int>();
  const c10::cuda::CUDAGuard guard(logits.device());
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  const dim3 grid((V + kCtlTile - 1) / kCtlTile, B);
  const size_t smem = kCtlTile * 8;
  auto go = [&](auto kern, auto* in, auto* o) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    LIBRA_CHECK(e == cudaSuccess, "control_logits: %s", cudaGetErrorString(e));
    kern<<<grid, kCtlThreads, smem, st>>>(in, logits.stride(0), o, out.stride(0), V, a);
    LIBRA_LAUNCH_CHECK();
  };
  using bf = __nv_bfloat16;
  const bool fi = logits.scalar_type() == at::kFloat, fo = out.scalar_type() == at::kFloat;
  void *pi = logits.data_ptr(), *po = out.data_ptr();
  if (fi && fo) go(control_kernel<float, float>, (const float*)pi, (float*)po);
  if (fi && !fo) go(control_kernel<float, bf>, (const float*)pi, (bf*)po);
  if (!fi && fo) go(control_kernel<bf, float>, (const bf*)pi, (float*)po);
  if (!fi && !fo) go(control_kernel<bf, bf>, (const bf*)pi, (bf*)po);
}

}  // namespace vocab
}  // namespace libra
