"""Operators on rows of vocabulary logits: what a sampler needs before it
(penalties, biases, grammar masks), what it reports beside the token (top
logprobs), and the distillation loss that trains on such a report.

They dispatch like the other operators of :mod:`libra_b200.ops`: CUDA tensors
run the kernels of ``logit_controls.cu``, ``top_logprobs.cu`` and
``distill.cu``; CPU tensors run :mod:`libra_b200.ops.reference`.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import reference as ref

MAX_TOP = 256  # slots of a teacher's table, and the largest k of top_logprobs

DIVERGENCES = {"forward": 0, "reverse": 1, "js": 2}
TAILS = ("bucket", "drop")


def _written(out: torch.Tensor) -> None:
    """A kernel wrote to a caller's tensor: autograd then refuses a backward pass that saved its old values."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def _rows(logits: torch.Tensor, op: str) -> torch.Tensor:
    if logits.dim() != 2:
        raise ValueError(f"{op}: logits must be [rows, vocabulary], got {tuple(logits.shape)}")
    if logits.is_cuda and logits.stride(1) != 1 and logits.shape[1] > 1:
        return logits.contiguous()
    return logits


def control_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                   history_lens: Optional[torch.Tensor] = None, prompt_lens: Optional[torch.Tensor] = None,
                   history_rows: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                   presence: Optional[torch.Tensor] = None, frequency: Optional[torch.Tensor] = None,
                   bias_offsets: Optional[torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                   mask_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties, biases and grammar masks on logits [B, V] (bf16 or fp32).

    * ``history`` int32 [H, L] holds token lists; batch row b reads row
      ``history_rows[b]`` (int32; row b without it), its first
      ``history_lens[b]`` tokens, of which the first ``prompt_lens[b]`` (0
      without it) are the prompt.  Tokens outside the vocabulary are ignored.
    * ``repetition`` fp32 [B] (> 0): a positive logit of a token in the history
      is divided by it, any other multiplied.  ``frequency`` fp32 [B] is
      subtracted once per occurrence behind the prompt and ``presence`` fp32
      [B] once if there is one.
    * row b's biases are the entries ``bias_offsets[b]`` to
      ``bias_offsets[b + 1]`` (int32 [B + 1]) of ``bias_ids`` int32 /
      ``bias_values`` fp32; a token listed twice gets the sum.  Made for
      hundreds of entries a row; a ban of most tokens is a mask.
    * ``mask`` int32 [M, >= ceil(V / 32)]: bit v % 32 of word v // 32 allows
      token v.  Batch row b reads row ``mask_rows[b]`` (int32; row b without
      it); a negative row number leaves the row unmasked.  Other tokens become
      -inf, whatever their logit was; a row may end up with nothing else.

    They apply in this order, in fp32, with one rounding to ``out`` (fp32
    unless given; it may be ``logits`` itself), and are not differentiated
    through.  Row numbers, lengths and offsets that point outside their tables
    are not followed: they set the error word that ``check_kernel_errors``
    raises (ValueError on the CPU).  A row whose penalties change nothing
    (1, 0 and 0) needs no history: its row number and length are not looked at.
    """
    logits = _rows(logits, "control_logits")
    if history is None and (history_lens is not None or history_rows is not None or prompt_lens is not None):
        raise ValueError("control_logits: history lengths or rows without a history")
    if mask is None and mask_rows is not None:
        raise ValueError("control_logits: mask rows without a mask")
    if (bias_offsets is None) != (bias_ids is None) or (bias_offsets is None) != (bias_values is None):
        raise ValueError("control_logits: biases need offsets, ids and values")
    if history is not None and history_lens is None:
        raise ValueError("control_logits: history needs history_lens")
    if logits.device.type != "cuda":
        with torch.no_grad():
            res = ref.control_logits(logits, history, history_lens, prompt_lens, history_rows, repetition, presence,
                                     frequency, bias_offsets, bias_ids, bias_values, mask, mask_rows)
            return res if out is None else out.copy_(res)
    from . import error_flag, ext

    if out is None:
        out = torch.empty(logits.shape, dtype=torch.float32, device=logits.device)
    else:
        _written(out)
    ext().control_logits(logits, history, history_rows, history_lens, prompt_lens, repetition, presence, frequency,
                         bias_offsets, bias_ids, bias_values, mask, mask_rows, out, error_flag(logits.device))
    return out


def top_logprobs(logits: torch.Tensor, k: int, temperature: Union[float, torch.Tensor] = 1.0
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``k`` (1 to 256) largest logits of every row [N, V], in descending
    order with ties at the lowest index first: token ids int64 [N, k], their
    logprobs under softmax(logits / temperature) fp32 [N, k] and the row's
    log-sum-exp fp32 [N].  ``temperature``: a number or fp32 [N]; what is not
    above 0 counts as 1.  A row of nothing but -inf has logprobs and
    log-sum-exp of -inf; NaN ranks above +inf and makes the row's logprobs NaN.
    Not differentiated through."""
    logits = _rows(logits, "top_logprobs")
    k = int(k)
    if not 1 <= k <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f"top_logprobs: k must lie in [1, {min(MAX_TOP, logits.shape[1])}], got {k}")
    per_row = isinstance(temperature, torch.Tensor)
    if logits.device.type != "cuda":
        with torch.no_grad():
            return ref.top_logprobs(logits, k, temperature)
    from . import ext

    return tuple(ext().top_logprobs(logits.detach(), k, temperature if per_row else None,
                                    1.0 if per_row else float(temperature)))


def _check_distill(op: str, logits, ids, lps, divergence, beta, tail, temperature) -> float:
    """Checks the arguments; returns the beta to use (a fixed one where the divergence has none)."""
    if divergence not in DIVERGENCES:
        raise ValueError(f"{op}: divergence must be one of {sorted(DIVERGENCES)}, got {divergence!r}")
    if tail not in TAILS:
        raise ValueError(f"{op}: tail must be one of {TAILS}, got {tail!r}")
    if tail == "drop" and divergence == "reverse":
        raise ValueError(f"{op}: the reverse divergence needs the rest bucket (it is infinite without one)")
    if divergence == "js" and not 0.0 < beta < 1.0:
        raise ValueError(f"{op}: beta must lie between 0 and 1, got {beta}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{op}: temperature must lie in [1e-6, 1e6], got {temperature}")
    if ids.dim() != 2 or ids.shape != lps.shape or ids.shape[0] != logits.shape[0]:
        raise ValueError(f"{op}: teacher_ids and teacher_logprobs must be [rows, K], got {tuple(ids.shape)} and "
                         f"{tuple(lps.shape)} for {logits.shape[0]} rows")
    if not 1 <= ids.shape[1] <= MAX_TOP:
        raise ValueError(f"{op}: 1 to {MAX_TOP} teacher tokens a row, got {ids.shape[1]}")
    return float(beta) if divergence == "js" else 0.5


def distill_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                 divergence: str = "forward", beta: float = 0.5, tail: str = "bucket", temperature: float = 1.0,
                 targets: Optional[torch.Tensor] = None):
    """Divergence of student rows [N, V] (bf16 or fp32) from a teacher's top
    logprobs, fp32 [N], differentiable with respect to the logits.

    ``teacher_ids`` int64 / ``teacher_logprobs`` fp32 [N, K] (``top_logprobs``
    of the teacher; K up to 256).  A slot whose id lies outside the vocabulary
    or whose logprob is -inf or NaN is empty, and so is a token's second slot;
    a row of empty slots has loss 0 and gradient 0, and so has a row of
    nothing but -inf logits.  ``divergence``: "forward" KL(teacher | student),
    "reverse" KL(student | teacher), or "js", beta KL(teacher | m) + (1 - beta)
    KL(student | m) with m = beta teacher + (1 - beta) student.  ``tail``:
    "bucket" compares the listed tokens and one bucket for all others (the
    teacher's mass there is at least 2^-24); "drop" divides the teacher's
    probabilities by their sum.  The student is softmax(logits / temperature).

    With ``targets`` int64 [N] the result is (loss, logprob of the targets),
    both from the same pass and both differentiable; targets outside the
    vocabulary have logprob -inf and no gradient, and set the error word that
    ``check_kernel_errors`` raises (ValueError on the CPU)."""
    logits = _rows(logits, "distill_loss")
    beta = _check_distill("distill_loss", logits, teacher_ids, teacher_logprobs, divergence, beta, tail, temperature)
    if logits.device.type != "cuda":
        loss, logp = ref.distill_loss(logits, teacher_ids, teacher_logprobs, divergence, beta, tail, temperature,
                                      targets)
    else:
        from . import error_flag, ext

        loss, logp = ext().distill_loss(logits, teacher_ids.contiguous(), teacher_logprobs.contiguous(),
                                        DIVERGENCES[divergence], beta, tail == "drop", float(temperature),
                                        None if targets is None else targets.contiguous(),
                                        error_flag(logits.device))
    return loss if targets is None else (loss, logp)


@torch.no_grad()
def distill_loss_grad(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                      divergence: str = "forward", beta: float = 0.5, tail: str = "bucket", temperature: float = 1.0,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``distill_loss`` and its gradient with respect to every row's logits for
    an upstream gradient of one: (loss fp32 [N], gradient [N, V] of the
    logits' type).  ``out``: where the gradient goes; it may be ``logits``."""
    logits = _rows(logits, "distill_loss_grad")
    beta = _check_distill("distill_loss_grad", logits, teacher_ids, teacher_logprobs, divergence, beta, tail,
                          temperature)
    if logits.device.type != "cuda":
        with torch.enable_grad():
            z = logits.detach().clone().requires_grad_(True)
            loss, _ = ref.distill_loss(z, teacher_ids, teacher_logprobs, divergence, beta, tail, temperature, None)
            (grad,) = torch.autograd.grad(loss.sum(), z)
        return loss.detach(), grad if out is None else out.copy_(grad)
    from . import error_flag, ext

    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    else:
        _written(out)
    loss = ext().distill_onepass(logits, teacher_ids.contiguous(), teacher_logprobs.contiguous(),
                                 DIVERGENCES[divergence], beta, tail == "drop", float(temperature), out,
                                 error_flag(logits.device))
    return loss, out


class _LMHeadDistill(torch.autograd.Function):
    """distill_loss of h W^T / T, chunk by chunk, without an fp32 logits tensor.

    Without targets every chunk's bf16 logits are rewritten by their unit
    gradients as soon as they are scored (one pass over them), and the upstream
    gradients of the rows scale the [R, H] operands of the two products instead
    of the [R, V] gradients.  With targets the two upstream gradients mix per
    token, so the logits are kept and rewritten in the backward pass."""

    @staticmethod
    def forward(ctx, h, w, ids, lps, kind, targets):
        from . import LOGPROB_CHUNK_ROWS, error_flag, ext, gemm

        C, err = ext(), error_flag(h.device)
        div, beta, drop, temperature = kind
        R = h.shape[0]
        loss = torch.empty(R, dtype=torch.float32, device=h.device)
        logp = None if targets is None else torch.empty(R, dtype=torch.float32, device=h.device)
        need = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        ctx.kept, ctx.rows = [], LOGPROB_CHUNK_ROWS
        for s in range(0, R, ctx.rows):
            e = min(R, s + ctx.rows)
            logits = gemm(h[s:e], w)
            saved = None
            if need and targets is None:
                loss[s:e] = C.distill_onepass(logits, ids[s:e], lps[s:e], div, beta, drop, temperature, logits, err)
            else:
                loss[s:e], lp, saved = C.distill_fwd(logits, ids[s:e], lps[s:e], div, beta, drop, temperature,
                                                     None if targets is None else targets[s:e], err)
                if logp is not None:
                    logp[s:e] = lp
            if need:
                ctx.kept.append((logits, saved))
        ctx.save_for_backward(h, w, targets)
        ctx.temperature, ctx.slots = temperature, ids.shape[1]
        ctx.set_materialize_grads(False)
        return loss, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_lp):
        from . import EPI_ACC_F32, EPI_F32, ext, gemm

        h, w, targets = ctx.saved_tensors
        if g is None and g_lp is None:
            return (None,) * 6
        R = h.shape[0]
        if R and not ctx.kept:
            raise RuntimeError("lm_head_distill: its backward pass runs once (the logits are gone)")
        g = torch.zeros(R, device=h.device) if g is None else g.contiguous()
        if targets is not None:
            g_lp = torch.zeros(R, device=h.device) if g_lp is None else g_lp.contiguous()
        dh = torch.empty_like(h) if ctx.needs_input_grad[0] else None
        main = getattr(w, "main_grad", None)
        dw = main
        if ctx.needs_input_grad[1] and main is None:
            dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        kept, ctx.kept = ctx.kept, []
        for n, s in enumerate(range(0, R, ctx.rows)):
            e = min(R, s + ctx.rows)
            logits, saved = kept[n]
            kept[n] = None
            x = h[s:e]
            if targets is None:  # logits are unit gradients already
                if dh is not None:
                    dh[s:e] = gemm(logits, w, b_mn=True, epi=EPI_F32) * g[s:e].unsqueeze(1)
                x = (x.float() * g[s:e].unsqueeze(1)).to(h.dtype)
            else:
                ext().distill_bwd(logits, logits, ctx.temperature, ctx.slots, targets[s:e], saved, g[s:e], g_lp[s:e])
                if dh is not None:
                    gemm(logits, w, b_mn=True, out=dh[s:e])
            if ctx.needs_input_grad[1]:
                gemm(logits, x, a_mn=True, b_mn=True, out=dw, epi=EPI_ACC_F32)
        return dh, (None if main is not None or dw is None else dw.to(w.dtype)), None, None, None, None


def lm_head_distill(h: torch.Tensor, w: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                    divergence: str = "forward", beta: float = 0.5, tail: str = "bucket", temperature: float = 1.0,
                    targets: Optional[torch.Tensor] = None):
    """``distill_loss`` of the LM head ``w`` [V, H] on hidden rows ``h`` [R, H]
    (the logits are rounded to bf16, as in ``lm_head_logprob``), differentiable
    with respect to both; the weight's gradient accumulates into its
    ``main_grad`` when it has one.  With ``targets`` int64 [R] the result is
    (loss, logprob of the targets), GRPO's logprobs and the distillation loss
    from one LM head product.  The backward pass runs once."""
    beta = _check_distill("lm_head_distill", h, teacher_ids, teacher_logprobs, divergence, beta, tail, temperature)
    if h.dim() != 2 or w.dim() != 2 or h.shape[1] != w.shape[1]:
        raise ValueError(f"lm_head_distill: h [R, H] and w [V, H], got {tuple(h.shape)} and {tuple(w.shape)}")
    if h.device.type != "cuda":
        logits = torch.nn.functional.linear(h.float(), w.float())
        loss, logp = ref.distill_loss(logits, teacher_ids, teacher_logprobs, divergence, beta, tail, temperature,
                                      targets)
    else:
        kind = (DIVERGENCES[divergence], beta, tail == "drop", float(temperature))
        loss, logp = _LMHeadDistill.apply(h.contiguous(), w, teacher_ids.contiguous(), teacher_logprobs.contiguous(),
                                          kind, None if targets is None else targets.contiguous())
    return loss if targets is None else (loss, logp)


@torch.no_grad()
def lm_head_top_logprobs(h: torch.Tensor, w: torch.Tensor, k: int, temperature: float = 1.0
                         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """``top_logprobs`` of the LM head ``w`` on hidden rows ``h``, chunk by
    chunk: token ids int64 [R, k] and logprobs fp32 [R, k], a teacher's side of
    ``lm_head_distill``."""
    from . import LOGPROB_CHUNK_ROWS, linear

    k = int(k)
    if not 1 <= k <= min(MAX_TOP, w.shape[0]):
        raise ValueError(f"lm_head_top_logprobs: k must lie in [1, {min(MAX_TOP, w.shape[0])}], got {k}")
    ids = torch.empty(h.shape[0], k, dtype=torch.long, device=h.device)
    lps = torch.empty(h.shape[0], k, dtype=torch.float32, device=h.device)
    for s in range(0, h.shape[0], LOGPROB_CHUNK_ROWS):
        e = min(h.shape[0], s + LOGPROB_CHUNK_ROWS)
        ids[s:e], lps[s:e], _ = top_logprobs(linear(h[s:e], w), k, temperature)
    return ids, lps
