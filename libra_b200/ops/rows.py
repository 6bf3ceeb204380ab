"""Operators that move rows by sorted indices: the embedding, whose gradient is
summed by sorted tokens, and a mixture-of-experts layer's router, plan, dispatch
and combine.

They dispatch like the other operators of :mod:`libra_b200.ops`: CUDA tensors
run the kernels of ``embedding.cu`` and ``expert_rows.cu`` (bf16 and fp32); CPU
tensors run :mod:`libra_b200.ops.reference`, whatever floats they hold.  The same
inputs give the same bits.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

import libra_b200.ops as _lib

from . import reference as ref

MAX_EXPERTS = 1024  # of route_topk and expert_plan


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------

def embedding_rows(tokens: torch.Tensor, weight: torch.Tensor, scale: float, first: int, whole: bool,
                   want_order: bool = False):
    """``embedding`` without a gradient: the rows, and with ``want_order`` what ``embedding_grad`` takes of the tokens."""
    if weight.device.type != "cuda":
        with torch.no_grad():
            return ref.embedding(tokens, weight, scale, first, whole), tokens
    return tuple(_lib.ext().embedding_fwd(tokens, weight, scale, first, whole, want_order,
                                          _lib.error_flag(weight.device)))


def embedding_grad(order: torch.Tensor, g: torch.Tensor, weight: torch.Tensor, scale: float,
                   first: int) -> Optional[torch.Tensor]:
    """Gradient of ``embedding`` with respect to ``weight`` from that of its
    result: added to ``weight.main_grad`` when there is one, else returned."""
    main = getattr(weight, "main_grad", None)
    if weight.device.type != "cuda":
        dw = ref.embedding_grad(order, g.reshape(-1, weight.shape[1]), weight.shape[0], scale, first, main)
        return None if dw is None else dw.to(weight.dtype)
    dw = _lib.ext().embedding_bwd(order, g, weight, scale, main)
    if main is not None:
        torch.autograd.graph.increment_version(main)
        return None
    return dw


class _EmbeddingCPU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, w, scale, first, whole):
        ctx.save_for_backward(tokens)
        ctx.w, ctx.scale, ctx.first = w, scale, first  # the gradient needs the table's shape, not its values
        return embedding_rows(tokens, w, scale, first, whole)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (tokens,) = ctx.saved_tensors
        return None, embedding_grad(tokens, g, ctx.w, ctx.scale, ctx.first), None, None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
              vocab_start: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``, of the weight's type (bf16 or fp32; any floats
    on the CPU) with one rounding: tokens int64 or int32 of any shape, weight
    [V, H], result [*tokens.shape, H].

    With ``vocab_start`` the weight is a shard that begins at that token:
    tokens outside it give rows of zeros and no gradient.  Without it they are
    an error: a row of zeros and the error word that ``check_kernel_errors``
    raises (ValueError on the CPU).

    Differentiable with respect to the weight.  The gradient sums each token's
    rows in fp32 in a fixed order, so that it does not change from run to run.
    It is added to ``weight.main_grad`` (contiguous fp32) when there is one, else
    it is a dense tensor like the weight.  Until the backward pass the tokens'
    order is kept, 16 bytes a token."""
    first, whole = (0, True) if vocab_start is None else (int(vocab_start), False)
    if weight.is_cuda:
        return _lib.ext().embedding(tokens, weight, scale, first, whole, _lib.error_flag(weight.device))
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"embedding: weight must be [V, H] of floats, got {tuple(weight.shape)} {weight.dtype}")
    if tokens.dtype not in (torch.int64, torch.int32) or tokens.device != weight.device:
        raise ValueError(f"embedding: tokens must be int64 or int32 on {weight.device}, got {tokens.dtype} on "
                         f"{tokens.device}")
    if weight.stride(1) != 1 and weight.shape[1] > 1:
        raise ValueError("embedding: the weight's rows must be contiguous")
    return _EmbeddingCPU.apply(tokens, weight, float(scale), first, whole)


# ---------------------------------------------------------------------------
# router
# ---------------------------------------------------------------------------

def route_topk(logits: torch.Tensor, k: int, *, normalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` largest of each row's router logits [T, E] (bf16 or
    fp32, E up to 1024) and their softmax weights: (weights fp32 [T, k],
    experts int64 [T, k]), in descending order, ties at the lowest index.

    ``normalize`` divides the k weights by their sum.  A logit of -inf has
    weight 0; a row of nothing but -inf has weights 0 and experts 0 to k - 1.
    NaN ranks above +inf and makes the row's weights NaN.  The weights are
    differentiable with respect to the logits."""
    if logits.is_cuda:
        return _lib.ext().route_topk(logits, k, normalize)
    k = int(k)
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"route_topk: logits must be [T, E] of floats, got {tuple(logits.shape)} {logits.dtype}")
    E = logits.shape[1]
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= E:
        raise ValueError(f"route_topk: 1 to {MAX_EXPERTS} experts and k in [1, {E}], got {E} and {k}")
    return ref.route_topk(logits, k, normalize)


# ---------------------------------------------------------------------------
# experts' rows
# ---------------------------------------------------------------------------

@dataclass
class ExpertPlan:
    """Where each (token, slot) pair j = t * k + i lives in the experts' layout of ``capacity`` rows."""

    rows: torch.Tensor    # int32 [T * k]: the pair's row, -1 for a pair without an expert
    offs: torch.Tensor    # int32 [E + 1]: expert e owns rows [offs[e], offs[e + 1])
    counts: torch.Tensor  # int32 [E]: of which the first counts[e] are its pairs', in the pairs' order
    num_tokens: int
    k: int
    align: int
    capacity: int


def expert_plan(experts: torch.Tensor, num_experts: int, *, align: int = 128) -> ExpertPlan:
    """Sorts (token, slot) pairs by expert: ``experts`` int64 or int32 [T, k]
    (``route_topk``'s), every expert's group of rows starting on a multiple of
    ``align`` (the grouped products want 128).  Nothing is read back to the
    host: the layout's capacity covers any choice of experts.

    A negative id leaves its pair without an expert (a padding token).  An id
    of ``num_experts`` or more does so too and sets the error word that
    ``check_kernel_errors`` raises (ValueError on the CPU)."""
    if experts.is_cuda:
        rows, offs, counts, capacity = _lib.ext().expert_plan(experts, num_experts, align,
                                                              _lib.error_flag(experts.device))
        return ExpertPlan(rows, offs, counts, experts.shape[0], experts.shape[1], align, capacity)
    if experts.dim() != 2 or experts.shape[1] < 1 or experts.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"expert_plan: experts must be int64 or int32 [T, k], got {tuple(experts.shape)} "
                         f"{experts.dtype}")
    num_experts, align = int(num_experts), int(align)
    if not 1 <= num_experts <= MAX_EXPERTS or align < 1:
        raise ValueError(f"expert_plan: 1 to {MAX_EXPERTS} experts and align >= 1, got {num_experts} and {align}")
    T, k = experts.shape
    capacity = T * k + (align - 1) * min(num_experts, T * k)
    if capacity == 0 and align > 1:
        capacity = align  # no pairs still leave one group's rows: the grouped products take no empty tensor
    if capacity >= 2 ** 31:
        raise ValueError(f"expert_plan: {capacity} rows do not fit 31 bits")
    return ExpertPlan(*ref.expert_plan(experts, num_experts, align), T, k, align, capacity)


def _check_rows(op: str, what: str, x: torch.Tensor, plan: ExpertPlan, count: int) -> None:
    if x.dim() != 2 or not x.is_floating_point() or x.shape[0] != count:
        raise ValueError(f"{op}: {what} must be [{count}, H] of floats, got {tuple(x.shape)} {x.dtype}")
    if x.device != plan.rows.device:
        raise ValueError(f"{op}: {what} on {x.device}, the plan on {plan.rows.device}")


def moe_dispatch(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """Rows x [T, H] (bf16 or fp32) copied to their experts' groups:
    [capacity, H], zeros in every row that is no pair's.  Differentiable: a
    token's gradient is the fp32 sum over its pairs' rows."""
    if x.is_cuda:
        return _lib.ext().moe_dispatch(x, plan.rows, plan.offs, plan.counts, plan.k, plan.align, plan.capacity)
    _check_rows("moe_dispatch", "x", x, plan, plan.num_tokens)
    return ref.moe_dispatch(x, plan.rows, plan.k, plan.capacity)


def moe_combine(y: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = residual[t] + sum_i weights[t, i] * y[row of pair (t, i)]``
    for the experts' rows y [capacity, H] (bf16 or fp32), weights [T, k] (fp32)
    and an optional residual [T, H] of y's type: summed in fp32 in the order of
    i, one rounding.  A pair without an expert adds nothing.  Differentiable
    with respect to y (zeros in rows that are no pair's), weights and residual."""
    if y.is_cuda:
        return _lib.ext().moe_combine(y, weights, residual, plan.rows, plan.offs, plan.counts, plan.k, plan.align,
                                      plan.capacity, plan.num_tokens)
    _check_rows("moe_combine", "y", y, plan, plan.capacity)
    if tuple(weights.shape) != (plan.num_tokens, plan.k) or weights.device != y.device:
        raise ValueError(f"moe_combine: weights must be [{plan.num_tokens}, {plan.k}] on {y.device}, got "
                         f"{tuple(weights.shape)} on {weights.device}")
    if residual is not None and (tuple(residual.shape) != (plan.num_tokens, y.shape[1]) or residual.dtype != y.dtype
                                 or residual.device != y.device):
        raise ValueError(f"moe_combine: the residual must be [{plan.num_tokens}, {y.shape[1]}] {y.dtype} on "
                         f"{y.device}, got {tuple(residual.shape)} {residual.dtype} on {residual.device}")
    return ref.moe_combine(y, weights.float(), plan.rows, plan.k, residual)
