"""Rows and tables at the ends of what the vocabulary-row operators accept:
probabilities that fp32, or fp64, holds only as subnormals or not at all."""

import math

import pytest
import torch

import vocab_oracle as oracle
from libra_b200 import ops
from test_vocab_ops import _close, _grad_limit

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U32 = 2.0 ** -24


def _both_forms(z, ids, lps, want_lps, div, beta, tail, T):
    """distill_loss (with its gradient) and distill_loss_grad on (ids, lps) against the oracle on (ids, want_lps)."""
    wl, _, wg = oracle.distill(z, ids.cpu(), want_lps.cpu(), div, beta, tail, T)
    lim = _grad_limit(z, ids, want_lps, div, beta, tail, T, wg, None, None, z.dtype)
    unit = _grad_limit(z, ids, want_lps, div, beta, tail, T, torch.zeros_like(wg), None, None, torch.float32)
    # as for moderate rows: the loss moves by the unlisted sum's error times its derivative, then a few roundings
    loss_lim = unit.sum(1) * T + 4 * U32 * wl.abs()
    kw = dict(divergence=div, beta=beta, tail=tail, temperature=T)
    x = z.detach().requires_grad_(True)
    loss = ops.distill_loss(x, ids, lps, **kw)
    (grad,) = torch.autograd.grad(loss.sum(), x)
    _close(loss.detach(), wl, loss_lim, "loss")
    _close(grad, wg, lim, "gradient")
    loss, grad = ops.distill_loss_grad(z, ids, lps, **kw)
    _close(loss, wl, loss_lim, "loss, one pass")
    _close(grad, wg, lim, "gradient, one pass")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [0.02, 0.05, 1.0])
@pytest.mark.parametrize("div", ["forward", "reverse", "js"])
def test_distill_listed_tokens_that_the_student_all_but_excludes(device, T, div):
    """Listed tokens 690 to 760 / T below the maximum: q is a subnormal of fp64, then 0, while p is ordinary."""
    gaps = [690.0, 708.0, 709.5, 712.0, 725.0, 740.0, 744.0, 760.0]
    g = torch.Generator().manual_seed(4)
    z = torch.randn(len(gaps), 300, generator=g) * T
    ids = torch.tensor([[7, 19, 250, 3]]).repeat(len(gaps), 1)
    for n, gap in enumerate(gaps):
        z[n, 100] = 6 * T
        for k in range(4):
            z[n, ids[n, k]] = (6 - gap - 0.3 * k) * T
    lps = torch.log(torch.tensor([[0.5, 0.3, 0.1, 0.05]])).repeat(len(gaps), 1)
    z, ids, lps = z.to(device), ids.to(device), lps.to(device)
    _both_forms(z, ids, lps, lps, div, 0.5, "bucket", T)
    if div == "js":
        _both_forms(z, ids, lps, lps, div, 0.1, "drop", T)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("div", ["forward", "js"])
def test_distill_drop_of_tables_with_little_mass(device, dtype, div):
    """tail="drop" divides by the table's mass, however small: adding a constant to a row's logprobs changes nothing."""
    levels = [0.0, -60.0, -86.0, -90.0, -110.0, -200.0, -700.0, -740.0, -800.0, -1e6]
    g = torch.Generator().manual_seed(8)
    z = torch.randn(len(levels), 500, generator=g).to(dtype).to(device)
    base = torch.tensor([-0.5, -1.0, -3.0, -6.5, -0.5])
    ids = torch.tensor([3, 40, 77, 499, 3])  # the last slot repeats a token, and does not count
    at = torch.tensor(levels).unsqueeze(1)
    for K in (1, 5):
        row_ids = ids[:K].repeat(len(levels), 1).to(device)
        lps = (at + base[:K]).to(device)  # (exact in fp32)
        want = base[:K].repeat(len(levels), 1)
        _both_forms(z, row_ids, lps, want, div, 0.4, "drop", 0.8)
    # a second slot that does not count may be the likelier one
    lps = torch.tensor([[-800.0, 0.0, -801.0]], device=device)
    row_ids = torch.tensor([[5, 5, 9]], device=device)
    _both_forms(z[:1], row_ids, lps, torch.tensor([[0.0, 0.0, -1.0]]), div, 0.4, "drop", 0.8)
