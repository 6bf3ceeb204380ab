"""What the vocabulary-row operators promise about their arguments: bad indices,
gradients, in-place outputs, arguments that a form does not use."""

import pytest
import torch

from libra_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _raises_outside(device, call):
    """A bad index raises on the CPU; the kernels report it through the error word."""
    if device == "cpu":
        with pytest.raises(ValueError, match="outside"):
            call()
        return
    dev = torch.device("cuda", torch.cuda.current_device())
    ops.check_kernel_errors(dev)
    call()
    with pytest.raises(ops.KernelError, match="bad argument"):
        ops.check_kernel_errors(dev)


@pytest.mark.parametrize("device", DEVICES)
def test_control_logits_with_empty_tables(device):
    z = torch.randn(2, 100, generator=torch.Generator().manual_seed(1)).to(device)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    rep = torch.tensor([1.5, 1.5], device=device)
    no_mask = torch.zeros(0, 4, dtype=torch.int32, device=device)
    out = ops.control_logits(z, mask=no_mask, mask_rows=i32(-1, -1))
    assert torch.equal(out, z)
    _raises_outside(device, lambda: ops.control_logits(z, mask=no_mask, mask_rows=i32(-1, 0)))
    no_width = torch.zeros(2, 0, dtype=torch.int32, device=device)
    out = ops.control_logits(z, history=no_width, history_lens=i32(0, 0), repetition=rep)
    assert torch.equal(out, z)
    _raises_outside(device, lambda: ops.control_logits(z, history=no_width, history_lens=i32(0, 1), repetition=rep))
    no_rows = torch.zeros(0, 8, dtype=torch.int32, device=device)
    _raises_outside(device, lambda: ops.control_logits(z, history=no_rows, history_rows=i32(0, 0),
                                                       history_lens=i32(1, 1), repetition=rep))


@pytest.mark.parametrize("device", DEVICES)
def test_controls_and_top_logprobs_are_not_differentiated_through(device):
    x = torch.randn(3, 200, generator=torch.Generator().manual_seed(1)).to(device).requires_grad_(True)
    frequency, presence = torch.ones(3, device=device), torch.ones(3, device=device)
    hist = torch.ones(3, 2, dtype=torch.int32, device=device)
    lens = torch.full((3,), 2, dtype=torch.int32, device=device)
    kw = dict(history=hist, history_lens=lens, frequency=frequency, presence=presence)
    assert not ops.control_logits(x, **kw).requires_grad
    assert not any(t.requires_grad for t in ops.top_logprobs(x, 4))
    assert not any(t.requires_grad for t in ops.distill_loss_grad(x, torch.ones(3, 1, dtype=torch.long, device=device),
                                                                  torch.zeros(3, 1, device=device)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["control_logits", "distill_loss_grad"])
def test_logits_overwritten_before_their_backward_pass_are_noticed(device, which):
    x = torch.randn(2, 64, generator=torch.Generator().manual_seed(1)).to(device).requires_grad_(True)
    ids = torch.tensor([[1, 2], [3, 4]], device=device)
    lps = torch.log(torch.tensor([[0.5, 0.2], [0.3, 0.3]], device=device))
    y = x * 1.0
    loss = y.exp().sum()  # (keeps exp(y); y * y keeps y itself)
    loss = loss + (y * y).sum()
    before = y._version
    if which == "control_logits":
        assert ops.control_logits(y, mask=torch.zeros(2, 2, dtype=torch.int32, device=device), out=y) is y
    else:
        assert ops.distill_loss_grad(y, ids, lps, out=y)[1] is y
    assert y._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("beta", [0.0, 1.0, 7.0])
def test_beta_belongs_to_js_alone(device, beta):
    z = torch.randn(2, 64, generator=torch.Generator().manual_seed(1)).to(device)
    ids = torch.tensor([[1, 2], [3, 4]], device=device)
    lps = torch.log(torch.tensor([[0.5, 0.2], [0.3, 0.3]], device=device))
    for div in ("forward", "reverse"):
        want = ops.distill_loss_grad(z, ids, lps, divergence=div)
        assert all(torch.equal(a, b) for a, b in zip(want, ops.distill_loss_grad(z, ids, lps, divergence=div, beta=beta)))
        assert torch.equal(want[0], ops.distill_loss(z, ids, lps, divergence=div, beta=beta))
    w, h = torch.randn(64, 64).bfloat16().to(device), torch.randn(2, 64).bfloat16().to(device)
    assert torch.equal(ops.lm_head_distill(h, w, ids, lps, beta=beta), ops.lm_head_distill(h, w, ids, lps))
    for f in (ops.distill_loss, ops.distill_loss_grad):
        with pytest.raises(ValueError, match="beta"):
            f(z, ids, lps, divergence="js", beta=beta)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_without_a_penalty_need_no_history(device):
    z = torch.randn(2, 100, generator=torch.Generator().manual_seed(1)).to(device)
    hist = torch.tensor([[5, 5, 6]], dtype=torch.int32, device=device)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)  # noqa: E731
    f32 = lambda *v: torch.tensor(v, device=device)  # noqa: E731
    ops.check_kernel_errors()
    out = ops.control_logits(z, history=hist, history_rows=i32(0, 99), history_lens=i32(3, -5), repetition=f32(1.0, 1.0),
                             presence=f32(0.5, 0.0), frequency=f32(0.25, 0.0))
    ops.check_kernel_errors()
    want = z.clone()
    want[0, 5] -= 1.0
    want[0, 6] -= 0.75
    # two roundings of values near 2
    assert float((out - want).abs().max()) <= 4 * 2.0 ** -24 * float(z.abs().max() + 1.0)
