"""control_logits, top_logprobs, distill_loss and distill_loss_grad against
plain 64-bit restatements: on the CPU (the torch reference) and on the GPU (the
kernels), at the sizes, alignments and masks where rows of logits go wrong."""

import math

import pytest
import torch

import vocab_oracle as oracle
from libra_b200 import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U32 = 2.0 ** -24  # half a step of fp32, relative
U16 = 2.0 ** -8   # half a step of bf16, relative


def _close(got, want, tol, what):
    got, want, tol = got.double().cpu(), want.double().cpu(), torch.as_tensor(tol, dtype=torch.float64).cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: non-finite values differ"
    assert torch.equal(got[~fin], want[~fin]), f"{what}: infinities differ"
    err = (got - want).abs()[fin]
    lim = tol.expand(want.shape)[fin]
    assert bool((err <= lim).all()), f"{what}: off by {float((err - lim).max()):.3g} more than allowed"


def _view(z, layout):
    """The same rows at other strides and alignments."""
    N, V = z.shape
    if layout == "dense":
        return z
    if layout == "padded":
        buf = torch.full((N, V + 24), 77.0, dtype=z.dtype, device=z.device)
        buf[:, :V] = z
        return buf[:, :V]
    if layout == "shifted":  # rows that start off a 16-byte boundary, each differently
        buf = torch.full((N * (V + 3) + 1,), 77.0, dtype=z.dtype, device=z.device)
        v = buf[1:].view(N, V + 3)[:, :V]
        v.copy_(z)
        return v
    if layout == "transposed":
        return z.t().contiguous().t()
    raise AssertionError(layout)


def _rand(shape, seed, dtype, device, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(device)


# --------------------------------------------------------------------------- control_logits

def _control_args(B, V, L, seed, device, bias=0, mask=False):
    g = torch.Generator().manual_seed(seed)
    a = {"history": torch.randint(-2, V + 2, (B + 2, L), generator=g).int()}
    a["history"][0] = a["history"][0] % max(1, min(V, 5))  # a row of few, often repeated tokens
    a["history_rows"] = torch.randperm(B + 2, generator=g)[:B].int()
    a["history_lens"] = torch.randint(0, L + 1, (B,), generator=g).int()
    a["history_lens"][0] = L
    a["prompt_lens"] = (a["history_lens"] * torch.rand(B, generator=g)).int()
    a["repetition"] = 0.7 + 0.9 * torch.rand(B, generator=g)
    a["presence"] = torch.randn(B, generator=g)
    a["frequency"] = torch.randn(B, generator=g) * 0.5
    if bias:
        counts = torch.randint(0, bias + 1, (B,), generator=g)
        a["bias_offsets"] = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).int()
        n = int(counts.sum())
        a["bias_ids"] = torch.randint(-1, V + 1, (n,), generator=g).int()
        a["bias_values"] = torch.randn(n, generator=g) * 4
    if mask:
        W = (V + 31) // 32
        a["mask"] = torch.randint(-2 ** 31, 2 ** 31, (3, W), generator=g).int()
        a["mask"][1] = 0
        a["mask"][2] = -1
        a["mask_rows"] = (torch.arange(B) % 4 - 1).int()
    return {k: v.to(device) for k, v in a.items()}


def _check_control(z, out, args):
    want, mag = oracle.control(z, **args)
    # a division or product, two subtractions and the biases' sum: at most 8 roundings of the magnitudes involved
    tol = 8 * U32 * mag + (U16 * want.abs().nan_to_num(posinf=0, neginf=0) if out.dtype == torch.bfloat16 else 0.0)
    _close(out, want, tol, "control_logits")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V,L,layout", [(1, 1, 1, "dense"), (5, 33, 7, "dense"), (6, 1000, 1, "shifted"),
                                          (3, 2048, 300, "padded"), (4, 20001, 513, "dense"),
                                          (2, 20001, 64, "transposed"), (9, 8192, 40, "shifted")])
def test_control_logits_matches_the_oracle(device, dtype, B, V, L, layout):
    z = _view(_rand((B, V), V + L, dtype, device), layout)
    before = z.clone()
    args = _control_args(B, V, L, B + V, device, bias=9, mask=True)
    _check_control(before, ops.control_logits(z, **args), args)
    assert torch.equal(z, before)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("keep", [("history", "history_lens", "repetition"), ("history", "history_lens", "presence"),
                                  ("history", "history_lens", "prompt_lens", "frequency", "history_rows"),
                                  ("bias_offsets", "bias_ids", "bias_values"), ("mask", "mask_rows"), ()])
def test_control_logits_each_control_alone(device, keep):
    z = _rand((4, 777), 3, torch.bfloat16, device)
    args = {k: v for k, v in _control_args(4, 777, 50, 4, device, bias=20, mask=True).items() if k in keep}
    _check_control(z, ops.control_logits(z, **args), args)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_control_logits_in_place_and_special_values(device, dtype):
    z = _rand((4, 999), 9, dtype, device)
    z[0, 5], z[0, 6], z[1, 7] = math.inf, -math.inf, torch.finfo(dtype).min
    z[2, 8] = math.nan
    args = _control_args(4, 999, 30, 2, device, mask=True)
    args["mask_rows"] = torch.tensor([0, -1, 1, 0], dtype=torch.int32, device=device)  # row 2: nothing allowed
    before = z.clone()
    out = ops.control_logits(z, out=z, **args)
    assert out is z
    assert bool((z[2] == -math.inf).all())  # a NaN at a masked place is gone too
    rows = [0, 1, 3]
    sub = {k: (v[rows] if v.shape[0] == 4 else v) for k, v in args.items() if k not in ("history", "mask")}
    _check_control(before[rows], z[rows], {**sub, "history": args["history"], "mask": args["mask"]})


@pytest.mark.parametrize("device", DEVICES)
def test_control_logits_many_repeats_and_long_history(device):
    V, L = 5000, 70000  # one token more often than 16 bits count
    z = _rand((1, V), 1, torch.float32, device)
    hist = torch.full((1, L), 17, dtype=torch.int32)
    hist[0, ::1000] = 4999
    args = {"history": hist.to(device), "history_lens": torch.tensor([L], dtype=torch.int32, device=device),
            "frequency": torch.tensor([0.001], device=device)}
    _check_control(z, ops.control_logits(z, **args), args)


@pytest.mark.parametrize("device", DEVICES)
def test_control_logits_empty_batch_and_refusals(device):
    z = _rand((2, 64), 0, torch.float32, device)
    assert ops.control_logits(z[:0]).shape == (0, 64)
    one = torch.ones(2, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="2|rows, vocabulary"):
        ops.control_logits(z[0])
    with pytest.raises(ValueError, match="history"):
        ops.control_logits(z, history_lens=one)
    with pytest.raises(ValueError, match="history_lens"):
        ops.control_logits(z, history=one.view(2, 1))
    with pytest.raises(ValueError, match="mask"):
        ops.control_logits(z, mask_rows=one)
    with pytest.raises(ValueError, match="biases"):
        ops.control_logits(z, bias_ids=one)


@pytest.mark.gpu
def test_control_logits_kernel_refusals():
    z = _rand((2, 64), 0, torch.float32, "cuda")
    i32 = torch.ones(2, dtype=torch.int32, device="cuda")
    f32 = torch.ones(2, device="cuda")
    h = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for bad in (dict(repetition=f32.double()), dict(repetition=f32[:1]), dict(presence=f32.cpu()),
                dict(history=h.long(), history_lens=i32), dict(history=h[:1], history_lens=i32),
                dict(history=h, history_lens=i32.long()), dict(mask=h[:, :1]), dict(mask=h[:1]),
                dict(out=torch.empty(2, 63, device="cuda")), dict(out=torch.empty(2, 64)),
                dict(out=torch.empty(2, 64, device="cuda", dtype=torch.float16)),
                dict(bias_offsets=i32, bias_ids=i32, bias_values=f32)):
        with pytest.raises(RuntimeError, match="control_logits"):
            ops.control_logits(z, **bad)
    with pytest.raises(RuntimeError, match="control_logits"):
        ops.control_logits(z.half())
    buf = torch.zeros(3, 64, device="cuda")
    with pytest.raises(RuntimeError, match="view"):
        ops.control_logits(buf[:2], out=buf[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", ["row", "negative row", "length", "bias", "mask"])
def test_control_logits_reports_indices_outside_the_tables(bad):
    dev = torch.device("cuda", torch.cuda.current_device())
    z = _rand((2, 300), 0, torch.float32, dev)
    args = _control_args(2, 300, 6, 1, dev, bias=4, mask=True)
    if bad == "row":
        args["history_rows"][1] = 4
    elif bad == "negative row":
        args["history_rows"][1] = -1
    elif bad == "length":
        args["history_lens"][1] = 7
    elif bad == "bias":
        args["bias_offsets"][2] = 1000
    else:
        args["mask_rows"][1] = 3
    ops.check_kernel_errors(dev)
    ops.control_logits(z, **args)
    with pytest.raises(ops.KernelError, match="bad argument"):
        ops.check_kernel_errors(dev)


@pytest.mark.parametrize("device", ["cpu"])
def test_control_logits_reference_refuses_indices_outside_the_tables(device):
    z = _rand((2, 300), 0, torch.float32, device)
    for key, at, val in (("history_rows", 1, 4), ("history_lens", 1, 7), ("bias_offsets", 2, 1000), ("mask_rows", 1, 3)):
        args = _control_args(2, 300, 6, 1, device, bias=4, mask=True)
        args[key][at] = val
        with pytest.raises(ValueError, match="outside"):
            ops.control_logits(z, **args)


# --------------------------------------------------------------------------- top_logprobs

def _check_top(z, k, temperature):
    ids, lp, lse = ops.top_logprobs(z, k, temperature)
    wi, wl, ws = oracle.top(z, k, temperature)
    assert ids.dtype == torch.int64 and lp.dtype == lse.dtype == torch.float32
    assert torch.equal(ids.cpu(), wi)
    # the sum of exponentials: a rounding an addition along a thread's share and the merge, 2^-22 and three roundings
    # of the argument a term; then a few roundings of the results
    s = (z.shape[1] / 256 + 128) * U32
    _close(lp, wl, s + 4 * U32 * (wl.abs().nan_to_num(posinf=0, neginf=0) + ws.abs().nan_to_num(neginf=0).unsqueeze(1)),
           "logprobs")
    _close(lse, ws, s + 4 * U32 * ws.abs().nan_to_num(neginf=0), "lse")


TOP_SIZES = [(1, 1, 1), (3, 7, 7), (2, 300, 256), (5, 2048, 20), (4, 4097, 64), (3, 20001, 5), (2, 50257, 256),
             (300, 1024, 8)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,V,k", TOP_SIZES)
def test_top_logprobs_matches_the_oracle(device, dtype, N, V, k):
    _check_top(_rand((N, V), N + V + k, dtype, device), k, 0.7)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("layout", ["padded", "shifted", "transposed"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_top_logprobs_strides(device, layout, dtype):
    _check_top(_view(_rand((5, 3001), 8, dtype, device), layout), 17, 1.0)


def _awkward(kind, V, dtype, device):
    g = torch.Generator().manual_seed(len(kind))
    z = torch.randn(3, V, generator=g)
    if kind == "constant":
        z.fill_(1.5)
    elif kind == "zeros of both signs":
        z = torch.where(torch.rand(3, V, generator=g) < 0.5, 0.0, -0.0)
    elif kind == "ascending":
        z = torch.arange(V).float().expand(3, V) / 8
    elif kind == "descending":
        z = -torch.arange(V).float().expand(3, V) / 8
    elif kind == "two values":
        z = (torch.rand(3, V, generator=g) < 0.5).float() * 5
    elif kind == "few allowed":
        keep = torch.rand(3, V, generator=g) < 4.0 / V
        z = torch.where(keep, z, -math.inf)
    elif kind == "one allowed":
        z = torch.full((3, V), -math.inf)
        z[:, V - 1] = -2.0
    elif kind == "nothing allowed":
        z[1] = -math.inf
    elif kind == "lowest values":
        z[:] = torch.finfo(dtype).min
        z[2, V // 2] = 0.0
    elif kind == "peaks at one stride":
        z[:, ::512] += 30.0
    elif kind == "low start":
        z[:, :V // 2] -= 50.0
    elif kind == "one block of peaks":
        z[:, V // 2:V // 2 + 300] += 30.0
    elif kind == "huge":
        z *= 1e30
    return z.to(dtype).to(device)


KINDS = ["constant", "zeros of both signs", "ascending", "descending", "two values", "few allowed", "one allowed",
         "nothing allowed", "lowest values", "peaks at one stride", "low start", "one block of peaks", "huge"]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("V,k,dtype", [(700, 20, torch.bfloat16), (33000, 100, torch.float32),
                                       (33000, 256, torch.bfloat16)])
def test_top_logprobs_awkward_rows(device, kind, V, k, dtype):
    _check_top(_awkward(kind, V, dtype, device), k, 1.3)


@pytest.mark.parametrize("device", DEVICES)
def test_top_logprobs_row_temperatures_and_refusals(device):
    z = _rand((4, 500), 2, torch.bfloat16, device)
    _check_top(z, 9, torch.tensor([0.5, 2.0, 0.0, 1.0], device=device))
    z[0, 7] = 50.0  # a single best token: all of the mass in the limit of a tiny temperature
    _, lp, _ = ops.top_logprobs(z[:1], 2, 1e-30)
    assert float(lp[0, 0]) == 0.0 and float(lp[0, 1]) < -1e30
    assert [t.shape for t in ops.top_logprobs(z[:0], 3)] == [(0, 3), (0, 3), (0,)]
    for k in (0, 257, 501):
        with pytest.raises(ValueError, match="k must"):
            ops.top_logprobs(z, k)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.top_logprobs(z[0], 3)


@pytest.mark.parametrize("device", DEVICES)
def test_top_logprobs_nan_ranks_first_and_spoils_its_row_only(device):
    z = _rand((2, 600), 2, torch.float32, device)
    z[0, 77] = math.nan
    ids, lp, lse = ops.top_logprobs(z, 4)
    assert int(ids[0, 0]) == 77 and bool(torch.isnan(lp[0]).all()) and bool(torch.isnan(lse[0]))
    assert not bool(torch.isnan(lp[1]).any())


@pytest.mark.gpu
def test_top_logprobs_kernel_refusals():
    z = _rand((2, 64), 0, torch.float32, "cuda")
    with pytest.raises(RuntimeError, match="top_logprobs"):
        ops.top_logprobs(z.half(), 3)
    with pytest.raises(RuntimeError, match="temperatures"):
        ops.top_logprobs(z, 3, torch.ones(2))
    with pytest.raises(RuntimeError, match="temperatures"):
        ops.top_logprobs(z, 3, torch.ones(3, device="cuda"))


# --------------------------------------------------------------------------- distillation

def _teacher(z, k, seed, T, noise=1.0):
    g = torch.Generator().manual_seed(seed)
    t = z.float().cpu().nan_to_num(neginf=-1e4) + noise * torch.randn(z.shape, generator=g)
    lp = torch.log_softmax(t.double() / T, 1)
    top = lp.topk(k, 1)
    return top.indices.to(z.device), top.values.float().to(z.device)


def _grad_limit(z, ids, lps, div, beta, tail, T, want, g, g_lp, dtype):
    """How far each gradient may be off.  The unlisted tokens' sum carries a relative error delta, which moves a
    token's gradient by at most delta q_j (1 + |h_j| + |mean|) / T; every value has its own relative error of the
    exponential (2^-22 and three roundings of an argument of up to 64)."""
    V = z.shape[1]
    delta = (V / 256 + 128) * U32
    x = z.double().cpu()
    soft = torch.softmax(x / T, 1).nan_to_num(0.0)
    scale = torch.zeros_like(x)
    for n in range(z.shape[0]):
        tab = {}
        for i, l in zip(ids[n].tolist(), lps[n].double().tolist()):
            if 0 <= i < V and l > -math.inf and i not in tab:
                tab[i] = l
        mass = sum(math.exp(l) for l in tab.values())
        pr = max(1 - mass, oracle.REST_FLOOR) if tail == "bucket" else 0.0
        qr = max(float(soft[n].sum() - sum(float(soft[n, i]) for i in tab)), 1e-300)
        if div == "forward":
            h = {i: math.exp(l) for i, l in tab.items()}
            scale[n] = soft[n] + soft[n] * pr / qr
            for i in tab:
                scale[n, i] = soft[n, i] + h[i]
        else:
            hr = abs(math.log(max(qr, 1e-300) / max(pr, 1e-30)))
            hs = {i: abs(float(x[n, i] / T - torch.logsumexp(x[n] / T, 0)) - l) for i, l in tab.items()}
            mean = sum(float(soft[n, i]) * v for i, v in hs.items() if math.isfinite(v)) + qr * hr
            scale[n] = soft[n] * (1 + hr + mean)
            for i, v in hs.items():
                scale[n, i] = soft[n, i] * (1 + (v if math.isfinite(v) else 0.0) + mean)
    up = torch.ones(z.shape[0]) if g is None else g.cpu().abs()
    lim = scale * up.double().unsqueeze(1)
    if g_lp is not None:
        lim = lim + (1 + soft) * g_lp.cpu().double().abs().unsqueeze(1)
    lim = 4 * delta * lim / T + 300 * U32 * want.abs()
    return lim + (U16 * want.abs() if dtype == torch.bfloat16 else 0.0) + 1e-37


def _check_distill(z, ids, lps, div="forward", beta=0.5, tail="bucket", T=1.0, targets=None, one_pass=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    N, V = z.shape
    g = None if one_pass else (torch.randn(N, generator=gen)).to(z.device)
    g_lp = None if targets is None else torch.randn(N, generator=gen).to(z.device)
    kw = dict(divergence=div, beta=beta, tail=tail, temperature=T)
    logp = None
    if one_pass:
        loss, grad = ops.distill_loss_grad(z, ids, lps, **kw)
    else:
        x = z.detach().requires_grad_(True)
        if targets is None:
            loss = ops.distill_loss(x, ids, lps, **kw)
            (grad,) = torch.autograd.grad(loss, x, g)
        else:
            loss, logp = ops.distill_loss(x, ids, lps, targets=targets, **kw)
            (grad,) = torch.autograd.grad((loss, logp), x, (g, g_lp))
    assert loss.dtype == torch.float32 and grad.dtype == z.dtype and grad.shape == z.shape
    wl, wp, wg = oracle.distill(z, ids.cpu(), lps.cpu(), div, beta, tail, T, targets, g, g_lp)
    delta = (V / 256 + 128) * U32
    lim = _grad_limit(z, ids, lps, div, beta, tail, T, wg, g, g_lp, z.dtype)
    unit = _grad_limit(z, ids, lps, div, beta, tail, T, torch.zeros_like(wg), None, None, torch.float32)
    # the loss moves by delta times its derivative by the unlisted sum, which the limits above bound
    _close(loss, wl, unit.sum(1) * T + 4 * U32 * wl.abs().nan_to_num(posinf=0), "loss")
    _close(grad, wg, lim, "gradient")
    if targets is not None:
        _close(logp, wp, delta + 4 * U32 * wp.abs().nan_to_num(posinf=0, neginf=0), "logprob")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("div,tail", [("forward", "bucket"), ("forward", "drop"), ("reverse", "bucket"),
                                      ("js", "bucket"), ("js", "drop")])
@pytest.mark.parametrize("N,V,K", [(1, 2, 1), (4, 33, 33), (3, 1000, 256), (2, 2047, 17), (3, 12289, 64)])
def test_distill_matches_the_oracle(device, dtype, div, tail, N, V, K):
    z = _rand((N, V), V + K, dtype, device)
    ids, lps = _teacher(z, K, V, 0.8)
    _check_distill(z, ids, lps, div, 0.3, tail, 0.8)
    _check_distill(z, ids, lps, div, 0.3, tail, 0.8, one_pass=True)
    targets = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(V)).to(device)
    targets[0] = ids[0, 0]
    _check_distill(z, ids, lps, div, 0.3, tail, 0.8, targets=targets)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("layout", ["padded", "shifted", "transposed"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_strides(device, layout, dtype):
    z = _view(_rand((4, 3001), 8, dtype, device), layout)
    ids, lps = _teacher(z, 12, 5, 1.0)
    _check_distill(z, ids, lps, "js", 0.5)
    _check_distill(z, ids, lps, "js", 0.5, one_pass=True)
    if layout != "transposed":
        # in place: the bits of a call out of place on rows that start as they do (a row's alignment orders its sum,
        # so rows aligned otherwise agree within the limits above only)
        loss, grad = ops.distill_loss_grad(z, ids, lps)
        w = _view(z.clone(), layout)
        loss2, out = ops.distill_loss_grad(w, ids, lps, out=w)
        assert out is w and torch.equal(loss, loss2) and torch.equal(grad, w)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("div", ["forward", "reverse", "js"])
def test_distill_empty_slots_and_rows(device, div):
    V = 900
    z = _rand((7, V), 4, torch.float32, device)
    ids, lps = _teacher(z, 10, 6, 1.0)
    ids[0] = -1                                # no teacher here
    lps[1] = -math.inf
    lps[2] = math.nan
    ids[3, 4:], lps[3, 4:] = -1, math.nan      # a short table
    ids[4, 5], ids[4, 6] = V, 2 ** 40          # tokens of another vocabulary
    ids[5, 3], ids[5, 7] = ids[5, 0], ids[5, 1]  # the same token twice: the first slot counts
    ids[6, 1:] = ids[6, 0]
    targets = torch.arange(7, device=device) * 11
    _check_distill(z, ids, lps, div)
    _check_distill(z, ids, lps, div, one_pass=True)
    _check_distill(z, ids, lps, div, targets=targets)
    loss, grad = ops.distill_loss_grad(z, ids, lps, divergence=div)
    assert not bool(loss[:3].any()) and not bool(grad[:3].any())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("div", ["forward", "reverse", "js"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_masked_student(device, div, dtype):
    V = 1200
    z = _rand((5, V), 14, dtype, device)
    ids, lps = _teacher(z, 8, 6, 1.0)
    z[0, torch.randperm(V, generator=torch.Generator().manual_seed(1))[:900].to(device)] = -math.inf
    z[1] = torch.finfo(dtype).min
    listed = torch.zeros(V, dtype=torch.bool, device=device)
    listed[ids[2]] = True
    z[2, ~listed] = -math.inf                   # the student holds nothing outside the table
    z[3, listed] += 200.0                       # and next to nothing
    keep0 = torch.isfinite(z[0, ids[0]])
    ids[0] = torch.where(keep0, ids[0], -1)     # (an infinite loss otherwise)
    _check_distill(z, ids, lps, div)
    _check_distill(z, ids, lps, div, one_pass=True)


@pytest.mark.parametrize("device", DEVICES)
def test_distill_row_of_nothing_but_minus_infinity(device):
    z = _rand((3, 700), 2, torch.bfloat16, device)
    ids, lps = _teacher(z, 5, 3, 1.0)
    z[1] = -math.inf
    targets = torch.tensor([1, 2, 3], device=device)
    x = z.clone().requires_grad_(True)
    loss, logp = ops.distill_loss(x, ids, lps, targets=targets)
    assert float(loss[1]) == 0.0 and float(logp[1]) == -math.inf
    (grad,) = torch.autograd.grad((loss.sum() + logp[[0, 2]].sum()), x)
    assert not bool(grad[1].any()) and bool(torch.isfinite(grad).all())


@pytest.mark.parametrize("device", DEVICES)
def test_distill_masked_target_has_the_softmax_gradient(device):
    z = _rand((2, 400), 2, torch.float32, device)
    ids, lps = _teacher(z, 5, 3, 1.0)
    targets = torch.tensor([7, 9], device=device)
    ids[ids == 7] = -1
    z[0, 7] = -math.inf
    x = z.clone().requires_grad_(True)
    loss, logp = ops.distill_loss(x, ids, lps, targets=targets)
    assert float(logp[0].detach()) == -math.inf
    (grad,) = torch.autograd.grad(logp, x, torch.ones_like(logp))
    want = torch.nn.functional.one_hot(targets, 400) - torch.softmax(z.double(), 1)
    assert torch.allclose(grad.double(), want, rtol=1e-4, atol=1e-7)


@pytest.mark.parametrize("device", DEVICES)
def test_distill_infinite_where_the_student_excludes_a_teacher_token(device):
    z = _rand((2, 400), 2, torch.float32, device)
    ids, lps = _teacher(z, 5, 3, 1.0)
    z[0, ids[0, 2]] = -math.inf
    loss, grad = ops.distill_loss_grad(z, ids, lps)
    assert float(loss[0]) == math.inf and math.isfinite(float(loss[1]))
    assert bool(torch.isfinite(grad).all())
    loss, _ = ops.distill_loss_grad(z, ids, lps, divergence="reverse")
    assert bool(torch.isfinite(loss).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("div", ["forward", "reverse", "js"])
def test_distill_gradient_against_differences(device, div):
    V, eps = 50, 1e-5
    z = _rand((2, V), 3, torch.float32, device, scale=1.0)
    ids, lps = _teacher(z, 6, 2, 0.9)
    _, grad = ops.distill_loss_grad(z, ids, lps, divergence=div, beta=0.25, temperature=0.9)
    for n in range(2):
        row = z[n].double().cpu()
        args = (ids[n].tolist(), lps[n].double().tolist(), div, 0.25, "bucket", 0.9)
        for j in range(V):
            up, dn = row.clone(), row.clone()
            up[j] += eps
            dn[j] -= eps
            d = (float(oracle.distill_row(up, *args)[0]) - float(oracle.distill_row(dn, *args)[0])) / (2 * eps)
            # central differences: eps^2 of the third derivative and 2^-52 / eps of the loss
            assert abs(d - float(grad[n, j])) < 1e-8 + 2e-5 * abs(d) + 4 * 178 * U32 * 10


@pytest.mark.parametrize("device", DEVICES)
def test_distill_same_teacher_gives_nothing_to_learn(device):
    z = _rand((3, 5000), 3, torch.float32, device)
    lp = torch.log_softmax(z.double(), 1)
    top = lp.topk(30, 1)
    for div in ("forward", "reverse", "js"):
        loss, grad = ops.distill_loss_grad(z, top.indices, top.values.float(), divergence=div)
        # the logprobs' own rounding (2^-24 of up to 16) is the teacher's difference from the student
        assert float(loss.abs().max()) < 64 * U32 and float(grad.abs().max()) < 600 * U32


@pytest.mark.parametrize("device", DEVICES)
def test_distill_upstream_gradients(device):
    """Broadcast upstream gradients, a loss that uses only one of the two outputs, and rows of zero weight."""
    z = _rand((4, 800), 3, torch.float32, device)
    ids, lps = _teacher(z, 6, 2, 1.0)
    t = torch.tensor([1, 2, 3, 4], device=device)
    _, unit = ops.distill_loss_grad(z, ids, lps)
    x = z.clone().requires_grad_(True)
    (a,) = torch.autograd.grad(ops.distill_loss(x, ids, lps).sum(), x)
    assert torch.allclose(a, unit, rtol=1e-6, atol=1e-9)
    loss, logp = ops.distill_loss(x, ids, lps, targets=t)
    (b,) = torch.autograd.grad(loss.mean(), x, retain_graph=True)
    assert torch.allclose(b, unit / 4, rtol=1e-6, atol=1e-9)
    (c,) = torch.autograd.grad(logp.sum(), x)
    want = torch.nn.functional.one_hot(t, 800) - torch.softmax(z.double(), 1)
    assert torch.allclose(c.double(), want, rtol=1e-4, atol=1e-7)
    w = torch.tensor([1.0, 0.0, 2.0, 0.0], device=device)
    (d,) = torch.autograd.grad((ops.distill_loss(x, ids, lps) * w).sum(), x)
    assert not bool(d[1].any()) and not bool(d[3].any())


@pytest.mark.parametrize("device", DEVICES)
def test_distill_refusals_and_empty_batch(device):
    z = _rand((2, 64), 0, torch.float32, device)
    ids, lps = _teacher(z, 3, 2, 1.0)
    for bad in (dict(divergence="kl"), dict(tail="none"), dict(divergence="reverse", tail="drop"),
                dict(divergence="js", beta=1.0), dict(divergence="js", beta=0.0), dict(temperature=0.0),
                dict(temperature=math.inf)):
        for f in (ops.distill_loss, ops.distill_loss_grad):
            with pytest.raises(ValueError, match=f.__name__):
                f(z, ids, lps, **bad)
    with pytest.raises(ValueError, match="K"):
        ops.distill_loss(z, ids[:1], lps[:1])
    with pytest.raises(ValueError, match="K"):
        ops.distill_loss(z, ids, lps[:, :2])
    with pytest.raises(ValueError, match="1 to 256"):
        ops.distill_loss(z, ids[:, :0], lps[:, :0])
    with pytest.raises(ValueError, match="vocabulary"):
        ops.distill_loss(z[0], ids, lps)
    loss, grad = ops.distill_loss_grad(z[:0], ids[:0], lps[:0])
    assert loss.shape == (0,) and grad.shape == (0, 64)


@pytest.mark.gpu
def test_distill_kernel_refusals():
    z = _rand((2, 64), 0, torch.float32, "cuda")
    ids, lps = _teacher(z, 3, 2, 1.0)
    for bad in ((z.half(), ids, lps), (z, ids.int(), lps), (z, ids, lps.double()), (z, ids.cpu(), lps)):
        with pytest.raises(RuntimeError, match="distill_loss"):
            ops.distill_loss(*bad)
    with pytest.raises(RuntimeError, match="targets"):
        ops.distill_loss(z, ids, lps, targets=torch.zeros(2, dtype=torch.int32, device="cuda"))
    buf = torch.zeros(3, 64, device="cuda")
    with pytest.raises(RuntimeError, match="view"):
        ops.distill_loss_grad(buf[:2], ids, lps, out=buf[1:])


@pytest.mark.gpu
def test_distill_refuses_second_derivatives_and_changed_logits():
    z = _rand((2, 64), 0, torch.float32, "cuda").requires_grad_(True)
    ids, lps = _teacher(z.detach(), 3, 2, 1.0)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(ops.distill_loss(z, ids, lps).sum(), z, create_graph=True)
    y = z * 1.0
    loss = ops.distill_loss(y, ids, lps).sum()
    y.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    assert not ops.distill_loss(z.detach(), ids, lps).requires_grad


@pytest.mark.gpu
def test_distill_reports_targets_outside_the_vocabulary():
    dev = torch.device("cuda", torch.cuda.current_device())
    z = _rand((3, 500), 0, torch.float32, dev).requires_grad_(True)
    ids, lps = _teacher(z.detach(), 3, 2, 1.0)
    ops.check_kernel_errors(dev)
    loss, logp = ops.distill_loss(z, ids, lps, targets=torch.tensor([1, 500, -1], device=dev))
    assert float(logp[1].detach()) == float(logp[2].detach()) == -math.inf
    with pytest.raises(ops.KernelError, match="bad argument"):
        ops.check_kernel_errors(dev)
    (grad,) = torch.autograd.grad(logp.sum(), z)  # no target, no gradient
    assert not bool(grad[1:].any()) and bool(grad[0].any())


# --------------------------------------------------------------------------- together

@pytest.mark.gpu
def test_vocab_ops_on_a_side_stream_and_in_two_graphs():
    """Calls on another stream, two calls in flight, and two captured graphs that replay independently."""
    z = [_rand((6, 9001), s, torch.bfloat16, "cuda") for s in (1, 2)]
    t = [_teacher(x, 16, 7, 1.0) for x in z]
    args = _control_args(6, 9001, 100, 5, "cuda", bias=6, mask=True)

    def work(i, x):
        loss, grad = ops.distill_loss_grad(x, *t[i])
        return (*ops.top_logprobs(x, 10, 0.9), loss, grad, ops.control_logits(x, **args))

    want = [work(i, z[i]) for i in (0, 1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    torch.cuda.synchronize()
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            got[i] = work(i, z[i])
    torch.cuda.synchronize()
    graphs, outs, inputs = [], [], [torch.zeros_like(x) for x in z]
    for i in (0, 1):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(work(i, inputs[i]))
        graphs.append(gr)
    for i in (0, 1):
        inputs[i].copy_(z[i])
    torch.cuda.synchronize()
    for _ in range(2):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        for w, a, b in zip(want[i], got[i], outs[i]):
            assert torch.equal(w, a) and torch.equal(w, b)


@pytest.mark.gpu
def test_distill_backward_in_a_captured_graph():
    z = _rand((5, 3000), 1, torch.bfloat16, "cuda")
    ids, lps = _teacher(z, 9, 7, 1.0)
    tg = torch.arange(5, device="cuda")
    x = z.clone().requires_grad_(True)

    def step():
        loss, logp = ops.distill_loss(x, ids, lps, targets=tg)
        return torch.autograd.grad(loss.mean() - logp.mean(), x)[0]

    want = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step()
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_controlled_rows_feed_the_other_operators(device):
    """A sampled batch as it is used: controls, then the top alternatives, then a student distilled on them."""
    V = 4000
    z = _rand((5, V), 1, torch.bfloat16, device)
    args = _control_args(5, V, 60, 5, device, bias=6, mask=True)
    args["mask_rows"] = torch.tensor([0, -1, 2, 0, -1], dtype=torch.int32, device=device)
    x = ops.control_logits(z, **args)
    want, _ = oracle.control(z, **args)
    ids, lp, lse = ops.top_logprobs(x, 12, 0.7)
    _check_top(x, 12, 0.7)
    assert torch.allclose(lse.double().cpu(), torch.logsumexp(want / 0.7, 1), atol=1e-4)
    _check_distill(_rand((5, V), 2, torch.bfloat16, device), ids, lp, "forward", T=0.7)
