"""The vocabulary-row kernels at batch and vocabulary sizes that cross each of
their dispatch limits, which smaller rows never reach: several rounds of loads
a thread, the mid-row bound and its overflow into the exact selection, splits
of a row of 1 to 32, clusters of 4, 8 and 16, held slices up to the shared
memory's limit and the two-pass form beyond it, and the controls' tiles of
16384 and 32768 tokens with 16- and 32-bit counters."""

import math

import pytest
import torch

from libra_b200 import ops
from test_vocab_ops import U16, U32, _view

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def _close_rows(got, want, tol, what):
    """``_close`` on the device the values are on."""
    got, want = got.double(), want.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: non-finite values differ"
    assert torch.equal(got[~fin], want[~fin]), f"{what}: infinities differ"
    over = torch.where(fin, (got - want).abs() - tol, -math.inf)
    assert float(over.max()) <= 0.0, f"{what}: off by {float(over.max()):.3g} more than allowed"


def _rows(N, V, dtype, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(N, V, device="cuda", generator=g) * scale).to(dtype)


# --------------------------------------------------------------------------- top_logprobs

def _shapes_of_rows(N, V, dtype):
    """Rows whose values defeat or stress the selection's bound, one kind after the other."""
    z = _rows(N, V, torch.float32, N + V)
    g = torch.Generator(device="cuda").manual_seed(1)
    at = torch.arange(V, device="cuda").float()
    z[1::9] = at / 64                                                       # rising: every octet is noted
    z[2::9] = -at / 64
    z[3::9] = 1.5                                                           # one long tie
    z[4::9] = (torch.rand(V, device="cuda", generator=g) < 0.5).float() * 5   # two of them
    z[5::9, :] = torch.where(torch.rand(V, device="cuda", generator=g) < 40.0 / V, z[5::9], -math.inf)
    z[6::9, :V // 2] -= 50.0                                                # the better half comes last
    z[7::9, V // 2:V // 2 + 600] += 40.0                                    # all of the best in one place
    z[8::9] = torch.where(torch.rand(V, device="cuda", generator=g) < 0.1, 9.0, z[8::9])  # a long tie at the k-th place
    return z.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,V,k", [(600, 50257, 20), (460, 50257, 256), (460, 151936, 64), (200, 151936, 5),
                                   (9, 151937, 256)])
def test_top_logprobs_of_many_and_long_rows(dtype, N, V, k):
    z = _shapes_of_rows(N, V, dtype)
    ids, lp, lse = ops.top_logprobs(z, k, 0.8)
    s = (V / 256 + 128) * U32  # (as in test_vocab_ops._check_top)
    for a in range(0, N, 100):
        x = z[a:a + 100].double()
        order = torch.sort(x, dim=1, descending=True, stable=True)
        ws = torch.logsumexp(x / 0.8, 1)
        wl = order.values[:, :k] / 0.8 - ws.unsqueeze(1)
        assert torch.equal(ids[a:a + 100], order.indices[:, :k])
        size = ws.abs().unsqueeze(1)
        _close_rows(lp[a:a + 100], wl, s + 4 * U32 * (wl.abs().nan_to_num(posinf=0) + size), "logprobs")
        _close_rows(lse[a:a + 100], ws, s + 4 * U32 * ws.abs(), "lse")


@pytest.mark.parametrize("dtype", DTYPES)
def test_top_logprobs_nan_and_infinity_in_long_rows(dtype):
    z = _rows(450, 50257, dtype, 3)
    z[7, 50256], z[8, 3], z[9, ::2] = math.nan, math.inf, math.nan
    ids, lp, lse = ops.top_logprobs(z, 30)
    for n in (7, 8, 9):
        want = torch.sort(z[n].double(), descending=True, stable=True).indices[:30]
        assert torch.equal(ids[n], want)
        assert n == 8 or (bool(torch.isnan(lp[n]).all()) and bool(torch.isnan(lse[n])))
    others = torch.ones(450, dtype=torch.bool, device="cuda")
    others[7:10] = False
    assert bool(torch.isfinite(lp[others]).all()) and bool(torch.isfinite(lse[others]).all())


# --------------------------------------------------------------------------- control_logits

def _control_case(B, V, L, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    a = {"history": (rand(B, L).pow(3) * (V + 3)).int() - 1}  # ids outside the vocabulary among them
    a["history"][0] %= 5                                      # few tokens, very often
    a["history_lens"] = torch.randint(0, L + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
    a["history_lens"][0] = L
    a["history_lens"][2] = 0
    a["prompt_lens"] = (a["history_lens"] * rand(B)).int()
    a["prompt_lens"][0] = 0
    a["repetition"] = 0.7 + 0.9 * rand(B)
    a["presence"], a["frequency"] = rand(B) - 0.3, rand(B) * 0.01
    a["repetition"][3], a["presence"][3], a["frequency"][3] = 1.0, 0.0, 0.0
    n = 300
    a["bias_offsets"] = torch.arange(B + 1, device="cuda", dtype=torch.int32) * n
    a["bias_ids"] = torch.randint(-1, V + 1, (B * n,), device="cuda", generator=g, dtype=torch.int32)
    a["bias_ids"][n:n + 50] = a["bias_ids"][n + 50:n + 100]  # tokens listed twice
    a["bias_values"] = (rand(B * n) - 0.5) * 8
    words = (V + 31) // 32
    a["mask"] = torch.randint(-2 ** 31, 2 ** 31, (3, words), device="cuda", generator=g).int()
    a["mask"][1], a["mask"][2] = 0, -1
    a["mask_rows"] = (torch.arange(B, device="cuda") % 5 - 2).int().clamp(min=-1)
    return a


def _control_rows(z, a):
    """The definition in fp64 (and the magnitudes that went into each value), a row at a time."""
    out = z.double().clone()
    mag = out.abs()
    V = z.shape[1]
    for b in range(z.shape[0]):
        n, p = int(a["history_lens"][b]), int(a["prompt_lens"][b])
        h = a["history"][b, :n].long()
        ok = (h >= 0) & (h < V)
        seen = torch.bincount(h[ok], minlength=V) > 0
        count = torch.bincount(h[p:][ok[p:]], minlength=V).double()
        r, pr, f = (a[k][b].double() for k in ("repetition", "presence", "frequency"))
        x = out[b]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        less = f * count + pr * (count > 0)
        mag[b] = torch.where(seen, x.abs(), mag[b]) + f.abs() * count + pr.abs() * (count > 0)
        x = x - less
        lo, hi = int(a["bias_offsets"][b]), int(a["bias_offsets"][b + 1])
        ids = a["bias_ids"][lo:hi].long()
        ok = (ids >= 0) & (ids < V)
        vals = a["bias_values"][lo:hi][ok].double()
        x = x.index_add(0, ids[ok], vals)
        mag[b].index_add_(0, ids[ok], vals.abs())
        mr = int(a["mask_rows"][b])
        if mr >= 0:
            v = torch.arange(V, device=z.device)
            x = torch.where(((a["mask"][mr][v // 32] >> (v % 32)) & 1) == 1, x, -math.inf)
        out[b] = x
    return out, mag


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                             (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("B,V,L,layout", [(100, 151936, 100, "dense"), (100, 151936, 40000, "dense"),
                                          (50, 151937, 5000, "shifted"), (50, 151936, 33000, "padded"),
                                          (450, 32771, 700, "dense")])
def test_control_logits_of_large_batches(dtype, out_dtype, B, V, L, layout):
    z = _view(_rows(B, V, dtype, V + L), layout)
    a = _control_case(B, V, L, B + L)
    want, mag = _control_rows(z, a)
    # a division or product, two subtractions and the biases' sum: at most 8 roundings of the magnitudes involved
    tol = 8 * U32 * mag + (U16 * want.abs().nan_to_num(posinf=0) if out_dtype == torch.bfloat16 else 0.0)
    dev = torch.device("cuda", torch.cuda.current_device())
    ops.check_kernel_errors(dev)
    out = ops.control_logits(z, out=torch.full((B, V), math.nan, dtype=out_dtype, device="cuda"), **a)
    ops.check_kernel_errors(dev)
    _close_rows(out, want, tol, "control_logits")
    if dtype == out_dtype:
        assert ops.control_logits(z, out=z, **a) is z
        _close_rows(z, want, tol, "control_logits in place")


# --------------------------------------------------------------------------- distillation

def _distill_definition(z, ids, lps, div, beta, tail, T):
    """Losses and log softmax of fp64 rows, differentiable, from the definition over buckets."""
    N, V = z.shape
    logq = torch.log_softmax(z / T, 1)
    listed = torch.zeros(N, V + 1, dtype=torch.bool, device=z.device).scatter_(1, torch.where(ids < 0, V, ids), True)
    listed = listed[:, :V]
    rest = torch.logsumexp(torch.where(listed, -math.inf, logq), 1, keepdim=True)
    on = ids >= 0
    lq = torch.cat([torch.where(on, logq.gather(1, ids.clamp(min=0)), 0.0), rest], 1)
    lp = torch.where(on, lps.double(), -math.inf)
    mass = lp.exp().sum(1, keepdim=True)
    if tail == "drop":
        lp, last = lp - mass.log(), torch.full_like(mass, -math.inf)
    else:
        last = (1 - mass).clamp(min=2.0 ** -24).log()
    lp = torch.cat([lp, last], 1)
    p, some = lp.exp(), torch.cat([on, torch.ones_like(on[:, :1])], 1)
    lp = torch.where(p > 0, lp, 0.0)
    q = torch.where(some, lq.exp(), 0.0)
    if div == "forward":
        terms = p * (lp - lq)
    elif div == "reverse":
        terms = torch.where(some, q * (lq - lp), 0.0)
    else:
        lm = torch.where(some, beta * p + (1 - beta) * q, 1.0).log()
        terms = torch.where(some, beta * p * (lp - lm) + (1 - beta) * q * (lq - lm), 0.0)
    return torch.where(on.any(1), terms.sum(1), 0.0), logq, listed, p, lp, q.detach(), lq.detach()


def _check_distill_rows(N, V, dtype, K, div, tail, targets, seed, step=64):
    T, beta = 0.8, 0.3
    z = _rows(N, V, dtype, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    teach = (z.float() + torch.randn(N, V, device="cuda", generator=g)) / T
    top = teach.topk(K, 1)
    ids, lps = top.indices, (top.values - torch.logsumexp(teach, 1, keepdim=True)).float()
    cut = torch.randint(1, K + 1, (N,), device="cuda", generator=g)
    cut[0] = K
    if N > 1:
        cut[1] = 0
    ids.masked_fill_(torch.arange(K, device="cuda") >= cut.unsqueeze(1), -1)
    del teach, top
    tg = torch.randint(0, V, (N,), device="cuda", generator=g)
    tg[0] = ids[0, 0]
    tg[N - 1] = V - 1
    up, up_lp = torch.randn(N, device="cuda", generator=g), torch.randn(N, device="cuda", generator=g)
    kw = dict(divergence=div, beta=beta, tail=tail, temperature=T)
    x = z.clone().requires_grad_(True)
    if targets:
        loss, logp = ops.distill_loss(x, ids, lps, targets=tg, **kw)
        (grad,) = torch.autograd.grad((loss, logp), x, (up, up_lp))
    else:
        loss, logp = ops.distill_loss(x, ids, lps, **kw), None
        (grad,) = torch.autograd.grad(loss, x, up)
    loss = loss.detach()
    one_loss, one_grad = ops.distill_loss_grad(z, ids, lps, **kw)
    held = z.clone()
    in_loss, in_grad = ops.distill_loss_grad(held, ids, lps, out=held, **kw)
    assert in_grad is held and torch.equal(in_loss, one_loss) and torch.equal(held, one_grad)
    delta = (V / 256 + 128) * U32  # the unlisted tokens' sum, as in test_vocab_ops._grad_limit
    half = U16 if dtype == torch.bfloat16 else 0.0
    for a in range(0, N, step):
        b = slice(a, min(N, a + step))
        y = z[b].double().requires_grad_(True)
        wl, logq, listed, p, lp, q, lq = _distill_definition(y, ids[b], lps[b], div, beta, tail, T)
        (unit,) = torch.autograd.grad(wl.sum(), y, retain_graph=True)
        wl = wl.detach()
        soft = logq.detach().exp()
        if div == "forward":
            at_rest = p[:, -1:] / q[:, -1:]
            spread = soft * (1 + at_rest)
            extra = soft.gather(1, ids[b].clamp(min=0)) + p[:, :-1]
        else:
            h = (lq - lp).abs()
            h[:, -1:] = torch.where(p[:, -1:] > 0, h[:, -1:], lq[:, -1:].abs() + 30 * math.log(10))
            mean = (q * h).sum(1, keepdim=True)
            spread = soft * (1 + h[:, -1:] + mean)
            extra = soft.gather(1, ids[b].clamp(min=0)) * (1 + h[:, :-1] + mean)
        wide = torch.zeros(spread.shape[0], V + 1, dtype=torch.float64, device="cuda")
        wide.scatter_(1, torch.where(ids[b] < 0, V, ids[b]), extra)
        spread = torch.where(listed, wide[:, :V], spread)
        loss_lim = 4 * delta * spread.sum(1) + 4 * U32 * wl.abs()
        _close_rows(loss[b], wl, loss_lim, "loss")
        _close_rows(one_loss[b], wl, loss_lim, "loss, one pass")
        lim = 4 * delta * spread / T + (300 * U32 + half) * unit.abs() + 1e-37
        _close_rows(one_grad[b], unit, lim, "gradient, one pass")
        want = unit * up[b].double().unsqueeze(1)
        lim = 4 * delta * spread * up[b].abs().double().unsqueeze(1) / T
        if targets:
            wp = logq.gather(1, tg[b].unsqueeze(1)).squeeze(1)
            (dl,) = torch.autograd.grad((wp * up_lp[b].double()).sum(), y)
            want = want + dl
            lim = lim + 4 * delta * (1 + soft) * up_lp[b].abs().double().unsqueeze(1) / T
            _close_rows(logp[b].detach(), wp.detach(), delta + 4 * U32 * wp.detach().abs(), "logprob")
        _close_rows(grad[b], want, lim + (300 * U32 + half) * want.abs() + 1e-37, "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("div,tail", [("forward", "bucket"), ("reverse", "bucket"), ("js", "drop")])
@pytest.mark.parametrize("N,V,K", [(2, 151936, 20), (3, 151937, 256), (300, 50257, 64), (1300, 50257, 16)])
def test_distill_of_many_and_long_rows(dtype, div, tail, N, V, K):
    _check_distill_rows(N, V, dtype, K, div, tail, True, N + K)


@pytest.mark.parametrize("V,dtype", [(600_001, torch.float32), (800_003, torch.float32), (1_570_001, torch.bfloat16)])
def test_distill_of_rows_at_the_limit_of_a_cluster(V, dtype):
    """16 CTAs hold 600 thousand fp32 tokens; the other two rows take the two-pass form."""
    _check_distill_rows(3, V, dtype, 12, "forward", "bucket", False, 5)
