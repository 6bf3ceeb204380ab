"""Embedding, router, expert plan, dispatch and combine against their definitions in 64 bits, on the CPU and on the GPU.

Tolerances count roundings: u = 2^-24 for each fp32 operation, half a step of the result's type for its one rounding.
A sum of n terms in fp32, in any order, is off by at most n u times the sum of the terms' magnitudes."""

import pytest
import torch

import rows_oracle as oracle
from libra_b200 import ops

U = 2.0 ** -24
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.bfloat16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _close(got, want, tol):
    """|got - want| <= tol element by element (tol a tensor or a number), NaN nowhere."""
    err = (got.detach().cpu().double() - want).abs()
    over = err - (tol if torch.is_tensor(tol) else torch.full_like(want, tol))
    assert got.shape == want.shape
    assert not torch.isnan(err).any()
    assert (over <= 0).all(), f"off by {float(err.max()):.3g}, {float(over.max()):.3g} more than allowed"


def _check(device):
    if device == "cuda":
        torch.cuda.synchronize()
        ops.check_kernel_errors()


# ------------------------------------------------------------------ embedding

def _tokens(n, vocab, gen, kind):
    if kind == "same":
        return torch.full((n,), vocab // 2)
    t = torch.randint(0, vocab, (n,), generator=gen)
    if kind == "few":
        t = torch.where(torch.rand(n, generator=gen) < 0.6, torch.full_like(t, vocab // 3), t)
    return t


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,H,kind,scale", [
    (1, 1, 8, "any", 1.0), (1, 151936, 16, "any", 1.0), (17, 7, 1, "any", 3.3), (33, 1000, 13, "few", 1.0),
    (300, 1023, 64, "same", 0.7), (300, 1024, 40, "few", 22.6), (2049, 5000, 24, "few", 1.0), (65, 3, 2560, "any", 1.0),
    (4100, 2, 9, "any", 1.0), (500, 200, 1032, "few", 1.0), (40, 1 << 20, 8, "any", 1.0), (0, 10, 8, "any", 1.0)])
def test_embedding_and_gradient(device, dtype, n, vocab, H, kind, scale):
    gen = _gen(n + vocab + H)
    tokens = _tokens(n, vocab, gen, kind)
    w = torch.randn(vocab, H, generator=gen).to(dtype)
    g = torch.randn(n, H, generator=gen).to(dtype)
    wd = w.to(device).requires_grad_(True)
    out = ops.embedding(tokens.to(device), wd, scale=scale)
    assert out.dtype == dtype
    want = oracle.embedding(tokens, w, scale)
    # the scale's own rounding, the product's, the result's (none of them for scale 1)
    _close(out, want, 0.0 if scale == 1.0 else want.abs() * (2.1 * U + _half(dtype)))
    (dw,) = torch.autograd.grad(out, wd, g.to(device))
    assert dw.dtype == dtype
    total, size, many = oracle.embedding_grad(tokens, g, vocab, scale)
    # n terms, the scale and its product; the result's rounding
    _close(dw, total, size * (many + 2) * U * 1.01 + total.abs() * _half(dtype) * 1.01)
    _check(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_embedding_adds_to_main_grad(device, index):
    gen = _gen(3)
    tokens = _tokens(700, 90, gen, "few").view(7, 100).to(index)
    w = torch.randn(90, 48, generator=gen).bfloat16()
    g = torch.randn(7, 100, 48, generator=gen).bfloat16()
    wd = w.to(device).requires_grad_(True)
    base = torch.randn(90, 48, generator=gen)
    wd.main_grad = base.clone().to(device)
    total, size, many = oracle.embedding_grad(tokens, g, 90, 1.0)
    for step in (1, 2):
        out = ops.embedding(tokens.to(device), wd)
        assert out.shape == (7, 100, 48)
        out.backward(g.to(device))
        assert wd.grad is None
        want = base.double() + step * total
        tol = step * (size * many * U + (size + base.abs().double()) * U) * 1.01
        _close(wd.main_grad, want, tol)
    untouched = many.squeeze(1) == 0
    assert torch.equal(wd.main_grad.cpu()[untouched], base[untouched])
    _check(device)


@pytest.mark.parametrize("device", DEVICES)
def test_embedding_shards_add_up_and_leave_other_tokens_out(device):
    gen = _gen(4)
    tokens = torch.randint(0, 100, (257,), generator=gen)
    w = torch.randn(100, 32, generator=gen)
    g = torch.randn(257, 32, generator=gen)
    outs, grads = [], []
    for lo, hi in ((0, 30), (30, 31), (31, 100)):
        shard = w[lo:hi].to(device).requires_grad_(True)
        out = ops.embedding(tokens.to(device), shard, vocab_start=lo)
        grads.append(torch.autograd.grad(out, shard, g.to(device))[0])
        outs.append(out.detach())
    _close(sum(outs), oracle.embedding(tokens, w, 1.0), 0.0)  # one of three terms is not zero
    total, size, many = oracle.embedding_grad(tokens, g, 100, 1.0)
    _close(torch.cat(grads), total, size * (many + 1) * U * 1.01)
    far = torch.tensor([-1, 2 ** 40, -2 ** 40, 100])
    shard = w.to(device).requires_grad_(True)
    out = ops.embedding(far.to(device), shard, vocab_start=0)
    assert not out.any() and not torch.autograd.grad(out.sum(), shard)[0].any()
    _check(device)


@pytest.mark.parametrize("device", DEVICES)
def test_vocab_parallel_embedding_of_one_rank_at_a_time(device):
    """The tensor-parallel lookup on each rank's shard, without the reduction: partial rows and the shards' gradients."""
    from libra_b200.parallel.tensor_parallel import vocab_parallel_embedding

    gen = _gen(14)
    tokens = _tokens(130, 64, gen, "few")
    w, g = torch.randn(64, 24, generator=gen).bfloat16(), torch.randn(130, 24, generator=gen).bfloat16()
    total, size, many = oracle.embedding_grad(tokens, g, 64, 1.0)
    whole = 0
    for rank in range(4):
        shard = w[16 * rank:16 * (rank + 1)].clone().to(device).requires_grad_(True)
        shard.main_grad = torch.zeros(16, 24, device=device) if rank % 2 else None
        out = vocab_parallel_embedding(tokens.to(device), shard, None, rank, reduce=False)
        out.backward(g.to(device))
        rows = slice(16 * rank, 16 * (rank + 1))
        got = shard.main_grad if rank % 2 else shard.grad
        _close(got, total[rows], size[rows] * (many[rows] + 1) * U * 1.01
               + (0 if rank % 2 else total[rows].abs() * _half(torch.bfloat16) * 1.01))
        whole = whole + out.detach()
    _close(whole, oracle.embedding(tokens, w, 1.0), 0.0)
    _check(device)


def test_embedding_refusals_on_the_cpu():
    w = torch.zeros(4, 8)
    for bad in (-1, 4):
        with pytest.raises(ValueError, match="outside the table"):
            ops.embedding(torch.tensor([0, bad]), w)
    with pytest.raises(ValueError, match="int64 or int32"):
        ops.embedding(torch.tensor([0.0]), w)
    with pytest.raises(ValueError, match="of floats"):
        ops.embedding(torch.tensor([0]), w.long())
    with pytest.raises(ValueError, match=r"\[V, H\]"):
        ops.embedding(torch.tensor([0]), w[0])
    with pytest.raises(ValueError, match="contiguous"):
        ops.embedding(torch.tensor([0]), torch.zeros(8, 4).t())


@pytest.mark.gpu
def test_embedding_reports_tokens_outside_the_table():
    w = torch.ones(4, 8, device="cuda", requires_grad=True)
    for bad in (-1, 4, 2 ** 40):
        out = ops.embedding(torch.tensor([1, bad, 3], device="cuda"), w)
        with pytest.raises(ops.KernelError):
            ops.check_kernel_errors()
        assert out.sum(1).tolist() == [8.0, 0.0, 8.0]
        (dw,) = torch.autograd.grad(out.sum(), w)
        assert dw.sum(1).tolist() == [0.0, 8.0, 0.0, 8.0]
    _check("cuda")
    with pytest.raises(ValueError, match="tokens must be"):
        ops.embedding(torch.tensor([0]), w)


@pytest.mark.gpu
@pytest.mark.parametrize("n,H", [(20000, 520), (3000, 33)])
def test_embedding_gradient_of_strided_and_expanded_rows_is_the_same_every_time(n, H):
    gen = _gen(n)
    tokens = _tokens(n, 500, gen, "few").cuda()
    table = torch.randn(500, H + 24, generator=gen).bfloat16().cuda()
    w = table[:, :H].detach().requires_grad_(True)  # rows further apart than they are wide
    assert w.stride(0) == H + 24
    out = ops.embedding(tokens, w)
    assert torch.equal(out, w.detach()[tokens])
    wide = torch.randn(n, H + 8, generator=gen).bfloat16().cuda()
    for g in (wide[:, :H], wide[:, 3:H + 3], wide[:1, :H].expand(n, H), wide[:, :1].expand(n, H)):
        first = torch.autograd.grad(out, w, g, retain_graph=True)[0]
        total, size, many = oracle.embedding_grad(tokens.cpu(), g.cpu(), 500, 1.0)
        _close(first, total, size * many * U * 1.01 + total.abs() * _half(torch.bfloat16) * 1.01)
        for _ in range(3):
            assert torch.equal(torch.autograd.grad(out, w, g, retain_graph=True)[0], first)
    _check("cuda")


def _grad64(tokens, g, rows):
    """As oracle.embedding_grad, without a loop."""
    g = g.double()
    total = torch.zeros(rows, g.shape[1], dtype=torch.float64).index_add_(0, tokens, g)
    size = torch.zeros_like(total).index_add_(0, tokens, g.abs())
    return total, size, torch.bincount(tokens, minlength=rows).double().unsqueeze(1)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 65, 1024, 1025, 8192, 16384, 16385, 40000])
@pytest.mark.parametrize("run", [1, 2, 15, 16, 17, 32, 33, 64, 65, 97, 1000])
def test_embedding_gradient_of_runs_that_end_anywhere(n, run):
    """Every token occurs `run` times (the last one less often), shuffled: sums that lie in one chunk of the sorted
    tokens, in two, or in many, with borders at every offset."""
    gen = _gen(n + run)
    tokens = (torch.arange(n) // run + 3)[torch.randperm(n, generator=gen)]
    rows = int(tokens.max()) + 5
    for H, dtype in ((40, torch.bfloat16), (12, torch.float32), (7, torch.float32)):
        w = torch.zeros(rows, H, dtype=dtype, device="cuda", requires_grad=True)
        g = torch.randn(n, H, generator=gen).to(dtype)
        total, size, many = _grad64(tokens, g, rows)
        for main in (None, torch.randn(rows, H, generator=gen)):
            w.main_grad = None if main is None else main.clone().cuda()
            out = ops.embedding(tokens.cuda(), w)
            w.grad = None
            out.backward(g.cuda())
            if main is None:
                _close(w.grad, total, size * many * U * 1.01 + total.abs() * _half(dtype) * 1.01)
            else:
                assert w.grad is None
                _close(w.main_grad, main.double() + total, (size * (many + 1) + main.abs().double()) * U * 1.01)
    _check("cuda")


@pytest.mark.gpu
def test_embedding_looked_up_twice_and_backward_twice():
    gen = _gen(5)
    a, b = torch.randint(0, 30, (100,), generator=gen), torch.randint(0, 30, (70,), generator=gen)
    ga, gb = torch.randn(100, 16, generator=gen), torch.randn(70, 16, generator=gen)
    w = torch.randn(30, 16, generator=gen).cuda().requires_grad_(True)
    total, size, many = _grad64(torch.cat([a, b]), torch.cat([ga, gb]), 30)
    for main in (False, True):
        w.grad = None
        w.main_grad = torch.zeros(30, 16, device="cuda") if main else None
        outs = [ops.embedding(a.cuda(), w), ops.embedding(b.cuda(), w)]
        for times in (1, 2):
            torch.autograd.backward(outs, [ga.cuda(), gb.cuda()], retain_graph=True)
            _close(w.main_grad if main else w.grad, times * total, times * size * (many + 2) * U * 1.01)
    with torch.no_grad():
        w.add_(1.0)  # an optimizer step between the passes: the gradient does not need the table's values
    torch.autograd.backward(outs, [ga.cuda(), gb.cuda()])
    _close(w.main_grad, 3 * total, 3 * size * (many + 2) * U * 1.01)


# ------------------------------------------------------------------ router

def _logits(n, E, gen, dtype):
    z = (torch.randn(n, E, generator=gen) * 2).to(dtype)
    if n > 4 and E > 2:
        z[1] = 0.5                              # all tied
        z[2, ::2] = float("-inf")               # half masked
        z[3] = float("-inf")                    # nothing left
        z[4] = torch.finfo(dtype).min           # a mask of the type's lowest value
        z[4, E // 2] = 1.0
    return z


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("n,E,k", [(1, 1, 1), (9, 8, 2), (33, 31, 3), (64, 128, 8), (7, 33, 32), (40, 200, 5),
                                   (10, 512, 32), (11, 1000, 17), (0, 8, 2), (6, 60, 4),
                                   (8, 100, 100), (6, 300, 33)])
def test_route_and_gradient(device, dtype, normalize, n, E, k):
    gen = _gen(n * E + k)
    z = _logits(n, E, gen, dtype)
    g = torch.randn(n, k, generator=gen)
    zd = z.to(device).requires_grad_(True)
    w, ids = ops.route_topk(zd, k, normalize=normalize)
    assert w.dtype == torch.float32 and ids.dtype == torch.int64
    want, order = oracle.route(z, k, normalize)
    assert torch.equal(ids.cpu(), order)
    # exponents: the difference's rounding moves exp by |z - top| u (a float of at most 90, beyond it the weight is
    # below 1e-39), exp itself is good to 2 u; a sum of E such terms, and a division
    tol = (90 + 4 + E + 2) * U
    _close(w, want, want * tol + 1e-38)
    with torch.no_grad():
        again = ops.route_topk(z.to(device), k, normalize=normalize)
    assert torch.equal(again[0], w) and torch.equal(again[1], ids)
    (dz,) = torch.autograd.grad(w, zd, g.to(device))
    assert dz.dtype == dtype
    exact = oracle.route_grad(z, order, g, normalize)
    # each term is a product of weights that are off by tol and g; the sum over k of them
    scale = (want * g.abs().double()).sum(1, keepdim=True) + g.abs().double().amax(1, keepdim=True) if n else 0.0
    _close(dz, exact, scale * (2 * tol + (k + 3) * U) + exact.abs() * _half(dtype) * 1.01 if n else 0.0)
    _check(device)


@pytest.mark.parametrize("device", DEVICES)
def test_route_with_infinities_and_nan(device):
    inf, nan = float("inf"), float("nan")
    z = torch.tensor([[0.0, nan, 1.0, 2.0], [inf, 0.0, 1.0, -inf], [-0.0, 0.0, -inf, -inf], [nan, nan, inf, 1.0]])
    w, ids = ops.route_topk(z.to(device), 3)
    assert ids.tolist() == [[1, 3, 2], [0, 2, 1], [0, 1, 2], [0, 1, 2]]
    w = w.cpu()
    assert torch.isnan(w[0]).all() and torch.isnan(w[1]).any() and torch.isnan(w[3]).all()
    assert w[2].tolist() == [0.5, 0.5, 0.0]
    # a large gradient beside a weight of zero, and logits far apart
    z = torch.tensor([[100.0, -100.0, -inf]], device=device, requires_grad=True)
    w, _ = ops.route_topk(z, 3)
    (dz,) = torch.autograd.grad(w, z, torch.tensor([[1.0, 1e30, 1e30]], device=device))
    assert torch.isfinite(dz).all() and dz[0, 2] == 0
    _check(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_against_differences(device, normalize):
    gen = _gen(8)
    z = torch.randn(5, 12, generator=gen)
    g = torch.randn(5, 3, generator=gen)
    zd = z.to(device).requires_grad_(True)
    w, ids = ops.route_topk(zd, 3, normalize=normalize)
    (dz,) = torch.autograd.grad(w, zd, g.to(device))
    step = 2.0 ** -7
    for e in range(12):
        up, down = z.clone(), z.clone()
        up[:, e] += step
        down[:, e] -= step
        hi, ih = ops.route_topk(up.to(device), 3, normalize=normalize)
        lo, il = ops.route_topk(down.to(device), 3, normalize=normalize)
        same = ((ih == ids) & (il == ids)).all(1).cpu()  # the choice did not change
        diff = ((hi - lo).cpu() * g).sum(1) / (2 * step)
        # third derivatives of a softmax are below 1: step^2 / 6 times the gradients; 40 u a weight over the step
        bound = g.abs().sum(1) * (step ** 2 / 6 + 40 * U / step)
        assert ((diff - dz[:, e].cpu()).abs()[same] <= bound[same]).all()


def test_route_refusals():
    z = torch.zeros(2, 8)
    for k in (0, 9, -1):
        with pytest.raises(ValueError, match="k in"):
            ops.route_topk(z, k)
    with pytest.raises(ValueError, match="1 to 1024 experts"):
        ops.route_topk(torch.zeros(2, 1025), 2)
    for bad in (z[0], z.long()):
        with pytest.raises(ValueError, match="route_topk"):
            ops.route_topk(bad, 2)


@pytest.mark.gpu
def test_route_of_strided_logits():
    z = torch.randn(50, 3, 40, generator=_gen(1)).cuda()
    for view in (z[:, 1], z[:, :, 5], z[::2, 0, 1:]):
        got, want = ops.route_topk(view, 3), ops.route_topk(view.contiguous(), 3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------ plan, dispatch, combine

def _experts(n, k, E, gen, kind):
    if kind == "one":
        return torch.full((n, k), E - 1)
    ids = torch.randint(0, E, (n, k), generator=gen)
    if kind == "gaps":  # padding tokens, a slot without an expert, experts that nobody chose
        ids = ids // 2 * 2
        ids[torch.rand(n, k, generator=gen) < 0.2] = -1
        ids[n // 2:n // 2 + 2] = -5
    return ids


SIZES = [(1, 1, 1, "any", 128), (1, 8, 128, "any", 128), (37, 2, 8, "any", 128), (300, 3, 5, "gaps", 16),
         (64, 8, 128, "any", 128), (257, 4, 60, "gaps", 1), (700, 6, 256, "any", 128), (50, 2, 1024, "gaps", 7),
         (1200, 2, 3, "one", 128), (40, 1, 300, "any", 64), (0, 2, 4, "any", 128), (9, 3, 1, "any", 128)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("n,k,E,kind,align", SIZES)
def test_plan(device, index, n, k, E, kind, align):
    ids = _experts(n, k, E, _gen(n + E), kind).to(index)
    plan = ops.expert_plan(ids.to(device), E, align=align)
    rows, offs, counts = oracle.plan(ids, E, align)
    assert plan.rows.tolist() == rows and plan.offs.tolist() == offs and plan.counts.tolist() == counts
    assert plan.rows.dtype == plan.offs.dtype == plan.counts.dtype == torch.int32
    assert offs[-1] <= plan.capacity
    _check(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,E,kind,align,H", [s + (h,) for i, s in enumerate(SIZES)
                                                for h in ((1, 24, 33) if s[0] < 100 else (24 + i % 2,))])
def test_dispatch_and_combine_with_gradients(device, dtype, n, k, E, kind, align, H):
    gen = _gen(n + E + H)
    ids = _experts(n, k, E, gen, kind)
    plan = ops.expert_plan(ids.to(device), E, align=align)
    rows, _, _ = oracle.plan(ids, E, align)
    cap = plan.capacity

    def rand(*shape, t=dtype):
        return torch.randn(*shape, generator=gen).to(t)

    x, gx = rand(n, H), rand(cap, H)
    xd = x.to(device).requires_grad_(True)
    xs = ops.moe_dispatch(xd, plan)
    _close(xs, oracle.dispatch(x, rows, k, cap), 0.0)
    assert xs.dtype == dtype
    (dx,) = torch.autograd.grad(xs, xd, gx.to(device))
    want, size = oracle.combine(gx, None, rows, k, None, n)
    _close(dx, want, size * k * U * 1.01 + want.abs() * _half(dtype) * 1.01)

    y, w, res, g = rand(cap, H), rand(n, k, t=torch.float32), rand(n, H), rand(n, H)
    if device == "cuda":  # whatever lies in rows that are no pair's has no effect
        live = torch.zeros(cap, dtype=torch.bool)
        live[[r for r in rows if r >= 0]] = True
        y[~live] = float("nan")
    yd, wd, rd = (t.to(device).requires_grad_(True) for t in (y, w, res))
    for with_res in (True, False):
        out = ops.moe_combine(yd, wd, plan, residual=rd if with_res else None)
        want, size = oracle.combine(y, w, rows, k, res if with_res else None, n)
        _close(out, want, size * (k + 2) * U * 1.01 + want.abs() * _half(dtype) * 1.01)
        assert out.dtype == dtype
        grads = torch.autograd.grad(out, (yd, wd, rd) if with_res else (yd, wd), g.to(device))
        dy, dw, size = oracle.combine_grad(g, y, w, rows, k)
        _close(grads[0], dy, dy.abs() * (U + _half(dtype)) * 1.01)
        _close(grads[1], dw, size * (H + 1) * U * 1.01)
        if with_res:
            assert torch.equal(grads[2].cpu(), g)
    _check(device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_moves_of_strided_rows_and_parts_of_the_gradients(dtype):
    gen = _gen(6)
    n, k, E, H = 130, 3, 9, 64
    ids = _experts(n, k, E, gen, "gaps").cuda()
    plan = ops.expert_plan(ids, E, align=8)
    wide = torch.randn(max(n, plan.capacity), 2 * H + 5, generator=gen).to(dtype).cuda()
    w = torch.rand(n, k, generator=gen).cuda()
    for a, b in ((0, H), (3, H + 3), (8, 2 * H + 5)):  # aligned, unaligned, odd width
        x, y, r = wide[:n, a:b], wide[:plan.capacity, a:b], wide[:n, a:b]
        assert torch.equal(ops.moe_dispatch(x, plan), ops.moe_dispatch(x.contiguous(), plan))
        want = ops.moe_combine(y.contiguous(), w, plan, residual=r.contiguous())
        assert torch.equal(ops.moe_combine(y, w, plan, residual=r), want)
        assert torch.equal(ops.moe_combine(y.t().contiguous().t(), w.t().contiguous().t(), plan, residual=r), want)
        leaves = [t.detach().clone().requires_grad_(True) for t in (y, w, r)]
        full = torch.autograd.grad(ops.moe_combine(*leaves[:2], plan, residual=leaves[2]).sum(), leaves)
        for i in range(3):  # one of them alone
            alone = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
            out = ops.moe_combine(*alone[:2], plan, residual=alone[2])
            assert torch.equal(torch.autograd.grad(out.sum(), alone[i])[0], full[i])
    _check("cuda")


def test_plan_and_move_refusals():
    ids = torch.tensor([[0, 1], [2, 3]])
    with pytest.raises(ValueError, match="not below num_experts"):
        ops.expert_plan(ids, 3)
    for bad in (ids[0], ids.float(), ids[:, :0]):
        with pytest.raises(ValueError, match="expert_plan"):
            ops.expert_plan(bad, 4)
    for E, align in ((0, 1), (1025, 1), (4, 0)):
        with pytest.raises(ValueError, match="align >= 1"):
            ops.expert_plan(ids, E, align=align)
    with pytest.raises(ValueError, match="31 bits"):
        ops.expert_plan(ids, 4, align=2 ** 30)
    plan = ops.expert_plan(ids, 4, align=2)
    x, w = torch.zeros(2, 8), torch.ones(2, 2)
    y = ops.moe_dispatch(x, plan)
    assert y.shape == (plan.capacity, 8)
    for bad in (torch.zeros(3, 8), torch.zeros(2, 8).long(), torch.zeros(2)):
        with pytest.raises(ValueError, match="moe_dispatch"):
            ops.moe_dispatch(bad, plan)
    with pytest.raises(ValueError, match="moe_combine: y"):
        ops.moe_combine(y[1:], w, plan)
    with pytest.raises(ValueError, match="weights"):
        ops.moe_combine(y, w[:, :1], plan)
    for bad in (torch.zeros(2, 7), torch.zeros(2, 8).bfloat16()):
        with pytest.raises(ValueError, match="residual"):
            ops.moe_combine(y, w, plan, residual=bad)


@pytest.mark.gpu
def test_plan_reports_ids_beyond_the_experts():
    plan = ops.expert_plan(torch.tensor([[0, 4], [2 ** 40, 1]], device="cuda"), 4, align=1)
    with pytest.raises(ops.KernelError):
        ops.check_kernel_errors()
    assert plan.rows.tolist() == [0, -1, -1, 1] and plan.counts.tolist() == [1, 1, 0, 0]
    _check("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,E,align", [(16384, 8, 128, 128), (8193, 1, 512, 128), (40000, 8, 513, 16),
                                         (20000, 4, 1024, 1), (100001, 3, 1, 128), (1, 8, 1024, 128), (5000, 7, 37, 3)])
def test_plan_of_many_pairs(n, k, E, align):
    gen = _gen(n + E)
    ids = (torch.rand(n, k, generator=gen).pow(2) * E).long()
    ids[torch.rand(n, k, generator=gen) < 0.01] = -1
    flat = ids.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=E)
    padded = (counts + align - 1) // align * align
    start = padded.cumsum(0) - padded
    order = torch.argsort(torch.where(flat >= 0, flat, E), stable=True)[:int(counts.sum())]
    rows = torch.full_like(flat, -1)
    rows[order] = torch.arange(order.numel()) - (counts.cumsum(0) - counts)[flat[order]] + start[flat[order]]
    plan = ops.expert_plan(ids.cuda(), E, align=align)
    assert torch.equal(plan.rows.cpu().long(), rows) and torch.equal(plan.counts.cpu().long(), counts)
    assert torch.equal(plan.offs.cpu().long(), torch.cat([start, padded.sum()[None] if E else start]))
    _check("cuda")


# ------------------------------------------------------------------ together

def _block(h, logits, res, plan_of):
    w, ids = ops.route_topk(logits, 2)
    plan = plan_of(ids)
    xs = ops.moe_dispatch(h, plan)
    ys = xs * torch.arange(1, 1 + xs.shape[0], device=h.device).remainder(5).to(h.dtype).unsqueeze(1)
    return ops.moe_combine(ys, w, plan, residual=res)


@pytest.mark.parametrize("device", DEVICES)
def test_routed_block_against_differences(device):
    """Router, plan, dispatch, combine and their gradients in one block: directional differences."""
    gen = _gen(11)
    n, E, H = 21, 6, 10
    base = [torch.randn(n, H, generator=gen), torch.randn(n, E, generator=gen) * 3, torch.randn(n, H, generator=gen)]
    g = torch.randn(n, H, generator=gen)
    leaves = [t.to(device).requires_grad_(True) for t in base]

    def plan_of(ids):
        return ops.expert_plan(ids, E, align=4)

    grads = torch.autograd.grad(_block(*leaves, plan_of), leaves, g.to(device))
    step = 2.0 ** -8
    for i in range(3):
        d = torch.randn(base[i].shape, generator=gen)
        hi, lo = ([t.to(device) if j != i else (t + s * d).to(device) for j, t in enumerate(base)]
                  for s in (step, -step))
        if i == 1:
            with torch.no_grad():
                assert torch.equal(ops.route_topk(hi[1], 2)[1], ops.route_topk(lo[1], 2)[1])
        diff = ((_block(*hi, plan_of) - _block(*lo, plan_of)).cpu().double() * g).sum() / (2 * step)
        slope = (grads[i].cpu().double() * d).sum()
        # outputs reach 4 * 4 a term: 40 u of them over the step, for n * H terms of g; the curvature of the weights
        size = float(g.abs().sum()) * 16
        assert abs(float((diff - slope).detach())) <= size * (40 * U / step + (step ** 2) * 8)
    _check(device)


@pytest.mark.gpu
def test_block_in_a_captured_graph_and_on_another_stream():
    gen = _gen(12)
    n, E, H = 300, 16, 256
    h, z, res = (torch.randn(n, w, generator=gen).cuda() for w in (H, E, H))
    tokens = torch.randint(0, 50, (n,), generator=gen).cuda()
    table = torch.randn(50, H, generator=gen).cuda()

    def plan_of(ids):
        return ops.expert_plan(ids, E)

    def both():
        with torch.no_grad():
            return _block(h + ops.embedding(tokens, table), z, res, plan_of)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    side.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for s in (1.0, -0.5):
        h.mul_(s)
        z.neg_()
        tokens.copy_(tokens.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, both())
    _check("cuda")


@pytest.mark.gpu
def test_training_block_in_a_captured_graph():
    gen = _gen(13)
    n, E, H = 200, 8, 128
    h, z, res, g = (torch.randn(n, w, generator=gen).cuda() for w in (H, E, H, H))
    tokens = torch.randint(0, 50, (n,), generator=gen).cuda()

    def step(table, main):
        table.main_grad = main
        zl, rl = z.detach().requires_grad_(True), res.detach().requires_grad_(True)
        out = _block(h + ops.embedding(tokens, table), zl, rl, lambda ids: ops.expert_plan(ids, E))
        return (out,) + torch.autograd.grad(out, (zl, rl, table), g, allow_unused=True)[:2]

    table = torch.randn(50, H, generator=gen).cuda().requires_grad_(True)
    main = torch.zeros(50, H, device="cuda")
    want = [t.detach().clone() for t in step(table, main)] + [main.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(table, main)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main.zero_()
        got = step(table, main)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(list(got) + [main], want):
        assert torch.equal(a, b)
    _check("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 33, 300])
def test_moe_block_gradients_match_the_loop(T):
    """The model's block on the row operators against its per-expert loop: outputs and the gradients of tokens, router
    and experts, to a few bf16 roundings (relative, in norm)."""
    from libra_b200.models.moe import moe_mlp, moe_mlp_looped
    from libra_b200.models.qwen3 import get_config

    cfg = get_config("tiny-moe")
    gen = _gen(T)
    H, E, F = cfg.hidden_size, cfg.num_experts, cfg.moe_intermediate_size
    data = [torch.randn(T, H, generator=gen).bfloat16(), torch.randn(T, H, generator=gen).bfloat16(),
            torch.randn(E, H, generator=gen) * 0.05, (torch.randn(E, 2 * F, H, generator=gen) * 0.05).bfloat16(),
            (torch.randn(E, H, F, generator=gen) * 0.05).bfloat16()]
    g = torch.randn(T, H, generator=gen).bfloat16().cuda()
    got = []
    for block in (moe_mlp, moe_mlp_looped):
        leaves = [t.cuda().requires_grad_(True) for t in data]
        out = block(*leaves, cfg)
        got.append([out.detach()] + list(torch.autograd.grad(out, leaves, g)))
    for a, b in zip(*got):
        # gate, up, their product, the expert's output, dy, dgu and dx each round once to bf16 on either side
        assert float((a.double() - b.double()).norm()) <= 2 * 7 * _half(torch.bfloat16) * float(b.double().norm())
    _check("cuda")


@pytest.mark.gpu
def test_refusals_of_cuda_tensors():
    ids = torch.tensor([[0, 1], [2, 3]], device="cuda")
    plan = ops.expert_plan(ids, 4, align=2)
    x, w, z = torch.zeros(2, 8, device="cuda"), torch.ones(2, 2, device="cuda"), torch.zeros(2, 8, device="cuda")
    y = ops.moe_dispatch(x, plan)
    calls = [lambda: ops.embedding(ids, x.half()), lambda: ops.embedding(ids.cpu(), x), lambda: ops.embedding(ids, x[0]),
             lambda: ops.embedding(ids.float(), x), lambda: ops.embedding(ids, torch.zeros(8, 4, device="cuda").t()),
             lambda: ops.route_topk(z.half(), 2), lambda: ops.route_topk(z[0], 1), lambda: ops.route_topk(z, 0),
             lambda: ops.route_topk(z, 9), lambda: ops.route_topk(torch.zeros(2, 1025, device="cuda"), 2),
             lambda: ops.expert_plan(ids[0], 4), lambda: ops.expert_plan(ids.float(), 4),
             lambda: ops.expert_plan(ids, 0), lambda: ops.expert_plan(ids, 1025), lambda: ops.expert_plan(ids, 4, align=0),
             lambda: ops.expert_plan(ids, 4, align=2 ** 30), lambda: ops.moe_dispatch(x[:1], plan),
             lambda: ops.moe_dispatch(x.half(), plan), lambda: ops.moe_dispatch(x.cpu(), plan),
             lambda: ops.moe_combine(y[1:], w, plan), lambda: ops.moe_combine(y, w[:, :1], plan),
             lambda: ops.moe_combine(y, w.cpu(), plan), lambda: ops.moe_combine(y, w, plan, residual=x[:, :7]),
             lambda: ops.moe_combine(y, w, plan, residual=x.bfloat16())]
    for call in calls:
        with pytest.raises(ValueError):
            call()
    _check("cuda")


@pytest.mark.parametrize("device", DEVICES)
def test_moe_block_without_tokens(device):
    from libra_b200.models.moe import moe_mlp
    from libra_b200.models.qwen3 import get_config

    cfg = get_config("tiny-moe")
    H, E, F = cfg.hidden_size, cfg.num_experts, cfg.moe_intermediate_size
    t = torch.bfloat16
    leaves = [torch.zeros(0, H, dtype=t), torch.zeros(0, H, dtype=t), torch.randn(E, H),
              torch.randn(E, 2 * F, H).to(t), torch.randn(E, H, F).to(t)]
    leaves = [x.to(device).requires_grad_(True) for x in leaves]
    out = moe_mlp(*leaves, cfg)
    assert out.shape == (0, H)
    # (the CPU's grouped products leave experts without rows out of the graph)
    for leaf, grad in zip(leaves, torch.autograd.grad(out, leaves, torch.zeros_like(out), allow_unused=device == "cpu")):
        assert grad is None or (grad.shape == leaf.shape and not grad.any())
    _check(device)


def test_doubles_on_the_cpu_keep_their_bits():
    gen = _gen(2)
    w = torch.randn(9, 4, generator=gen, dtype=torch.float64, requires_grad=True)
    tokens = torch.randint(0, 9, (20,), generator=gen)
    assert torch.autograd.gradcheck(lambda t: ops.embedding(tokens, t, scale=1.5), w)
    plan = ops.expert_plan(torch.randint(0, 3, (5, 2), generator=gen), 3, align=4)
    assert torch.autograd.gradcheck(lambda t: ops.moe_dispatch(t, plan),
                                    torch.randn(5, 4, generator=gen, dtype=torch.float64, requires_grad=True))
