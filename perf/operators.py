"""Measured cases of the vocabulary-row operators: logit controls, top logprobs
and distillation from a teacher's top logprobs.

Each case is one pass through one operator of ``libra_b200.ops`` on rows of
vocabulary logits.  ``run`` computes the plain torch form, or with ``own`` set
calls the framework's operator; ``exact`` restates each definition in 64 bits.
"""

import math

import torch

own = False

VOCAB = 151936  # vocabulary of the model configurations
REST_FLOOR = 2.0 ** -24


def listed():
    return [
        # one interactive request in the middle of a chat turn, every control on: the latency of a single row
        {"name": "control-1row", "op": "control", "rows": 1, "vocab": VOCAB, "dtype": "bf16", "history": 700,
         "bias": 16, "mask": True},
        # a decode batch of the rollout engine: ragged histories, a third of the rows under a grammar
        {"name": "control-64rows", "op": "control", "rows": 64, "vocab": VOCAB, "dtype": "bf16", "history": 4096,
         "bias": 64, "mask": True},
        # the engine's largest batch (256 running requests) of long agentic episodes, fp32 logits, penalties only
        {"name": "control-256rows-fp32", "op": "control", "rows": 256, "vocab": VOCAB, "dtype": "fp32",
         "history": 16384, "bias": 0, "mask": False},
        # top five alternatives of a small decode batch (logprobs=5 of a completion request)
        {"name": "top5-16rows", "op": "top", "rows": 16, "vocab": VOCAB, "dtype": "bf16", "k": 5},
        # an odd vocabulary in fp32, the logits of a prompt's positions
        {"name": "top20-500rows-odd", "op": "top", "rows": 500, "vocab": 50257, "dtype": "fp32", "k": 20},
        # a teacher scores one chunk of packed action tokens for distillation
        {"name": "top64-4096rows", "op": "top", "rows": 4096, "vocab": VOCAB, "dtype": "bf16", "k": 64},
        # a small micro-batch, forward KL with its gradient, beside the sampled tokens' logprobs
        {"name": "distill-64rows", "op": "distill", "rows": 64, "vocab": VOCAB, "dtype": "bf16", "k": 16,
         "divergence": "forward", "tail": "bucket", "targets": True},
        # one chunk of a training step: forward KL and GRPO's token logprobs from the same logits
        {"name": "distill-4096rows", "op": "distill", "rows": 4096, "vocab": VOCAB, "dtype": "bf16", "k": 64,
         "divergence": "forward", "tail": "bucket", "targets": True},
        # odd vocabulary, fp32 logits, reverse KL
        {"name": "distill-777rows-odd-fp32", "op": "distill", "rows": 777, "vocab": 50257, "dtype": "fp32", "k": 32,
         "divergence": "reverse", "tail": "bucket", "targets": False},
        # the one-pass form on a short chunk: loss and unit gradient together
        {"name": "distillgrad-128rows", "op": "distill_grad", "rows": 128, "vocab": VOCAB, "dtype": "bf16", "k": 20,
         "divergence": "js", "tail": "bucket", "targets": False},
        # the one-pass form on a full chunk of the LM head's rows
        {"name": "distillgrad-4096rows", "op": "distill_grad", "rows": 4096, "vocab": VOCAB, "dtype": "bf16", "k": 64,
         "divergence": "forward", "tail": "bucket", "targets": False},
        # fp32 logits of a large vocabulary, a wide teacher table without the rest bucket
        {"name": "distillgrad-1000rows-fp32", "op": "distill_grad", "rows": 1000, "vocab": VOCAB, "dtype": "fp32",
         "k": 128, "divergence": "forward", "tail": "drop", "targets": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["control", "top", "distill", "distill_grad"])
    vocab = VOCAB if rng.random() < 0.4 else _log_int(rng, 1000, 200_000)
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "control":
        rows = _log_int(rng, 1, max(1, min(256, 256 * VOCAB // vocab // (1 if dtype == "fp32" else 2))))
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "history": _log_int(rng, 1, 12000),
                "bias": rng.choice([0, 1, 7, 300]), "mask": rng.random() < 0.6}
    rows = _log_int(rng, 1, max(2, min(6000, 2000 * VOCAB // vocab // (2 if dtype == "fp32" else 1))))
    k = min(_log_int(rng, 1, 128), vocab)
    if op == "top":
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "k": k}
    div = rng.choice(["forward", "reverse", "js"])
    tail = "bucket" if div == "reverse" else rng.choice(["bucket", "bucket", "drop"])
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "divergence": div, "tail": tail,
            "targets": op == "distill" and rng.random() < 0.5}


_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_TEMPERATURE = 0.8
_BETA = 0.4


def _logits(rows, vocab, gen, dev):
    """Rows as a language model gives them: a broad bulk that falls off along the
    vocabulary (rarer tokens sit at higher ids) and a few candidates well above it."""
    z = torch.randn(rows, vocab, device=dev, generator=gen)
    z.mul_(2.0).sub_(torch.log1p(torch.arange(vocab, device=dev) / 64.0).mul_(0.5))
    n = min(24, vocab)
    peaks = torch.rand(rows, n, device=dev, generator=gen).mul_(12.0)
    at = torch.randint(0, vocab, (rows, n), device=dev, generator=gen)
    return z.scatter_add_(1, at, peaks)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    z = _logits(rows, vocab, gen, dev)
    st = {"case": case, "logits": z.to(dtype)}
    if case["op"] == "control":
        length = case["history"]
        u = torch.rand(rows, length, device=dev, generator=gen)
        st["history"] = (u.pow(3) * vocab).long().clamp_(0, vocab - 1).int()  # frequent tokens repeat
        lens = torch.randint(0, length + 1, (rows,), device=dev, generator=gen, dtype=torch.int32)
        lens[0] = length
        st["history_lens"] = lens
        st["prompt_lens"] = (lens * torch.rand(rows, device=dev, generator=gen)).int()
        st["repetition"] = 1.0 + 0.3 * torch.rand(rows, device=dev, generator=gen)
        st["presence"] = torch.rand(rows, device=dev, generator=gen) - 0.2
        st["frequency"] = torch.rand(rows, device=dev, generator=gen) * 0.3
        if rows > 2:  # one request of the batch uses no penalty
            st["repetition"][1], st["presence"][1], st["frequency"][1] = 1.0, 0.0, 0.0
        st["bias_offsets"] = st["bias_ids"] = st["bias_values"] = None
        if case["bias"]:
            n = min(case["bias"], vocab)
            ids = torch.rand(rows, vocab, device=dev, generator=gen).topk(n, dim=1).indices
            st["bias_ids"] = ids.reshape(-1).int()
            st["bias_values"] = torch.randn(rows * n, device=dev, generator=gen) * 5
            st["bias_offsets"] = torch.arange(rows + 1, device=dev, dtype=torch.int32) * n
        st["mask"] = st["mask_rows"] = None
        if case["mask"]:
            words = (vocab + 31) // 32
            on = torch.arange(rows, device=dev) % 3 == 0
            some = int(on.sum())
            r = torch.randint(-2 ** 31, 2 ** 31, (4, some, words), device=dev, generator=gen)
            m = r[0] & r[1] & r[2] & r[3]  # a grammar state allows about one token in sixteen
            if some > 2:
                m[1] = 0       # a state that allows nothing
                m[2] = -1      # and one that allows everything
            st["mask"] = m.int()
            st["mask_rows"] = torch.where(on, torch.cumsum(on, 0) - 1, -1).int()
        return st
    if case["op"] == "top":
        return st
    k = case["k"]
    # a larger model's view of the same positions: the student's logits moved about
    t = z.add_(torch.randn(rows, vocab, device=dev, generator=gen)).div_(_TEMPERATURE)
    lse = torch.logsumexp(t, 1, keepdim=True)
    top = t.topk(k, dim=1)
    st["ids"], st["lps"] = top.indices, top.values - lse
    cut = torch.randint(1, k + 1, (rows,), device=dev, generator=gen)
    cut[torch.rand(rows, device=dev, generator=gen) < 0.7] = k    # most rows carry a full table
    if rows > 4:
        cut[3] = 0                                                # and some positions have no teacher at all
    st["ids"].masked_fill_(torch.arange(k, device=dev) >= cut.unsqueeze(1), -1)
    st["grad"] = torch.rand(rows, device=dev, generator=gen) + 0.5
    if case["targets"]:
        st["targets"] = torch.where(torch.rand(rows, device=dev, generator=gen) < 0.5, st["ids"][:, 0].clamp(min=0),
                                    torch.randint(0, vocab, (rows,), device=dev, generator=gen))
        st["grad_lp"] = torch.randn(rows, device=dev, generator=gen)
    if case["op"] == "distill":
        st["logits"].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _plain_control(st):
    z = st["logits"].float()
    rows, vocab = z.shape
    dev = z.device
    ids = st["history"].long()
    at = torch.arange(ids.shape[1], device=dev)
    live = at < st["history_lens"].unsqueeze(1)
    out_part = live & (at >= st["prompt_lens"].unsqueeze(1))
    zeros = torch.zeros(rows, vocab, device=dev, dtype=torch.int32)
    count = zeros.scatter_add(1, ids, out_part.int()).float()
    seen = zeros.scatter_add(1, ids, live.int()) > 0
    rep = st["repetition"].unsqueeze(1)
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - st["frequency"].unsqueeze(1) * count - st["presence"].unsqueeze(1) * (count > 0)
    if st["bias_ids"] is not None:
        bias = torch.zeros_like(z)
        n = st["bias_ids"].numel() // rows
        bias.scatter_add_(1, st["bias_ids"].long().view(rows, n), st["bias_values"].view(rows, n))
        z = z + bias
    if st["mask"] is not None:
        v = torch.arange(vocab, device=dev)
        words = st["mask"][st["mask_rows"].clamp(min=0).long()][:, v // 32]
        allowed = ((words >> (v % 32)) & 1).bool() | (st["mask_rows"] < 0).unsqueeze(1)
        z = torch.where(allowed, z, -math.inf)
    return z


def _plain_top(st):
    z, k = st["logits"].float(), st["case"]["k"]
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -2 ** 31 - 1 - bits, bits)         # orders as the values do
    key = (order << 32) - torch.arange(z.shape[1], device=z.device)  # ties: lowest index first
    ids = (-(key.topk(k, dim=1).values)) & 0xFFFFFFFF
    m = z.amax(1, keepdim=True)
    log_s = torch.exp((z - m) / _TEMPERATURE).sum(1, keepdim=True).log()
    return ids, (z.gather(1, ids) - m) / _TEMPERATURE - log_s, (m / _TEMPERATURE + log_s).squeeze(1)


def _plain_parts(st):
    """Loss, the gradient with respect to the logits for a unit upstream gradient,
    the softmax and the targets' logprobs."""
    case = st["case"]
    z = st["logits"].detach().float()
    rows, vocab = z.shape
    ids, lp = st["ids"], st["lps"].double()
    ok = (ids >= 0) & (ids < vocab) & (lp > -math.inf)
    slot = torch.where(ok, ids, vocab)
    member = torch.zeros(rows, vocab + 1, device=z.device, dtype=torch.bool).scatter_(1, slot, True)[:, :vocab]
    m = z.amax(1, keepdim=True)
    e = torch.exp((z - m) / _TEMPERATURE)
    at = slot.clamp(max=vocab - 1)
    s_top = (e.gather(1, at) * ok).double().sum(1, keepdim=True)
    s_rest = torch.where(member, 0.0, e).sum(1, keepdim=True).double()
    s = s_top + s_rest
    lq = torch.where(ok, (z.gather(1, at) - m).double() / _TEMPERATURE - s.log(), 0.0)
    q = torch.where(ok, lq.exp(), 0.0)
    lp = torch.where(ok, lp, 0.0)
    p = torch.where(ok, lp.exp(), 0.0)
    mass = p.sum(1, keepdim=True)
    some, rest = ok.any(1, keepdim=True), s_rest > 0
    if case["tail"] == "drop":
        p, lp = p / mass, torch.where(ok, lp - mass.log(), 0.0)
        p_rest = torch.zeros_like(mass)
    else:
        p_rest = torch.where(rest, (1 - mass).clamp(min=REST_FLOOR), 0.0)
    q_rest = s_rest / s
    lq_rest = torch.where(rest, q_rest, 1.0).log()
    lp_rest = torch.where(p_rest > 0, p_rest, 1.0).log()
    if case["divergence"] == "forward":
        loss = (p * (lp - lq)).sum(1, keepdim=True) + p_rest * (lp_rest - lq_rest)
        total = p.sum(1, keepdim=True) + p_rest
        d_top = q * total - p
        c_rest = total - torch.where(rest, p_rest / q_rest, 0.0)
    else:
        if case["divergence"] == "reverse":
            h, h_rest = lq - lp, torch.where(rest, lq_rest - lp_rest, 0.0)
            loss = (q * h).sum(1, keepdim=True) + q_rest * h_rest
        else:
            b = _BETA
            lm = torch.where(ok, b * p + (1 - b) * q, 1.0).log()
            lm_rest = torch.where(rest, b * p_rest + (1 - b) * q_rest, 1.0).log()
            h, h_rest = (1 - b) * (lq - lm), (1 - b) * (lq_rest - lm_rest)
            loss = (b * p * (lp - lm)).sum(1, keepdim=True) + b * p_rest * (lp_rest - lm_rest)
            loss = loss + (q * h).sum(1, keepdim=True) + q_rest * h_rest
        mean = (q * h).sum(1, keepdim=True) + q_rest * h_rest
        d_top = q * (h - mean)
        c_rest = h_rest - mean
    soft = e / s.float()
    grad = soft * c_rest.float()
    d = torch.zeros(rows, vocab + 1, device=z.device).scatter_(1, slot, d_top.float())[:, :vocab]
    grad = torch.where(member, d, grad) / _TEMPERATURE
    loss = torch.where(some, loss, 0.0).squeeze(1).float()
    grad = torch.where(some, grad, 0.0)
    logp = None
    if "targets" in st:
        t = st["targets"].unsqueeze(1)
        logp = ((z.gather(1, t) - m).double() / _TEMPERATURE - s.log()).squeeze(1).float()
    return loss, grad, soft, logp


def _plain_distill(st):
    loss, grad, soft, logp = _plain_parts(st)
    grad = grad * st["grad"].unsqueeze(1)
    if logp is None:
        return loss, grad.to(st["logits"].dtype)
    g = st["grad_lp"].unsqueeze(1) / _TEMPERATURE
    grad = (grad - g * soft).scatter_add(1, st["targets"].unsqueeze(1), g)
    return loss, logp, grad.to(st["logits"].dtype)


def _plain_distill_grad(st):
    loss, grad, _, _ = _plain_parts(st)
    return loss, grad.to(st["logits"].dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    st = state
    case = st["case"]
    op = case["op"]
    if own:
        from libra_b200 import ops

        if op == "control":
            return ops.control_logits(
                st["logits"], history=st["history"], history_lens=st["history_lens"], prompt_lens=st["prompt_lens"],
                repetition=st["repetition"], presence=st["presence"], frequency=st["frequency"],
                bias_offsets=st["bias_offsets"], bias_ids=st["bias_ids"], bias_values=st["bias_values"],
                mask=st["mask"], mask_rows=st["mask_rows"])
        if op == "top":
            return ops.top_logprobs(st["logits"], case["k"], _TEMPERATURE)
        kw = dict(divergence=case["divergence"], beta=_BETA, tail=case["tail"], temperature=_TEMPERATURE)
        if op == "distill_grad":
            return ops.distill_loss_grad(st["logits"], st["ids"], st["lps"], **kw)
        z = st["logits"]
        if not case["targets"]:
            loss = ops.distill_loss(z, st["ids"], st["lps"], **kw)
            (grad,) = torch.autograd.grad(loss, z, st["grad"])
            return loss.detach(), grad
        loss, logp = ops.distill_loss(z, st["ids"], st["lps"], targets=st["targets"], **kw)
        (grad,) = torch.autograd.grad((loss, logp), z, (st["grad"], st["grad_lp"]))
        return loss.detach(), logp.detach(), grad
    return {"control": _plain_control, "top": _plain_top, "distill": _plain_distill,
            "distill_grad": _plain_distill_grad}[op](st)


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    n = rows * vocab
    if case["op"] == "control":
        masked = (rows + 2) // 3 * vocab / 8 if case["mask"] else 0
        return {"bytes": n * (size + 4) + rows * case["history"] * 2 + masked + rows * case["bias"] * 8,
                "flops": 4 * n}
    if case["op"] == "top":
        return {"bytes": n * size + rows * case["k"] * 12 + rows * 4, "flops": 5 * n}
    return {"bytes": 2 * n * size + rows * case["k"] * 12 + rows * 8, "flops": 9 * n}


# ---------------------------------------------------------------------------
# definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_control(st):
    z = st["logits"].double()
    rows, vocab = z.shape
    for r in range(rows):
        n, p = int(st["history_lens"][r]), int(st["prompt_lens"][r])
        hist = st["history"][r, :n].long()
        count = torch.bincount(hist[p:], minlength=vocab)
        used = torch.bincount(hist, minlength=vocab).bool()
        rep = st["repetition"][r].double()
        row = z[r]
        row[used] = torch.where(row[used] > 0, row[used] / rep, row[used] * rep)
        row -= count * st["frequency"][r].double()
        row[count > 0] -= st["presence"][r].double()
        if st["bias_ids"] is not None:
            a, b = int(st["bias_offsets"][r]), int(st["bias_offsets"][r + 1])
            row.index_add_(0, st["bias_ids"][a:b].long(), st["bias_values"][a:b].double())
        if st["mask"] is not None and int(st["mask_rows"][r]) >= 0:
            w = st["mask"][int(st["mask_rows"][r])]
            bit = (w.unsqueeze(1) >> torch.arange(32, device=w.device)) & 1
            row[bit.reshape(-1)[:vocab] == 0] = -math.inf
    return z


def _exact_top(st):
    z = st["logits"].double()
    order = torch.sort(z, dim=1, descending=True, stable=True)
    ids = order.indices[:, :st["case"]["k"]]
    lse = torch.logsumexp(z / _TEMPERATURE, 1)
    return ids, order.values[:, :st["case"]["k"]] / _TEMPERATURE - lse.unsqueeze(1), lse


def _buckets(z, ids, lps, case):
    """Loss of each row as a function of its logits: both distributions as the
    listed tokens and one bucket for all others."""
    vocab = z.shape[1]
    ok = (ids >= 0) & (ids < vocab) & (lps > -math.inf)
    at = torch.where(ok, ids, 0)
    logq = torch.log_softmax(z / _TEMPERATURE, 1)
    others = torch.ones(z.shape[0], vocab + 1, dtype=torch.bool, device=z.device)
    others = others.scatter(1, torch.where(ok, ids, vocab), False)[:, :vocab]
    left = others.any(1)
    lq_rest = torch.logsumexp(torch.where(others, logq, torch.where(left, -math.inf, 0.0).unsqueeze(1)), 1)
    lp = torch.where(ok, lps.double(), -math.inf)
    mass = lp.exp().sum(1)
    if case["tail"] == "drop":
        lp = lp - mass.clamp(min=1e-300).log().unsqueeze(1)
        p_rest = torch.zeros_like(mass)
    else:
        p_rest = torch.where(left, (1 - mass).clamp(min=REST_FLOOR), 0.0)
    p = torch.cat([lp.exp(), p_rest.unsqueeze(1)], 1)
    lp = torch.cat([torch.where(ok, lp, 0.0), torch.where(p_rest > 0, p_rest, 1.0).log().unsqueeze(1)], 1)
    on = torch.cat([ok, left.unsqueeze(1)], 1)
    lq = torch.where(on, torch.cat([logq.gather(1, at), lq_rest.unsqueeze(1)], 1), 0.0)
    q = torch.where(on, lq.exp(), 0.0)
    if case["divergence"] == "forward":
        terms = p * (lp - lq)
    elif case["divergence"] == "reverse":
        terms = q * (lq - lp)
    else:
        lm = torch.where(on, _BETA * p + (1 - _BETA) * q, 1.0).log()
        terms = _BETA * p * (lp - lm) + (1 - _BETA) * q * (lq - lm)
    return torch.where(ok.any(1), terms.sum(1), 0.0), logq


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "control":
        return _exact_control(st)
    if case["op"] == "top":
        return _exact_top(st)
    losses, logps, grads = [], [], []
    for a in range(0, case["rows"], 512):
        z = st["logits"][a:a + 512].detach().double().requires_grad_(True)
        loss, logq = _buckets(z, st["ids"][a:a + 512], st["lps"][a:a + 512], case)
        up = st["grad"][a:a + 512].double() if case["op"] == "distill" else torch.ones_like(loss)
        total = (loss * up).sum()
        if case["targets"]:
            logp = logq.gather(1, st["targets"][a:a + 512].unsqueeze(1)).squeeze(1)
            logps.append(logp.detach())
            total = total + (logp * st["grad_lp"][a:a + 512].double()).sum()
        grads.append(torch.autograd.grad(total, z)[0])
        losses.append(loss.detach())
    out = [torch.cat(losses)] + ([torch.cat(logps)] if logps else []) + [torch.cat(grads)]
    return tuple(out)
