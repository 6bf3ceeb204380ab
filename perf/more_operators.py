"""Measured cases of the operators that move rows by sorted indices: the
embedding with its gradient by sorted tokens, the router, and the experts' plan,
dispatch and combine.

Each case is one pass through ``libra_b200.ops`` with ``own`` set, or through
the plain torch form; ``exact`` restates each definition in 64 bits.
"""

import math

import torch

own = False

VOCAB = 151936  # vocabulary of the model configurations
ALIGN = 128     # rows: the expert products want every group to start on a multiple of this


def listed():
    return [
        # a decode batch of the rollout engine looks its tokens up
        {"name": "embed-64tok", "op": "embed", "tokens": 64, "vocab": VOCAB, "hidden": 2560, "dtype": "bf16",
         "scale": 1.0, "mode": "lookup"},
        # a packed micro-batch of a training step, gradient into the engine's flat fp32 buffer
        {"name": "embed-8192tok-train", "op": "embed", "tokens": 8192, "vocab": VOCAB, "hidden": 2560,
         "dtype": "bf16", "scale": 1.0, "mode": "main_grad"},
        # an fp32 table with rows of an odd width, scaled, whose gradient is a tensor like the table
        {"name": "embed-3001tok-odd-fp32", "op": "embed", "tokens": 3001, "vocab": 50257, "hidden": 1001,
         "dtype": "fp32", "scale": 31.75, "mode": "dense"},
        # the router of a decode batch
        {"name": "route-64tok", "op": "route", "tokens": 64, "experts": 128, "k": 8, "dtype": "fp32",
         "normalize": True, "train": False},
        # the router of a packed training batch, with its gradient
        {"name": "route-16384tok-train", "op": "route", "tokens": 16384, "experts": 128, "k": 8, "dtype": "fp32",
         "normalize": True, "train": True},
        # rows of a decode batch sorted by expert
        {"name": "plan-64tok", "op": "plan", "tokens": 64, "experts": 128, "k": 8},
        # rows of a packed training batch sorted by expert
        {"name": "plan-16384tok", "op": "plan", "tokens": 16384, "experts": 128, "k": 8},
        # a decode batch goes to its experts
        {"name": "dispatch-64tok", "op": "dispatch", "tokens": 64, "experts": 128, "k": 8, "hidden": 2048,
         "dtype": "bf16", "train": False},
        # a packed training batch goes to its experts, with its gradient
        {"name": "dispatch-16384tok-train", "op": "dispatch", "tokens": 16384, "experts": 128, "k": 8,
         "hidden": 2048, "dtype": "bf16", "train": True},
        # a decode batch comes back, weighted and added to the residual stream
        {"name": "combine-64tok", "op": "combine", "tokens": 64, "experts": 128, "k": 8, "hidden": 2048,
         "dtype": "bf16", "train": False},
        # a packed training batch comes back, with all three gradients
        {"name": "combine-16384tok-train", "op": "combine", "tokens": 16384, "experts": 128, "k": 8,
         "hidden": 2048, "dtype": "bf16", "train": True},
        # plan, dispatch and combine as the block uses them, fp32 rows of odd width, padding tokens without experts
        {"name": "round-1777tok-odd-fp32", "op": "round", "tokens": 1777, "experts": 60, "k": 3, "hidden": 1001,
         "dtype": "fp32", "train": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed", "route", "plan", "dispatch", "combine", "round"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "embed":
        vocab = VOCAB if rng.random() < 0.3 else _log_int(rng, 1000, 200_000)
        hidden = rng.choice([512, 2048, 2560, 5120]) if rng.random() < 0.5 else _log_int(rng, 8, 2560)
        hidden = min(hidden, VOCAB * 2560 // vocab // (2 if dtype == "fp32" else 1))
        return {"op": op, "tokens": _log_int(rng, 1, 8192), "vocab": vocab, "hidden": hidden, "dtype": dtype,
                "scale": rng.choice([1.0, math.sqrt(hidden)]), "mode": rng.choice(["lookup", "main_grad", "dense"])}
    experts = _log_int(rng, 2, 256)
    k = min(_log_int(rng, 1, 12), experts)
    if op == "route":
        return {"op": op, "tokens": _log_int(rng, 1, 32768), "experts": experts, "k": k, "dtype": dtype,
                "normalize": rng.random() < 0.6, "train": rng.random() < 0.6}
    if op == "plan":
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "experts": experts, "k": k}
    hidden = rng.choice([256, 512, 2048, 5120]) if rng.random() < 0.5 else _log_int(rng, 8, 2560)
    most = 16384 * 8 * 2048 // (2 if dtype == "fp32" else 1) // hidden // k
    tokens = _log_int(rng, 1, min(16384, most // (2 if op == "round" else 1)))
    return {"op": op, "tokens": tokens, "experts": experts, "k": k, "hidden": hidden, "dtype": dtype,
            "train": True if op == "round" else rng.random() < 0.6}


_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _capacity(case):
    n = case["tokens"] * case["k"]
    return n + (ALIGN - 1) * min(case["experts"], n)


def _tokens(case, gen, dev):
    """Token ids as text has them: low ids far more often than high ones, and one (a line break) in every twenty."""
    n, vocab = case["tokens"], case["vocab"]
    t = (torch.rand(n, device=dev, generator=gen, dtype=torch.float64).pow(3) * vocab).long().clamp_(0, vocab - 1)
    return torch.where(torch.rand(n, device=dev, generator=gen) < 0.05, torch.full_like(t, vocab // 7), t)


def _experts(case, gen, dev):
    """Each token's experts: distinct, some experts far more popular than others; in a padded batch the last tokens
    have none (-1)."""
    n, experts, k = case["tokens"], case["experts"], case["k"]
    pull = torch.randn(experts, device=dev, generator=gen) * 0.7
    z = torch.randn(n, experts, device=dev, generator=gen) + pull
    ids = z.topk(k, dim=1).indices
    if case["op"] == "round":
        ids[n - n // 16:] = -1
    return ids


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    n, op = case["tokens"], case["op"]

    def rows(count, width, dtype=None, std=1.0):
        x = torch.randn(count, width, device=dev, generator=gen) * std
        return x.to(_DTYPES[case["dtype"]] if dtype is None else dtype)

    st = {"case": case}
    if op == "embed":
        st["tokens"] = _tokens(case, gen, dev)
        st["weight"] = rows(case["vocab"], case["hidden"], std=0.02)
        if case["mode"] != "lookup":
            st["grad"] = rows(n, case["hidden"])
            st["weight"].requires_grad_(own)
        if case["mode"] == "main_grad":
            st["main"] = rows(case["vocab"], case["hidden"], dtype=torch.float32)  # an earlier micro-batch's gradients
            st["weight"].main_grad = st["main"]
        return st
    if op == "route":
        st["logits"] = rows(n, case["experts"], std=1.5)
        if case["train"]:
            st["logits"].requires_grad_(own)
            st["grad"] = torch.randn(n, case["k"], device=dev, generator=gen)
        return st
    st["experts"] = _experts(case, gen, dev)
    if op == "plan":
        return st
    cap, hidden, k = _capacity(case), case["hidden"], case["k"]
    if op in ("dispatch", "round"):
        st["x"] = rows(n, hidden)
    if op in ("combine", "round"):
        w = torch.rand(n, k, device=dev, generator=gen) + 0.05
        st["weights"] = w / w.sum(1, keepdim=True)
        st["residual"] = rows(n, hidden)
    if op == "combine":
        st["y"] = rows(cap, hidden)
    if case["train"]:
        st["grad"] = rows(cap if op == "dispatch" else n, hidden)
        for name in ("x", "y", "weights", "residual"):
            if name in st:
                st[name].requires_grad_(own)
    if op != "round":  # a layer has its plan in hand here
        if own:
            from libra_b200 import ops

            st["plan"] = ops.expert_plan(st["experts"], case["experts"], align=ALIGN)
        else:
            st["rows"], _, _ = _plan_plain(st["experts"], case["experts"])
    return st


# ------------------------------------------------------------------ plain forms

def _plan_plain(experts, count):
    """(row of each (token, slot) pair or -1, group starts, group counts)"""
    flat = experts.reshape(-1)
    here = flat >= 0
    key = torch.where(here, flat, count)
    counts = torch.zeros(count + 1, dtype=torch.int64, device=flat.device)
    counts.scatter_add_(0, key, torch.ones_like(key))
    padded = (counts + ALIGN - 1) // ALIGN * ALIGN
    start = padded.cumsum(0) - padded
    first = counts.cumsum(0) - counts
    order = torch.argsort(key, stable=True)
    rank = torch.empty_like(key)
    rank[order] = torch.arange(key.numel(), device=key.device) - first[key[order]]
    rows = torch.where(here, start[key] + rank, -1)
    return rows.int(), start.int(), counts[:count].int()


def _dispatch_plain(x, rows, k, cap, scale=None):
    """x[t] (times scale[t, i]) at row rows[t * k + i], zeros elsewhere, 32 bits."""
    out = torch.zeros(cap + 1, x.shape[1], device=x.device)
    v = x.float().repeat_interleave(k, dim=0)
    if scale is not None:
        v = v * scale.reshape(-1, 1)
    out[torch.where(rows >= 0, rows, cap).long()] = v
    return out[:cap]


def _pick_plain(y, rows, k):
    """[T, k, H]: row rows[t * k + i] of y, zeros for none, 32 bits."""
    v = y[rows.clamp(min=0).long()].float() * (rows >= 0).unsqueeze(1)
    return v.view(-1, k, y.shape[1])


def _run_plain(st):
    case = st["case"]
    op, dtype = case["op"], _DTYPES[case.get("dtype", "fp32")]
    if op == "embed":
        w, t = st["weight"], st["tokens"]
        out = {"out": (w[t].float() * case["scale"]).to(dtype)}
        if case["mode"] == "lookup":
            return out
        g = st["grad"].float() * case["scale"]
        if case["mode"] == "main_grad":
            out["dw"] = st["main"].index_add_(0, t, g)
        else:
            out["dw"] = torch.zeros(w.shape, device=w.device).index_add_(0, t, g).to(dtype)
        return out
    if op == "route":
        z, k = st["logits"].float(), case["k"]
        e = (z - z.max(1, keepdim=True).values).exp()
        p = e / e.sum(1, keepdim=True)
        ids = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
        w = p.gather(1, ids)
        if case["normalize"]:
            w = w / w.sum(1, keepdim=True)
        out = {"weights": w, "experts": ids}
        if case["train"]:
            g = st["grad"]
            inner = (w * g).sum(1, keepdim=True)
            if case["normalize"]:
                dz = torch.zeros_like(z).scatter_(1, ids, w * (g - inner))
            else:
                dz = (-p * inner).scatter_add_(1, ids, w * g)
            out["dlogits"] = dz.to(dtype)
        return out
    if op == "plan":
        return dict(zip(("rows", "offs", "counts"), _plan_plain(st["experts"], case["experts"])))
    k, cap = case["k"], _capacity(case)
    if op == "dispatch":
        out = {"xs": _dispatch_plain(st["x"], st["rows"], k, cap).to(dtype)}
        if case["train"]:
            out["dx"] = _pick_plain(st["grad"], st["rows"], k).sum(1).to(dtype)
        return out
    if op == "combine":
        y, rows, out = st["y"], st["rows"], {}
    else:
        rows, _, _ = _plan_plain(st["experts"], case["experts"])
        y = _dispatch_plain(st["x"], rows, k, cap).to(dtype)
        out = {"xs": y}
    w = st["weights"]
    picked = _pick_plain(y, rows, k)
    out["out"] = ((picked * w.unsqueeze(-1)).sum(1) + st["residual"].float()).to(dtype)
    if case["train"]:
        g = st["grad"]
        dy = _dispatch_plain(g, rows, k, cap, w).to(dtype)
        out["dweights"] = (picked * g.float().unsqueeze(1)).sum(2)
        out["dresidual"] = g
        if op == "round":
            out["dx"] = _pick_plain(dy, rows, k).sum(1).to(dtype)
        else:
            out["dy"] = dy
    return out


# ------------------------------------------------------------------ the framework's operators

def _run_own(st):
    from libra_b200 import ops

    case = st["case"]
    op = case["op"]
    if op == "embed":
        if case["mode"] == "lookup":
            with torch.no_grad():
                return {"out": ops.embedding(st["tokens"], st["weight"], scale=case["scale"])}
        out = ops.embedding(st["tokens"], st["weight"], scale=case["scale"])
        if case["mode"] == "main_grad":
            out.backward(st["grad"])
            return {"out": out, "dw": st["main"]}
        return {"out": out, "dw": torch.autograd.grad(out, st["weight"], st["grad"])[0]}
    if op == "route":
        if not case["train"]:
            with torch.no_grad():
                w, ids = ops.route_topk(st["logits"], case["k"], normalize=case["normalize"])
            return {"weights": w, "experts": ids}
        w, ids = ops.route_topk(st["logits"], case["k"], normalize=case["normalize"])
        return {"weights": w, "experts": ids, "dlogits": torch.autograd.grad(w, st["logits"], st["grad"])[0]}
    if op == "plan":
        plan = ops.expert_plan(st["experts"], case["experts"], align=ALIGN)
        return {"rows": plan.rows, "offs": plan.offs, "counts": plan.counts}
    if op == "dispatch":
        if not case["train"]:
            with torch.no_grad():
                return {"xs": ops.moe_dispatch(st["x"], st["plan"])}
        xs = ops.moe_dispatch(st["x"], st["plan"])
        return {"xs": xs, "dx": torch.autograd.grad(xs, st["x"], st["grad"])[0]}
    if op == "combine":
        if not case["train"]:
            with torch.no_grad():
                return {"out": ops.moe_combine(st["y"], st["weights"], st["plan"], residual=st["residual"])}
        out = ops.moe_combine(st["y"], st["weights"], st["plan"], residual=st["residual"])
        dy, dw, dres = torch.autograd.grad(out, (st["y"], st["weights"], st["residual"]), st["grad"])
        return {"out": out, "dy": dy, "dweights": dw, "dresidual": dres}
    plan = ops.expert_plan(st["experts"], case["experts"], align=ALIGN)
    xs = ops.moe_dispatch(st["x"], plan)
    out = ops.moe_combine(xs, st["weights"], plan, residual=st["residual"])
    dx, dw, dres = torch.autograd.grad(out, (st["x"], st["weights"], st["residual"]), st["grad"])
    return {"xs": xs, "out": out, "dweights": dw, "dresidual": dres, "dx": dx}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def _distinct(case):
    """Expected number of different tokens among those of ``_tokens``."""
    n, vocab = case["tokens"], case["vocab"]
    edge = (torch.arange(vocab + 1, dtype=torch.float64) / vocab).pow(1.0 / 3.0)
    p = 0.95 * (edge[1:] - edge[:-1])
    p[vocab // 7] += 0.05
    return float((1 - (1 - p).pow(n)).sum())


def work(case):
    n, op = case["tokens"], case["op"]
    size = 4 if case.get("dtype") == "fp32" else 2
    if op == "embed":
        row = case["hidden"] * size
        uniq = _distinct(case)
        b, f = 8 * n + (uniq + n) * row, n * case["hidden"]
        if case["mode"] != "lookup":
            b += n * row + (2 * uniq * case["hidden"] * 4 if case["mode"] == "main_grad" else case["vocab"] * row)
            f += 2 * n * case["hidden"]
        return {"bytes": b, "flops": f}
    k, experts = case["k"], case["experts"]
    if op == "route":
        b, f = n * experts * size + n * k * 12, 4 * n * experts
        if case["train"]:
            b += n * experts * size + n * k * 4
            f += 4 * n * (k if case["normalize"] else experts)
        return {"bytes": b, "flops": f}
    plan = n * k * 12 + (2 * experts + 1) * 4
    if op == "plan":
        return {"bytes": plan, "flops": n * k}
    row, cap, h = case["hidden"] * size, _capacity(case), case["hidden"]
    there = n * row + n * k * 4 + cap * row           # tokens read, all rows of the experts' layout written
    back = n * k * row + n * k * 4 + n * row          # the tokens' rows read, their sums written
    if op == "dispatch":
        return {"bytes": there + (back if case["train"] else 0), "flops": n * k * h if case["train"] else 0}
    back += n * row + n * k * 4                       # the residual and the weights
    grads = n * row + n * k * row + cap * row + n * k * 12
    if op == "combine":
        return {"bytes": back + (grads if case["train"] else 0), "flops": (5 if case["train"] else 2) * n * k * h}
    return {"bytes": plan + there + back + grads + n * k * row + n * row, "flops": 6 * n * k * h}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    op, n = case["op"], case["tokens"]
    if op == "embed":
        scale, t = case["scale"], st["tokens"]
        out = {"out": torch.index_select(st["weight"], 0, t).double().mul_(scale)}
        if case["mode"] != "lookup":
            # each token's occurrences side by side, summed between their borders
            order = torch.argsort(t, stable=True)
            at, many = torch.unique_consecutive(t[order], return_counts=True)
            total = torch.segment_reduce(st["grad"].double()[order], "sum", lengths=many, axis=0).mul_(scale)
            base = st["main"].double() if case["mode"] == "main_grad" else torch.zeros(
                case["vocab"], case["hidden"], dtype=torch.float64, device=t.device)
            base[at] += total
            out["dw"] = base
        return out
    k, experts = case["k"], case["experts"]
    if op == "route":
        z = st["logits"].double().requires_grad_(True)
        # rank of each expert: how many stand before it (larger, or as large with a lower index)
        ids = torch.empty(n, k, dtype=torch.int64, device=z.device)
        below = torch.arange(experts, device=z.device)
        with torch.no_grad():
            for s in range(0, n, 1024):
                zs = z[s:s + 1024]
                before = (zs[:, None, :] > zs[:, :, None]) | ((zs[:, None, :] == zs[:, :, None])
                                                             & (below[None, None, :] < below[None, :, None]))
                rank = before.sum(2)
                hit = rank[:, None, :] == torch.arange(k, device=z.device)[None, :, None]
                ids[s:s + 1024] = hit.int().argmax(2)
        w = torch.softmax(z, 1).gather(1, ids)
        if case["normalize"]:
            w = torch.softmax(z.gather(1, ids), 1)
        out = {"weights": w.detach(), "experts": ids}
        if case["train"]:
            out["dlogits"] = torch.autograd.grad(w, z, st["grad"].double())[0]
        return out
    ids = st["experts"].reshape(-1)
    # a pair's row: its group's start, and how many pairs before it chose the same expert
    hot = (ids[:, None] == torch.arange(experts, device=ids.device)[None, :])
    before = hot.int().cumsum(0, dtype=torch.int32)
    counts = before[-1].long()
    start = torch.cat([counts.new_zeros(1), (-(-counts // ALIGN) * ALIGN).cumsum(0)])
    safe = ids.clamp(min=0)
    rows = torch.where(ids >= 0, start[safe] + before.gather(1, safe[:, None])[:, 0] - 1, -1)
    del hot, before
    if op == "plan":
        return {"rows": rows, "offs": start, "counts": counts}
    cap, hidden = _capacity(case), case["hidden"]
    pair = torch.full((cap,), -1, dtype=torch.int64, device=ids.device)
    pair[rows[rows >= 0]] = (rows >= 0).nonzero()[:, 0]

    def spread(x):  # row by row of the experts' layout: the token's row there, or zeros
        return torch.where((pair >= 0)[:, None], x.double()[(pair // k).clamp(min=0)], 0.0)

    def sums(y, weights):
        total = torch.zeros(n, hidden, dtype=torch.float64, device=ids.device)
        for i in range(k):
            r = rows.view(n, k)[:, i]
            total += torch.where((r >= 0)[:, None], y[r.clamp(min=0)].double(), 0.0) * weights[:, i:i + 1]
        return total

    ones = torch.ones(n, k, dtype=torch.float64, device=ids.device)
    if op == "dispatch":
        out = {"xs": spread(st["x"])}
        if case["train"]:
            out["dx"] = sums(st["grad"], ones)
        return out
    w = st["weights"].double()
    y = st["y"] if op == "combine" else spread(st["x"])
    out = {"out": sums(y, w) + st["residual"].double()}
    if op == "round":
        out["xs"] = y
    if case["train"]:
        g = st["grad"].double()
        out["dresidual"] = g
        dw = torch.zeros(n, k, dtype=torch.float64, device=ids.device)
        for i in range(k):
            r = rows.view(n, k)[:, i]
            dw[:, i] = torch.where(r >= 0, (y[r.clamp(min=0)].double() * g).sum(1), 0.0)
        out["dweights"] = dw
        dy = spread(g).mul_(torch.where(pair >= 0, w.reshape(-1)[pair.clamp(min=0)], 0.0)[:, None])
        if op == "round":
            out["dx"] = sums(dy, ones)
        else:
            out["dy"] = dy
    return out
