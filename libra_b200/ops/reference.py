"""Plain PyTorch fp32 implementations of every fused op.

These are the numerics oracle for the CUDA kernels (tests compare against
them) and the execution path for CPU tensors (gloo plumbing runs, unit tests).
They follow the maths of the reference's library calls:

* RMSNorm / q-k norm / RoPE / SwiGLU as in the HF/Megatron Qwen3 block.
* token logprob = log_softmax(logits)[target] (reference
  ``engine/train_engine.py:35`` ``_selected_token_logprobs`` and
  ``engine/megatron_core_train_engine.py:905-948``).
* GRPO loss (reference ``engine/megatron_core_train_engine.py:950-986``).
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (xf * rstd * w.float()).to(x.dtype)


def rope_tables(max_positions: int, head_dim: int, theta: float, device=None):
    """cos/sin tables [P, D/2] in fp32, computed in float64."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    pos = torch.arange(max_positions, dtype=torch.float64)
    ang = torch.outer(pos, inv)
    return ang.cos().float().to(device), ang.sin().float().to(device)


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """x: [T, heads, D]; rotate-half convention."""
    half = x.shape[-1] // 2
    c = cos[pos.long()].unsqueeze(1)
    s = sin[pos.long()].unsqueeze(1)
    x1, x2 = x[..., :half], x[..., half:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def qk_norm_rope(qkv, qw, kw, pos, cos, sin, nq, nkv, eps):
    T = qkv.shape[0]
    D = qkv.shape[1] // (nq + 2 * nkv)
    x = qkv.float().view(T, nq + 2 * nkv, D)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    q = rmsnorm(q, qw, eps).float()
    k = rmsnorm(k, kw, eps).float()
    q = apply_rope(q, cos, sin, pos)
    k = apply_rope(k, cos, sin, pos)
    dt = qkv.dtype
    return q.to(dt).contiguous(), k.to(dt).contiguous(), v.to(dt).contiguous()


def swiglu(gu: torch.Tensor) -> torch.Tensor:
    g, u = gu.float().chunk(2, dim=-1)
    return (F.silu(g) * u).to(gu.dtype)


def varlen_causal_attention(q, k, v, cu_seqlens, scale=None):
    """q [T, Hq, D], k/v [T, Hkv, D]; packed sequences delimited by cu_seqlens."""
    T, hq, d = q.shape
    hkv = k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(d)
    out = torch.empty_like(q)
    bounds = cu_seqlens.tolist()
    for s, e in zip(bounds[:-1], bounds[1:]):
        if e <= s:
            continue
        qs = q[s:e].float().transpose(0, 1)
        ks = k[s:e].float().transpose(0, 1).repeat_interleave(hq // hkv, dim=0)
        vs = v[s:e].float().transpose(0, 1).repeat_interleave(hq // hkv, dim=0)
        att = (qs @ ks.transpose(-1, -2)) * scale
        L = e - s
        mask = torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1)
        att = att.masked_fill(mask, float("-inf")).softmax(-1)
        out[s:e] = (att @ vs).transpose(0, 1).to(q.dtype)
    return out


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, temperature: float = 1.0):
    z = logits.float() / temperature
    lp = torch.log_softmax(z, dim=-1)
    sel = lp.gather(-1, targets.long().unsqueeze(-1)).squeeze(-1)
    ent = -(lp.exp() * lp).sum(-1)
    return sel, ent


def grpo_loss(logp, old_logp, mask, adv, clip_eps: float, kl_coef: float):
    """PPO-clip with log-ratio clamped to [-20, 20] and the k3 KL estimator.

    All inputs are per-token vectors of the same shape except ``adv`` which is
    broadcast per token already.
    """
    log_ratio = logp - old_logp
    ratio = torch.exp(log_ratio.clamp(-20.0, 20.0))
    clipped = ratio.clamp(1.0 - clip_eps, 1.0 + clip_eps)
    pg = torch.maximum(-adv * ratio, -adv * clipped)
    count = mask.sum().clamp(min=1.0)
    pg_loss = (pg * mask).sum() / count
    kl = (((ratio - 1.0) - log_ratio) * mask).sum() / count
    return pg_loss + kl_coef * kl, pg_loss, kl


def control_logits(logits, history=None, history_lens=None, prompt_lens=None, history_rows=None, repetition=None,
                   presence=None, frequency=None, bias_offsets=None, bias_ids=None, bias_values=None, mask=None,
                   mask_rows=None):
    """Penalties, biases and grammar masks of ``ops.control_logits``, row by row; fp32 (fp64 for fp64 logits)."""
    z = logits.to(torch.float64 if logits.dtype == torch.float64 else torch.float32).clone()
    B, V = z.shape
    for b in range(B):
        row = z[b]
        idle = all(t is None or float(t[b]) == v for t, v in ((repetition, 1.0), (presence, 0.0), (frequency, 0.0)))
        if history is not None and not idle:
            hr = b if history_rows is None else int(history_rows[b])
            n = int(history_lens[b])
            if not 0 <= hr < history.shape[0] or not 0 <= n <= history.shape[1]:
                raise ValueError(f"control_logits: history row {hr} or length {n} outside the table")
            p = 0 if prompt_lens is None else max(0, int(prompt_lens[b]))
            toks = history[hr, :n].long()
            ok = (toks >= 0) & (toks < V)
            seen = torch.zeros(V, dtype=torch.bool, device=z.device)
            seen[toks[ok]] = True
            count = torch.bincount(toks[p:][ok[p:]], minlength=V).to(z.dtype)
            if repetition is not None:
                r = repetition[b].to(z.dtype)
                row.copy_(torch.where(seen, torch.where(row > 0, row / r, row * r), row))
            if frequency is not None:
                row.copy_(torch.where(count > 0, row - frequency[b] * count, row))
            if presence is not None:
                row.copy_(torch.where(count > 0, row - presence[b], row))
        if bias_offsets is not None:
            lo, hi = int(bias_offsets[b]), int(bias_offsets[b + 1])
            if not 0 <= lo <= hi <= bias_ids.numel():
                raise ValueError(f"control_logits: bias offsets {lo}..{hi} outside the entries")
            ids = bias_ids[lo:hi].long()
            ok = (ids >= 0) & (ids < V)
            row.index_add_(0, ids[ok], bias_values[lo:hi][ok].to(z.dtype))
        mr = -1 if mask is None else (b if mask_rows is None else int(mask_rows[b]))
        if mr >= 0:
            if mr >= mask.shape[0]:
                raise ValueError(f"control_logits: mask row {mr} outside the table")
            bits = (mask[mr].unsqueeze(1) >> torch.arange(32, dtype=torch.int32, device=z.device)) & 1
            row.masked_fill_(bits.reshape(-1)[:V] == 0, float("-inf"))
    return z


def top_logprobs(logits, k: int, temperature=1.0):
    """``ops.top_logprobs``: a stable descending sort, logprobs in fp64."""
    x = logits.double()
    t = temperature.double() if isinstance(temperature, torch.Tensor) else torch.full((x.shape[0],), float(temperature))
    t = torch.where(t > 0, t, torch.ones_like(t)).to(x.device).unsqueeze(1)
    vals, ids = torch.sort(x, dim=1, descending=True, stable=True)
    lse = torch.logsumexp(x / t, 1)
    none = lse == float("-inf")
    lp = vals[:, :k] / t - torch.where(none, torch.zeros_like(lse), lse).unsqueeze(1)
    return ids[:, :k].contiguous(), lp.float(), lse.float()


def distill_loss(logits, ids, lps, divergence: str, beta: float, tail: str, temperature: float, targets=None):
    """``ops.distill_loss`` in fp64 with autograd: (loss fp32 [N], target logprobs or None)."""
    z = logits.double()
    N, V = z.shape
    K = ids.shape[1]
    lp = lps.double()
    ok = (ids >= 0) & (ids < V) & (lp > float("-inf"))
    same = (ids.unsqueeze(2) == ids.unsqueeze(1)) & ok.unsqueeze(2) & ok.unsqueeze(1)
    ok = ok & ~(same & torch.ones(K, K, dtype=torch.bool, device=z.device).tril(-1)).any(2)
    dead = (z.detach() == float("-inf")).all(1)
    z = torch.where(dead.unsqueeze(1), torch.zeros_like(z), z)
    logq = torch.log_softmax(z / temperature, 1)
    others = torch.ones(N, V + 1, dtype=torch.bool, device=z.device)
    others = others.scatter(1, torch.where(ok, ids, torch.full_like(ids, V)), False)[:, :V]
    left = (others & (z.detach() != float("-inf"))).any(1)
    ninf = torch.full_like(z, float("-inf"))
    lq_rest = torch.logsumexp(torch.where(left.unsqueeze(1), torch.where(others, logq, ninf), torch.zeros_like(z)), 1)
    zero, one = torch.zeros_like(lp), torch.ones_like(lp)
    if tail == "drop":  # only the ratios of the p count: relative to the row's largest, none of them underflows
        most = torch.where(ok, lp, ninf[:, :1]).amax(1, keepdim=True)
        lp = lp - torch.where(most > float("-inf"), most, zero[:, :1])
    p = torch.where(ok, torch.where(ok, lp, zero).exp(), zero)
    mass = p.sum(1)
    valid = ok.any(1) & ~dead
    if tail == "drop":
        by = torch.where(mass > 0, mass, torch.ones_like(mass)).unsqueeze(1)
        p, lp = p / by, lp - by.log()
        p_rest = torch.zeros_like(mass)
    else:
        p_rest = torch.where(left, (1 - mass).clamp(min=2.0 ** -24), torch.zeros_like(mass))
    on = torch.cat([ok, left.unsqueeze(1)], 1)
    p = torch.cat([p, p_rest.unsqueeze(1)], 1)
    lp = torch.cat([torch.where(ok, lp, zero), torch.where(p_rest > 0, p_rest, torch.ones_like(p_rest)).log().unsqueeze(1)], 1)
    lq = torch.cat([logq.gather(1, torch.where(ok, ids, torch.zeros_like(ids))), lq_rest.unsqueeze(1)], 1)
    zero, one = torch.zeros_like(lq), torch.ones_like(lq)
    lq = torch.where(on, lq, zero)
    q = torch.where(on, lq.exp(), zero)
    live = q.detach() > 0
    safe = torch.where(live, lq, zero)  # q log q is 0 at q = 0, and so is its gradient here
    if divergence == "forward":
        terms = torch.where(p > 0, p * (lp - lq), zero)
    elif divergence == "reverse":
        terms = torch.where(on & live, q * (safe - lp), zero)
    else:
        mix = beta * p + (1 - beta) * q
        lm = torch.where(mix.detach() > 0, mix, one).log()
        terms = torch.where(p > 0, beta * p * (lp - lm), zero) + torch.where(live, (1 - beta) * q * (safe - lm), zero)
    loss = torch.where(valid, terms.sum(1), torch.zeros_like(mass)).float()
    if targets is None:
        return loss, None
    t = targets.long()
    if bool(((t < 0) | (t >= V)).any()):
        raise ValueError("distill_loss: target outside the vocabulary")
    logp = logq.gather(1, t.unsqueeze(1)).squeeze(1)
    return loss, torch.where(dead, torch.full_like(logp, float("-inf")), logp).float()


def embedding(tokens, w, scale, first, whole):
    """Rows ``tokens - first`` of ``w`` times ``scale``, zeros for tokens outside the table."""
    r = tokens.reshape(-1).long() - first
    here = (r >= 0) & (r < w.shape[0])
    if whole and not bool(here.all()):
        raise ValueError("embedding: a token lies outside the table")
    out = w.index_select(0, r.clamp(0, max(w.shape[0] - 1, 0))) if w.shape[0] else w.new_zeros(r.numel(), w.shape[1])
    if scale != 1.0:
        out = (out.to(torch.promote_types(w.dtype, torch.float32)) * scale).to(w.dtype)
    if not whole:
        out = out.masked_fill(~here.unsqueeze(1), 0)
    return out.view(*tokens.shape, w.shape[1])


def embedding_grad(tokens, g, rows, scale, first, main):
    """Adds scale * sum of g over each token's positions to ``main``, or returns it as [rows, H] of g's type."""
    r = tokens.reshape(-1).long() - first
    here = (r >= 0) & (r < rows)
    g = g.to(torch.float32 if main is not None else torch.promote_types(g.dtype, torch.float32))
    if not bool(here.all()):
        g, r = g[here], r[here]
    if scale != 1.0:
        g = g * scale
    if main is not None:
        main.view(rows, -1).index_add_(0, r, g)
        return None
    return torch.zeros(rows, g.shape[1], dtype=g.dtype).index_add_(0, r, g)


def route_topk(logits, k, normalize):
    """Softmax weights and indices of the k largest logits of each row, ties at the lowest index."""
    z = logits.float()
    empty = (z == float("-inf")).all(-1, keepdim=True)
    p = z.masked_fill(empty, 0.0).softmax(dim=-1).masked_fill(empty, 0.0)
    ids = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    if normalize:
        w = w / w.sum(-1, keepdim=True).masked_fill(empty, 1.0)
    return w, ids


def expert_plan(experts, num_experts, align):
    """(rows int32 [T*k], offs int32 [E+1], counts int32 [E]) of (token, slot) pairs sorted by expert."""
    flat = experts.reshape(-1).long()
    if bool((flat >= num_experts).any()):
        raise ValueError("expert_plan: an expert id is not below num_experts")
    here = flat >= 0
    key = torch.where(here, flat, torch.full_like(flat, num_experts))
    counts = torch.bincount(key, minlength=num_experts + 1)
    padded = (counts + align - 1) // align * align
    start = padded.cumsum(0) - padded
    first = counts.cumsum(0) - counts
    order = torch.argsort(key, stable=True)
    rank = torch.empty_like(key)
    rank[order] = torch.arange(key.numel()) - first[key[order]]
    rows = torch.where(here, start[key] + rank, torch.full_like(key, -1))
    return rows.int(), start.int(), counts[:num_experts].int()


def moe_dispatch(x, rows, k, capacity):
    to = torch.where(rows >= 0, rows, capacity).long()
    v = x.to(torch.promote_types(x.dtype, torch.float32))  # the gradient's sums too
    out = v.new_zeros(capacity + 1, x.shape[1])
    return out.index_copy(0, to, v.repeat_interleave(k, dim=0))[:capacity].to(x.dtype)


def moe_combine(y, weights, rows, k, residual):
    here = (rows >= 0).unsqueeze(1)
    picked = y.index_select(0, rows.clamp(min=0).long()).float().masked_fill(~here, 0.0)
    out = (picked.view(rows.numel() // k, k, y.shape[1]) * weights.unsqueeze(-1)).sum(1)
    if residual is not None:
        out = out + residual.float()
    return out.to(y.dtype)
