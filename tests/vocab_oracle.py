"""Plain 64-bit restatements of the vocabulary-row operators, row by row, for the tests."""

import math

import torch

REST_FLOOR = 2.0 ** -24


def control(z, history=None, history_lens=None, prompt_lens=None, history_rows=None, repetition=None, presence=None,
            frequency=None, bias_offsets=None, bias_ids=None, bias_values=None, mask=None, mask_rows=None):
    """(controlled rows, sum of the magnitudes that went into each value) in fp64."""
    out, mag = z.double().cpu().clone(), z.double().cpu().abs().clone()
    B, V = out.shape
    for b in range(B):
        r = float(repetition[b]) if repetition is not None else 1.0
        p = float(presence[b]) if presence is not None else 0.0
        f = float(frequency[b]) if frequency is not None else 0.0
        seen, count = set(), {}
        if history is not None:
            row = history[int(history_rows[b]) if history_rows is not None else b].tolist()
            start = int(prompt_lens[b]) if prompt_lens is not None else 0
            for i, t in enumerate(row[:int(history_lens[b])]):
                if 0 <= t < V:
                    seen.add(t)
                    if i >= start:
                        count[t] = count.get(t, 0) + 1
        for t in seen:
            x = float(out[b, t])
            out[b, t] = x / r if x > 0 else x * r
            mag[b, t] = abs(float(out[b, t]))
        for t, n in count.items():
            out[b, t] -= f * n + p
            mag[b, t] += abs(f) * n + abs(p)
        if bias_offsets is not None:
            for e in range(int(bias_offsets[b]), int(bias_offsets[b + 1])):
                t, v = int(bias_ids[e]), float(bias_values[e])
                if 0 <= t < V:
                    out[b, t] += v
                    mag[b, t] += abs(v)
        mr = -1 if mask is None else (b if mask_rows is None else int(mask_rows[b]))
        if mr >= 0:
            words = mask[mr].tolist()
            for t in range(V):
                if not (words[t // 32] >> (t % 32)) & 1:
                    out[b, t] = -math.inf
    return out, mag


def top(z, k, temperature):
    z = z.double().cpu()
    vals, ids = torch.sort(z, dim=1, descending=True, stable=True)
    t = torch.as_tensor(temperature, dtype=torch.float64).cpu().expand(z.shape[0])
    t = torch.where(t > 0, t, torch.ones_like(t)).unsqueeze(1)
    lse = torch.logsumexp(z / t, 1)
    lp = vals[:, :k] / t - lse.unsqueeze(1)
    lp[lse == -math.inf] = -math.inf  # by definition: nothing is allowed
    return ids[:, :k], lp, lse


def distill_row(z, ids, lps, divergence, beta, tail, T):
    """One row as a differentiable function: (loss, log softmax).  z [V] fp64, ids / lps lists."""
    V = z.shape[0]
    table = {}
    for i, lp in zip(ids, lps):
        if 0 <= i < V and lp > -math.inf and i not in table:
            table[i] = lp
    logq = torch.log_softmax(z / T, 0)
    zero = torch.where(torch.isfinite(z), z, 0.0).sum() * 0.0
    others = [j for j, v in enumerate(z.tolist()) if j not in table and v > -math.inf]
    mass = sum(math.exp(lp) for lp in table.values())
    if not table or not bool((z > -math.inf).any()) or (tail == "drop" and mass == 0):
        return zero, logq
    lp = dict(table)
    if tail == "drop":
        lp = {i: v - math.log(mass) for i, v in lp.items()}
    buckets = [(v, logq[i]) for i, v in lp.items()]
    if others:
        lq_rest = torch.logsumexp(logq[torch.tensor(others)], 0)
        buckets.append((math.log(max(1.0 - mass, REST_FLOOR)) if tail == "bucket" else -math.inf, lq_rest))
    loss = zero
    for a, lq in buckets:
        p, q = math.exp(a), lq.exp()
        dead = float(lq.detach()) == -math.inf
        if divergence == "forward":
            if p > 0:
                loss = loss + p * (a - lq)
        elif divergence == "reverse":
            if not dead:
                loss = loss + q * (lq - a)
        else:
            lm = torch.log(beta * p + (1 - beta) * q)
            if p > 0:
                loss = loss + beta * p * (a - lm)
            if not dead:
                loss = loss + (1 - beta) * q * (lq - lm)
    return loss, logq


def distill(z, ids, lps, divergence, beta, tail, T, targets=None, g=None, g_lp=None):
    """fp64 (loss [N], logp [N] or None, gradient [N, V])."""
    N = z.shape[0]
    losses, logps, grads = [], [], []
    for n in range(N):
        x = z[n].double().cpu().clone().requires_grad_(True)
        loss, logq = distill_row(x, ids[n].tolist(), lps[n].double().tolist(), divergence, beta, tail, T)
        total = loss * (1.0 if g is None else float(g[n]))
        if targets is not None:
            lt = logq[int(targets[n])]
            logps.append(float(lt))
            if g_lp is not None:
                total = total + lt * float(g_lp[n])
        grads.append(torch.autograd.grad(total, x)[0])
        losses.append(float(loss.detach()))
    return (torch.tensor(losses, dtype=torch.float64),
            torch.tensor(logps, dtype=torch.float64) if targets is not None else None, torch.stack(grads))
