"""Definitions in 64 bits of the operators that move rows by sorted indices, written as loops over rows."""

import torch


def embedding(tokens, w, scale, first=0):
    out = torch.zeros(*tokens.shape, w.shape[1], dtype=torch.float64)
    flat = out.view(-1, w.shape[1])
    for i, t in enumerate(tokens.reshape(-1).tolist()):
        if 0 <= t - first < w.shape[0]:
            flat[i] = scale * w[t - first].double()
    return out


def embedding_grad(tokens, g, rows, scale, first=0):
    """(gradient, sum of the magnitudes, number of terms of each row)"""
    g = g.double().reshape(-1, g.shape[-1])
    total = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    size = torch.zeros_like(total)
    many = torch.zeros(rows, 1, dtype=torch.float64)
    for i, t in enumerate(tokens.reshape(-1).tolist()):
        if 0 <= t - first < rows:
            total[t - first] += g[i] * scale
            size[t - first] += g[i].abs() * abs(scale)
            many[t - first] += 1
    return total, size, many


def route(z, k, normalize):
    """(weights, experts): NaN ranks highest, ties at the lowest index, a row of nothing but -inf has weights 0."""
    z = z.double()
    w = torch.zeros(z.shape[0], k, dtype=torch.float64)
    ids = torch.zeros(z.shape[0], k, dtype=torch.int64)
    for r, row in enumerate(z.tolist()):
        order = sorted(range(len(row)), key=lambda e: (0, 0.0, e) if row[e] != row[e] else (1, -row[e], e))[:k]
        ids[r] = torch.tensor(order)
        top = row[order[0]]
        if top == float("-inf"):
            continue
        zr = z[r]
        ex = (zr - top).exp()
        den = ex[order].sum() if normalize else ex.sum()
        w[r] = ex[order] / den
    return w, ids


def route_grad(z, ids, g, normalize):
    z = z.double().clone().requires_grad_(True)
    dead = (z.detach() == float("-inf")).all(1)
    p = z.masked_fill(dead[:, None], 0.0)
    w = p.gather(1, ids).softmax(1) if normalize else p.softmax(1).gather(1, ids)
    (dz,) = torch.autograd.grad((w * g.double() * ~dead[:, None]).sum(), z)
    return dz


def plan(experts, E, align):
    counts = [0] * E
    flat = experts.reshape(-1).tolist()
    for e in flat:
        if 0 <= e < E:
            counts[e] += 1
    offs = [0]
    for c in counts:
        offs.append(offs[-1] + -(-c // align) * align)
    seen, rows = [0] * E, []
    for e in flat:
        if 0 <= e < E:
            rows.append(offs[e] + seen[e])
            seen[e] += 1
        else:
            rows.append(-1)
    return rows, offs, counts


def dispatch(x, rows, k, cap):
    out = torch.zeros(cap, x.shape[1], dtype=torch.float64)
    for j, r in enumerate(rows):
        if r >= 0:
            out[r] = x[j // k].double()
    return out


def combine(y, w, rows, k, residual, n):
    """(sums, sum of the magnitudes)"""
    out = torch.zeros(n, y.shape[1], dtype=torch.float64) if residual is None else residual.double().clone()
    size = out.abs()
    for j, r in enumerate(rows):
        if r >= 0:
            v = y[r].double() * (1.0 if w is None else w.reshape(-1)[j].double())
            out[j // k] += v
            size[j // k] += v.abs()
    return out, size


def combine_grad(g, y, w, rows, k):
    """(dy, dw, sum of the magnitudes behind dw)"""
    dy = torch.zeros(y.shape, dtype=torch.float64)
    dw = torch.zeros(len(rows), dtype=torch.float64)
    size = torch.zeros(len(rows), dtype=torch.float64)
    for j, r in enumerate(rows):
        if r >= 0:
            gj = g[j // k].double()
            dy[r] = w.reshape(-1)[j].double() * gj
            dw[j] = (gj * y[r].double()).sum()
            size[j] = (gj * y[r].double()).abs().sum()
    return dy, dw.view(w.shape), size.view(w.shape)
