"""What the paged cache and the verification of drafts compute, in fp64, token by token: written from the definitions."""
import math

import torch

LARGEST = {"int8": 127.0, "e4m3": 448.0}


def held(x, kind):
    """fp64 rows [..., D] as they are held: (values, scales or None)."""
    x = x.double()
    if kind == "bf16":
        return x.to(torch.bfloat16).double(), None
    s = torch.clamp(x.abs().amax(-1) / LARGEST[kind], min=2.0 ** -80)
    y = x / s[..., None]
    y = torch.round(y) if kind == "int8" else y.float().to(torch.float8_e4m3fn).double()
    return y * s[..., None], s


def step(kind):
    """How far a held value may be from its row's element: half a step of bf16 or e4m3 relative to the element (of e4m3 also half of its
    smallest step, 2^-9 of a scale), of int8 relative to the row's largest. On top of that what fp32 does to a rotated pair (a, b): each
    table entry, product and sum is off by half a step, together 3 2^-24 (|a| + |b|), and |a|, |b| are at most sqrt(2) times the largest
    of the rotated row, so 2^-20 of that covers it, and the scale's and the quotient's roundings with it. Rows of nearly nothing have
    the least scale, 2^-80."""
    def of(x):
        most = x.abs().amax(-1, keepdim=True)
        if kind == "bf16":
            return x.abs() * 2.0 ** -8 + most * 2.0 ** -20
        if kind == "int8":
            return most * (0.5 / 127 + 2.0 ** -20) + 2.0 ** -81
        return torch.maximum(x.abs() * 2.0 ** -4, torch.clamp(most / 448, min=2.0 ** -80) * 2.0 ** -10) + most * 2.0 ** -20
    return of


def rotated(x, pos, base=10000.0):
    """x [..., D] at fp64 position ``pos``: half-split pairs."""
    D = x.shape[-1]
    a = torch.as_tensor(pos, dtype=torch.float64) * base ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)
    c, s = torch.cos(a), torch.sin(a)
    lo, hi = x[..., :D // 2].double(), x[..., D // 2:].double()
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def tables(n, D, base=10000.0, device="cpu"):
    a = torch.arange(n, dtype=torch.float64)[:, None] * base ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)
    return torch.cos(a).float().to(device), torch.sin(a).float().to(device)


def cached(cache, table, b, n):
    """fp64 (K, V) [n, KVH, D] of sequence b's first n tokens as the pool holds them, and which of them are there."""
    pages, KVH, page, D = cache.k.shape
    t = torch.arange(n)
    ok = t < table.shape[1] * page
    at = torch.where(ok, table[b].cpu().long()[(t // page).clamp_max(table.shape[1] - 1)], -1)
    there = (at >= 0) & (at < pages)
    out = []
    for x, s in zip(cache[:2], cache[2:]):
        x = x.cpu()[torch.unique(at[there])].double() if n else x.cpu()[:0].double()
        nth = torch.searchsorted(torch.unique(at[there]), at[there])
        rows = torch.zeros(n, KVH, D, dtype=torch.float64)
        rows[there] = x[nth, :, t[there] % page]
        if s is not None:
            rows[there] *= s.cpu().double()[at[there], :, t[there] % page, None]
        out.append(rows)
    return out[0], out[1], there


def attend(q, k, v, pos, key_pos, scale, cap=0.0, slopes=None):
    """q [QH, D] over k, v [n, KVH, D]: [QH, D], zeros over nothing."""
    QH, (n, KVH, D) = q.shape[0], k.shape
    o = torch.zeros(QH, D, dtype=torch.float64)
    if n == 0:
        return o
    for h in range(QH):
        x = k[:, h // (QH // KVH)] @ q[h].double() * scale
        if cap:
            x = cap * torch.tanh(x / cap)
        if slopes is not None:
            x = x - float(slopes[h]) * (pos - key_pos).double()
        o[h] = torch.softmax(x, 0) @ v[:, h // (QH // KVH)]
    return o


def verify(logits, tokens, parents, u, temp, top, q=None, accept=None):
    """Lists (tokens, path) per sequence: one walk down each tree, probabilities as they are defined."""
    got = []
    B, n, V = logits.shape
    for b in range(B):
        node, out, path = 0, [], []
        while True:
            x = logits[b, node].double()
            x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x).clamp_max(3.4028234663852886e38)
            if bool((x == -math.inf).all()):
                out.append(-1)
                break
            if temp == 0:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1
            else:
                p = torch.softmax((x - x.max()) / temp, 0)
                order = sorted(range(V), key=lambda j: (-float(x[j]), j))
                mass, kept = 0.0, []
                for j in order:
                    if mass >= top:
                        break
                    kept.append(j)
                    mass += float(p[j])
                if top < 1:
                    cut = torch.zeros_like(p)
                    cut[kept] = p[kept]
                    p = cut / cut.sum()
            kids, go = [j for j in range(node + 1, n) if int(parents[b, j]) == node], None
            whole = p
            if q is not None:
                for j in kids:
                    t = int(tokens[b, j])
                    if not 0 <= t < V:
                        continue
                    if float(accept[b, j]) * float(q[b, node, t]) < float(p[t]):
                        go = j
                        break
                    left = (p - q[b, node].double()).clamp_min(0)
                    if float(left.sum()) <= 0:
                        p = whole
                        break
                    p = left / left.sum()
            if go is None:
                sums = torch.cumsum(p, 0) / p.sum()
                t = min(int((sums <= float(u[b, node])).sum()), int(p.nonzero()[-1]))
                if q is None:
                    go = next((j for j in kids if int(tokens[b, j]) == t), None)
            if go is None:
                out.append(t)
                break
            out.append(int(tokens[b, go]))
            path.append(go)
            node = go
        got.append((out, path))
    return got
