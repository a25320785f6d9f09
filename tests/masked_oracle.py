"""Span and tree attention from their definitions, in fp64, with a bound on what the kernels' roundings can make of the results.

The kernels take bf16 operands, form scores and all sums in fp32 and round three things to bf16 (8 significant bits: half a unit in the
last place is U = 2^-8 of the value at most): the weights P
before they meet V, dS before it meets K and Q, and the results. From that, element by element:

  o      weights and result              (2 U) sum p |v|
  dv     weights and result              (2 U) sum p |do|
  delta  = sum do o of the rounded o     e = sum |do| (err o), so dS is off by p scale (U (|dp| + |delta|) + e), and by U of itself
                                         again where the kept P was rounded (U in all: twice), and by its own rounding (U)
  dq, dk                                 sum (err dS) |k|, |q| and U of the result

Scores are exact products with fp32 sums; what they and the exponentials add is far below U and covered by SLACK.
"""
import math

import torch

U = 2.0 ** -8
SLACK = 1.1
TINY = 1e-6


def span_oracle(q, k, v, seen, scale, softcap=0.0, slopes=None, dout=None, dist=None):
    """q [B, T, QH, D], k, v [B, S, KVH, D], seen bool [B, T, S]; ``dist`` [B, T, S] distances for ``slopes`` (default |t - s|). Returns a
    dict of (value, bound) in fp64."""
    B, T, QH, D = q.shape
    S, KVH = k.shape[1:3]
    R = QH // KVH
    q, k, v = (x.double() for x in (q, k, v))
    if dist is None:
        dist = (torch.arange(T, device=q.device)[:, None] - torch.arange(S, device=q.device)[None]).abs()[None].expand(B, T, S)
    res = {n: torch.zeros(B, T, QH, D, dtype=torch.float64, device=q.device) for n in ("o", "o_b", "dq", "dq_b")}
    res.update({n: torch.zeros(B, S, KVH, D, dtype=torch.float64, device=q.device) for n in ("dk", "dk_b", "dv", "dv_b")})
    res["lse"] = torch.full((B, QH, T), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        for h in range(QH):
            g = h // R
            x = q[b, :, h] @ k[b, :, g].T * scale
            one = torch.ones_like(x)
            if softcap:
                th = torch.tanh(x / softcap)
                x, one = softcap * th, 1 - th * th
            if slopes is not None:
                x = x - float(slopes[h]) * dist[b].double()
            x = torch.where(seen[b], x, torch.full_like(x, -math.inf))
            lse = torch.logsumexp(x, -1)
            p = torch.where(seen[b], torch.exp(x - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(x))
            vv, kk, qq = v[b, :, g], k[b, :, g], q[b, :, h]
            res["lse"][b, h] = lse
            o = p @ vv
            o_b = 2 * U * SLACK * (p @ vv.abs())
            res["o"][b, :, h], res["o_b"][b, :, h] = o, o_b
            if dout is None:
                continue
            do = dout[b, :, h].double()
            dp, delta = do @ vv.T, (do * o).sum(-1, keepdim=True)
            e = (do.abs() * o_b).sum(-1, keepdim=True)
            ds = p * one * (dp - delta) * scale
            ds_b = SLACK * (p * one * scale * (2 * U * (dp.abs() + delta.abs()) + e) + U * ds.abs())
            res["dq"][b, :, h] = ds @ kk
            res["dq_b"][b, :, h] = ds_b @ kk.abs() + U * (ds @ kk).abs()
            res["dk"][b, :, g] += ds.T @ qq
            res["dk_b"][b, :, g] += ds_b.T @ qq.abs()
            res["dv"][b, :, g] += p.T @ do
            res["dv_b"][b, :, g] += 2 * U * SLACK * (p.T @ do.abs())
    res["dk_b"] += U * res["dk"].abs()
    return res


def within(got, want, bound, what):
    got = got.double().to(want.device)
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    over = (got - want).abs() - bound - TINY
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0, f"{what}: {worst} beyond its bound"


def tree_oracle(kqv, kcache, vcache, lens, parents, QH, KVH, cos, sin, scale, softcap=0.0, slopes=None):
    """Draft by draft: parents[b][i] is the draft that draft i continues, -1 none, None a draft that sees the cached tokens alone. Returns
    ([B, n, QH, D] results, bound, the caches as they should be afterwards)."""
    B, KVH_, Tmax, D = kcache.shape
    n, R = kqv.shape[0] // B, QH // KVH
    kc, vc = kcache.double().clone(), vcache.double().clone()
    o = torch.zeros(B, n, QH, D, dtype=torch.float64, device=kqv.device)
    bound = torch.zeros_like(o)
    rows = kqv.double().view(B, n, 2 * KVH + QH, D)
    for b in range(B):
        L = int(lens[b])
        anc, depth = [], []
        for i in range(n):
            par = parents[b][i]
            anc.append([] if par is None else (anc[par] if par >= 0 else []) + [i])
            depth.append(max(len(anc[i]) - 1, 0))
        pos = torch.tensor([L + x for x in depth], dtype=torch.float64, device=kqv.device)
        at = pos.long().clamp_max(cos.shape[0] - 1)
        c, s = cos[at].double()[:, None], sin[at].double()[:, None]
        a, z = rows[b, ..., :D // 2], rows[b, ..., D // 2:]
        turned = torch.cat([a * c - z * s, z * c + a * s], -1)
        keep = max(0, min(n, Tmax - L))
        kc[b, :, L:L + keep] = turned[:keep, :KVH].transpose(0, 1)
        vc[b, :, L:L + keep] = rows[b, :keep, KVH + QH:].transpose(0, 1)
        for i in range(n):
            at = list(range(L)) + [L + j for j in anc[i]]
            if not at:
                continue
            kpos = torch.tensor(list(range(L)) + [L + depth[j] for j in anc[i]], dtype=torch.float64, device=kqv.device)
            for h in range(QH):
                g = h // R
                kk, vv, qq = kc[b, g][at].to(torch.bfloat16).double(), vc[b, g][at], turned[i, KVH + h]
                x = kk @ qq * scale
                # q is rounded to bf16, and a key to the cache's type from fp32 (U of one of the two more, where that rounds the other way)
                e = 2 * U * (kk.abs() @ qq.abs()) * scale
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                if slopes is not None:
                    x = x - float(slopes[h]) * (pos[i] - kpos).abs()
                p = torch.softmax(x, -1)
                o[b, i, h] = p @ vv
                # scores off by e_j: a weight by the factor exp(e_j) / sum p exp(e)
                worst = torch.exp(e) * (p @ torch.exp(e)) - 1
                bound[b, i, h] = SLACK * ((p * worst) @ vv.abs() + 2 * U * (p @ vv.abs()))
    return o, bound, kc, vc
