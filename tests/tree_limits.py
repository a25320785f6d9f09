"""Tree attention from its definition in fp64, over the cache rows as the call left them, with limits close to the kernel's own roundings.

The kernel reads K and V of the drafts from the caches too, so of its inputs nothing is rounded but the rotated Q, which goes in as two
bf16 parts: what they leave is 2^-16 of a component at most, and fp32 sums of D <= 128 products add less than that again, so a score is
off by e = 2^-15 scale sum |q| |k| at most. Weights and results are rounded to bf16, U = 2^-8 of each at most:

  element by element   sum p (exp(2 e) - 1) |v| + 2 U sum p |v|
  root mean square     two independent roundings. Of a mantissa m in [1, 2) one is evenly spread over +-U / m of the value, and mantissas
                       of such values are spread as 1 / m, so the mean of 1 / m^2 is 3 / (8 ln 2) and a rounding
                       U sqrt(1 / (8 ln 2)) = 0.425 U: 0.6 U of the result's norm together (values V of random signs: sums of
                       p^2 v^2 are what both are made of)
"""
import math
import random

import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A

U = 2.0 ** -8
SLACK = 1.1
RMS = 1.15 * math.sqrt(2 / (8 * math.log(2))) * U

# name: (lens, drafts, QH, KVH, D, cap, biased, std of K | Q | V and the cache)
CASES = {
    "one token": ([1801, 90], 1, 16, 4, 128, 0.0, False, 1.2),
    "one token, large scores": ([1200, 77], 1, 16, 4, 128, 0.0, False, 2.0),
    "one token, capped": ([1801, 300], 1, 16, 4, 128, 6.0, False, 1.6),
    "one token, far beyond the cap": ([700], 1, 8, 2, 64, 1.0, False, 2.0),
    "tree of 16": ([500], 16, 12, 4, 64, 0.0, False, 0.8),
    "tree of 24": ([700, 0, 129], 24, 16, 4, 128, 0.0, False, 0.8),
    "large scores": ([400, 33], 12, 8, 4, 128, 0.0, False, 2.4),
    "two row tiles, capped": ([130, 1000, 0], 63, 16, 4, 128, 5.0, False, 1.6),
    "biased": ([300, 2000], 9, 8, 2, 64, 0.0, True, 0.9),
    "long": ([9000], 16, 4, 2, 64, 0.0, False, 0.7),
    "long, capped": ([9000], 8, 4, 2, 128, 4.0, False, 1.5),
}


def make(name, dev):
    """Inputs of a case: made on the CPU, the same on every device. Rows behind the cached tokens may hold anything."""
    lens, n, QH, KVH, D, cap, biased, std = CASES[name]
    rng, g = random.Random(name), torch.Generator().manual_seed(len(name))
    B, Tmax = len(lens), max(lens) + n + 3
    parents = [[-1] + [rng.randrange(-1, i) for i in range(1, n)] for _ in range(B)]
    kqv = (torch.randn(B * n, (2 * KVH + QH) * D, generator=g) * std).to(torch.bfloat16)
    kc, vc = ((torch.randn(B, KVH, Tmax, D, generator=g) * s).to(torch.bfloat16) for s in (std, 1.0))
    for b, L in enumerate(lens):
        kc[b, :, L:], vc[b, :, L:] = math.nan, math.inf
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / QH) for h in range(QH)]) if biased else None
    cos, sin = F.rope_table(Tmax, D, 10000.0, "cpu")
    to = lambda x: x if x is None else x.to(dev)           # noqa: E731
    return dict(kqv=to(kqv), kcache=to(kc), vcache=to(vc), lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                tree=A.tree_mask(parents, dev), QH=QH, KVH=KVH, cos=to(cos), sin=to(sin), softcap=cap, slopes=to(slopes)), parents


def rows_of(a, parents, b):
    """(rotated Q [n, QH, D], rotated K [n, KVH, D], V [n, KVH, D], sees [n, L + n], query and key positions) of sequence ``b``, fp64."""
    n, QH, KVH = a["tree"].shape[1], a["QH"], a["KVH"]
    D, L, dev = a["kcache"].shape[3], int(a["lens"][b]), a["kqv"].device
    anc, depth = [], []
    for i, par in enumerate(parents[b]):
        anc.append((anc[par] if par >= 0 else []) + [i])
        depth.append(len(anc[i]) - 1)
    pos = L + torch.tensor(depth, device=dev)
    x = a["kqv"].double().view(-1, n, 2 * KVH + QH, D)[b]
    c, s = a["cos"][pos].double()[:, None], a["sin"][pos].double()[:, None]
    y, z = x[..., :D // 2], x[..., D // 2:]
    turned = torch.cat([y * c - z * s, z * c + y * s], -1)
    sees = torch.zeros(n, L + n, dtype=torch.bool, device=dev)
    sees[:, :L] = True
    for i in range(n):
        sees[i, [L + j for j in anc[i]]] = True
    return turned[:, KVH:KVH + QH], turned[:, :KVH], x[:, KVH + QH:], sees, pos, torch.cat([torch.arange(L, device=dev), pos])


def attention(a, parents, q_of=lambda q: q, p_of=lambda p: p, cap=None, lost=None):
    """([B, n, QH, D] results, bounds) over the caches as they are. ``q_of`` and ``p_of`` make other queries and weights of them, ``cap``
    another cap, ``lost`` leaves out a position: what a check has to notice."""
    B, n = a["tree"].shape
    QH, D = a["QH"], a["kcache"].shape[3]
    R, scale, cap = QH // a["KVH"], 1 / math.sqrt(D), a["softcap"] if cap is None else cap
    o = torch.zeros(B, n, QH, D, dtype=torch.float64, device=a["kqv"].device)
    bound = torch.zeros_like(o)
    for b in range(B):
        q, _, _, sees, pos, kpos = rows_of(a, parents, b)
        m = sees.shape[1]
        if lost is not None:
            sees = sees.clone()
            sees[:, lost] = False
        for h in range(QH):
            kk, vv = a["kcache"][b, h // R, :m].double(), a["vcache"][b, h // R, :m].double()
            x = q_of(q[:, h]) @ kk.T * scale
            e = 2.0 ** -15 * scale * (q[:, h].abs() @ kk.abs().T)
            if cap:
                x = cap * torch.tanh(x / cap)
            if a["slopes"] is not None:
                x = x - float(a["slopes"][h]) * (pos[:, None] - kpos[None]).abs()
            x = x.masked_fill(~sees, -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            total = p.sum(-1, keepdim=True)
            o[b, :, h] = (p_of(p) @ vv) / total
            p = p / total
            bound[b, :, h] = SLACK * ((p * torch.expm1(2 * e)) @ vv.abs() + 2 * U * (p @ vv.abs()))
    return o, bound


def good(got, want, bound):
    """Whether results keep both limits."""
    off = got.double() - want
    return bool((off.abs() <= bound + 1e-6).all()) and float(off.norm()) <= RMS * float(want.norm())
