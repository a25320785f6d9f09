"""Drafts that do not fit behind the cached tokens, in the plain restatement: the result is that of the keys that were kept."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A


@pytest.mark.parametrize("room", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (3.0, False), (0.0, True)])
def test_results_of_drafts_that_do_not_fit(room, softcap, bias):
    g = torch.Generator().manual_seed(room)
    QH, KVH, D, n, L = 4, 2, 8, 4, 5
    Tmax, parents = L + room, [-1, 0, 0, 2]
    cos, sin = F.rope_table(L + n, D, 10000.0, "cpu")
    kqv = torch.randn(n, (2 * KVH + QH) * D, generator=g, dtype=torch.float64)
    kc, vc = (torch.randn(1, KVH, Tmax, D, generator=g, dtype=torch.float64) for _ in range(2))
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625]) if bias else None
    got = A.tree_attn_append(kqv, kc, vc, torch.tensor([L], dtype=torch.int32), A.tree_mask([parents], "cpu"), QH, KVH, cos, sin,
                             softcap=softcap, slopes=slopes)
    anc, depth = [], []
    for i, par in enumerate(parents):
        anc.append((anc[par] if par >= 0 else []) + [i])
        depth.append(len(anc[i]) - 1)
    for i in range(n):
        at = list(range(L)) + [L + j for j in anc[i] if j < room]
        kpos = torch.tensor(list(range(L)) + [L + depth[j] for j in anc[i] if j < room])
        pos = L + depth[i]
        q = kqv.view(n, 2 * KVH + QH, D)[i, KVH:KVH + QH]
        c, s = cos[pos].double(), sin[pos].double()
        q = torch.cat([q[:, :4] * c - q[:, 4:] * s, q[:, 4:] * c + q[:, :4] * s], -1)
        for h in range(QH):
            x = kc[0, h // 2, at] @ q[h] / math.sqrt(D)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            if bias:
                x = x - float(slopes[h]) * (pos - kpos).abs()
            assert torch.allclose(got[0, i, h], torch.softmax(x, 0) @ vc[0, h // 2, at], atol=1e-10)
