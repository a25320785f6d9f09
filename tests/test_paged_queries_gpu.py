"""Queries over 8-bit and bf16 pages whose numbers are far from 1, or far from one another: what the products see of them.

Tolerances. An output: half a bf16 step, 2^-8 |o|, and what the weights are off by times the largest |v|. With S = sum |q||k| a score is
off by at most 2^-17 S over bf16 rows (two bf16 parts), 2^-23 S and 2^-35 of the head's largest element times sum |k| over e4m3 rows (two
fp16 parts, whose smallest step is at most 2^-34 of the largest), and 2^-30 of the largest element times sum |k| over int8 rows (half a
whole number); fp32 sums add D 2^-23 S, int8 rows, whose sums are whole, eight roundings, 2^-20 S. Weights change by at most expm1 of
twice that, and by 2^-15 for their own two parts, the exponential's and the sums' error."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops import paged as P

from . import paged_oracle as O
from .test_paged_gpu import DEV, KINDS, poisoned

pytestmark = pytest.mark.gpu
QH, KVH, D, LEN = 8, 2, 128, 300


def attended(kind, k, v, kqv, scale, room):
    """(what the kernel makes of a token behind ``LEN`` rows, the definition over the rows that are held, its limits)"""
    pages = (LEN + 32) // 32
    table = torch.arange(pages, dtype=torch.int32)[None]
    table = torch.cat([table, torch.full((1, room), -1, dtype=torch.int32)], 1)
    cache = poisoned(pages, KVH, 32, D, kind)
    cos, sin = O.tables(LEN + 1, D, device=DEV)
    seq, pos = torch.zeros(LEN, dtype=torch.int32, device=DEV), torch.arange(LEN, dtype=torch.int32, device=DEV)
    P.paged_append(k.to(DEV, torch.bfloat16), v.to(DEV, torch.bfloat16), cache, table.to(DEV), seq, pos, cos, sin)
    kqv = kqv.to(torch.bfloat16)
    o = P.paged_attn_append(kqv.to(DEV), cache, table.to(DEV), torch.tensor([LEN], dtype=torch.int32, device=DEV), QH, KVH, cos, sin,
                            scale=scale)[0].cpu().double()
    k, v, there = O.cached(cache, table, 0, LEN + 1)
    assert bool(there.all())
    q = O.rotated(kqv[0].view(2 * KVH + QH, D)[KVH:KVH + QH], LEN)
    want = O.attend(q, k, v, LEN, torch.arange(LEN + 1), scale)
    tol = torch.zeros_like(want)
    for h in range(QH):
        kh, vh = k[:, h // (QH // KVH)].abs(), v[:, h // (QH // KVH)].abs()
        size = float((kh @ q[h].abs()).max()) * scale
        all_k = float(q[h].abs().max()) * float(kh.sum(-1).max()) * scale
        off = {"bf16": (2.0 ** -17 + D * 2.0 ** -23) * size,
               "int8": 2.0 ** -20 * size + 2.0 ** -30 * all_k,
               "e4m3": (2.0 ** -23 + D * 2.0 ** -23) * size + 2.0 ** -35 * all_k}[kind]
        tol[h] = 2.0 ** -8 * want[h].abs() + (math.expm1(2 * off) + 2.0 ** -15) * float(vh.max())
    return o, want, tol


def rows(seed, ratio=1.0):
    """K, V and the projection's row; the dims 5 and 70 of the queries, and the dims that the rotation pairs them with, are ``ratio``
    times the others, those of K as much smaller."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(LEN, KVH, D, generator=g) for _ in range(2))
    kqv = torch.randn(1, 2 * KVH + QH, D, generator=g)
    far = [5, 5 + D // 2, 70 - D // 2, 70]
    kqv[:, KVH:KVH + QH, far] *= ratio
    k[..., far] /= ratio
    kqv[:, :KVH, far] /= ratio
    return k * 1.5, v, kqv


@pytest.mark.parametrize("ratio", [30.0, 100.0, 1000.0])
@pytest.mark.parametrize("room", [1, 300])                   # clusters, and pieces that another kernel joins
def test_a_few_large_dims(ratio, room):
    """Heads as trained models have them, over int8 keys: the small dims count as much as the large ones."""
    k, v, kqv = rows(3, ratio)
    o, want, tol = attended("int8", k, v, kqv.flatten(1), 1 / math.sqrt(D), room)
    assert bool(((o - want).abs() <= tol).all()), (float(((o - want).abs() - tol).max()), float((o - want).abs().max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [126, 100, -90, -112])
def test_queries_near_the_ends_of_the_range(kind, power):
    """bf16 reaches from 2^-126 to 2^128; keys and the scale bring the scores back, as those of a model with such queries would be."""
    k, v, kqv = rows(1)
    q = kqv[:, KVH:KVH + QH]
    q.copy_(torch.sign(q) * (1 + 0.5 * torch.rand(q.shape, generator=torch.Generator().manual_seed(2))) * 2.0 ** power)
    left = 54 if power > 0 else -54                          # as far as scales go
    k, kqv[:, :KVH] = k * 2.0 ** (left - power), kqv[:, :KVH] * 2.0 ** (left - power)
    o, want, tol = attended(kind, k, v, kqv.flatten(1), 2.0 ** -left / math.sqrt(D), 1)
    assert float((want - want.mean()).abs().max()) > 0.05    # not the mean of V, which equal weights would give
    assert bool(((o - want).abs() <= tol).all()), (float(((o - want).abs() - tol).max()), float((o - want).abs().max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("room", [1, 300])
def test_keys_near_the_end_of_the_range(kind, room):
    """Keys of 2^120 and queries that bring the scores back: a score is finite, and so is all on the way to it."""
    k, v, kqv = rows(4)
    kqv[:, KVH:KVH + QH] *= 2.0 ** -110
    k, kqv[:, :KVH] = k * 2.0 ** 120, kqv[:, :KVH] * 2.0 ** 120
    o, want, tol = attended(kind, k, v, kqv.flatten(1), 2.0 ** -10 / math.sqrt(D), room)
    assert bool(((o - want).abs() <= tol).all()), (float(((o - want).abs() - tol).max()), float((o - want).abs().max()))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("room", [1, 300])
@pytest.mark.parametrize("order", ["turns", "last", "first"])
@pytest.mark.parametrize("power", [45, 70, 110])
def test_values_of_any_scale(kind, room, order, power):
    """Rows of V up to 2^110 beside rows of nothing, which count in the sum of weights all the same: in turns, the large ones in the last
    tiles alone, in the first alone."""
    k, v, kqv = rows(5)
    t = torch.arange(LEN)
    large = {"turns": t % 2 == 0, "last": t >= 270, "first": t < 40}[order]
    v = torch.where(large[:, None, None], v * 2.0 ** power, torch.where((t % 3 == 0)[:, None, None], v * 2.0 ** -70, torch.zeros(())))
    o, want, tol = attended(kind, k, v, kqv.flatten(1), 1 / math.sqrt(D), room)
    assert bool(((o - want).abs() <= tol).all()), (float(((o - want).abs() - tol).max()), float((o - want).abs().max()))
