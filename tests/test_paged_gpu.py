"""The paged cache's kernels against the definitions in fp64, on the rows that the cache holds.

Tolerances. A held value: half a step (``paged_oracle.step``). An output: half a bf16 step, 2^-8 |o|, and what the weights are off by
times the largest |v|. A score's error is at most (2^-16 + D 2^-23) sum |q||k| (Q in two bf16 parts and fp32 sums; two fp16 parts are
finer); over int8 rows Q is rounded to whole numbers of 1 / 32512 of its largest, off by half of one, so that 1 / 65024 of the largest
times sum |k| comes on top. A bias's or cap's is 2^-21 of the largest score. Weights change by at most expm1 of twice that, and by 2^-15
for their own two parts, the exponential's and the sums' error."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops import native
from create_llm_by_cupy_b200.ops import paged as P

from . import paged_oracle as O

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "int8", "e4m3"]
DEV = "cuda"


def poisoned(pages, KVH, page, D, kind):
    """A pool in which nothing is a number."""
    c = P.paged_cache(pages, KVH, page, D, DEV, kind)
    for x in c:
        if x is None:
            continue
        if x.dtype == torch.float8_e4m3fn:
            x.view(torch.uint8).fill_(0x7f)
        elif x.dtype == torch.int8:
            x.fill_(-128)
        else:
            x.fill_(math.nan)
    return c


def filled(kind, lens, KVH, D, page, seed=0, room=1, rows=None):
    """Cached sequences whose pages stand in random order in a poisoned pool; their un-rotated K and V on the CPU."""
    g = torch.Generator().manual_seed(seed)
    B, width = len(lens), max(max(lens), 0) // page + room
    pages = B * width + 2
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32)
    cache = poisoned(pages, KVH, page, D, kind)
    kqv = (torch.randn(sum(max(n, 0) for n in lens), 3 * KVH * D, generator=g) * 1.5).to(torch.bfloat16)
    seq = torch.cat([torch.full((max(n, 0),), b, dtype=torch.int32) for b, n in enumerate(lens)])
    pos = torch.cat([torch.arange(max(n, 0), dtype=torch.int32) for n in lens])
    cos, sin = O.tables(rows or width * page, D, device=DEV)
    x = kqv.to(DEV)
    k, v = x[:, :KVH * D].unflatten(1, (KVH, D)), x[:, 2 * KVH * D:].unflatten(1, (KVH, D))
    P.paged_append(k, v, cache, table.to(DEV), seq.to(DEV), pos.to(DEV), cos, sin)
    return cache, table, k.cpu(), v.cpu(), seq, pos, cos, sin


def same(a, b):
    return all(x is None and y is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def check_token(cache, table, kqv, o, lens, QH, KVH, D, cap=0.0, slopes=None, cos_rows=1 << 30):
    """``o`` against the definition over the rows that the cache holds now."""
    kqv, o, page = kqv.cpu(), o.cpu().double(), cache.k.shape[2]
    scale = 1 / math.sqrt(D)
    for b, n in enumerate(lens):
        if n < 0:
            assert bool((o[b] == 0).all())
            continue
        rows = kqv[b].view(2 * KVH + QH, D)
        kept = n < table.shape[1] * page and n < cos_rows
        k, v, there = O.cached(cache, table, b, n + 1 if kept else min(n, table.shape[1] * page))
        at = torch.arange(len(there))[there]
        k, v = k[there], v[there]
        q = O.rotated(rows[KVH:KVH + QH], min(n, cos_rows - 1))
        if kept and bool(there[n]):
            for got, want in ((k[-1], O.rotated(rows[:KVH], n)), (v[-1], rows[KVH + QH:].double())):
                kind = {torch.int8: "int8", torch.float8_e4m3fn: "e4m3"}.get(cache.k.dtype, "bf16")
                assert bool(((got - want).abs() <= O.step(kind)(want)).all())
        want = O.attend(q, k, v, n, at, scale, cap, slopes)
        if len(at) == 0:
            assert bool((o[b] == 0).all())
            continue
        for h in range(QH):
            size = float((k[:, h // (QH // KVH)].abs() @ q[h].abs()).max()) * scale
            big = size + (0 if slopes is None else float(slopes[h]) * n)
            off = (2.0 ** -16 + D * 2.0 ** -23) * size + 2.0 ** -21 * big
            if cache.k.dtype == torch.int8:
                off += float(q[h].abs().max()) / 65024 * float(k[:, h // (QH // KVH)].abs().sum(-1).max()) * scale
            tol = 2.0 ** -8 * want[h].abs() + (math.expm1(2 * off) + 2.0 ** -15) * float(v[:, h // (QH // KVH)].abs().max())
            assert bool(((o[b, h] - want[h]).abs() <= tol).all()), (b, h, float((o[b, h] - want[h]).abs().max()), float(tol.max()))


# --------------------------------------------------------------------------- rows in and out
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [32, 128])
def test_append_and_read(kind, D, page):
    lens, KVH = [1, 131, 0, 97], 3
    cache, table, k, v, seq, pos, cos, sin = filled(kind, lens, KVH, D, page)
    m = 0
    for b, n in enumerate(lens):
        kk, vv, there = O.cached(cache, table, b, n)
        assert bool(there.all())
        for t in range(n):
            for got, want in ((kk[t], O.rotated(k[m], t)), (vv[t], v[m].double())):
                assert bool(((got - want).abs() <= O.step(kind)(want)).all())
            m += 1
    start = torch.tensor([0, 100, 0, 96], dtype=torch.int32, device=DEV)
    for first in (None, start):
        kc, vc = (torch.full((4, KVH, 120, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        P.paged_read(cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), kc, vc, start=first)
        for b, n in enumerate(lens):
            s = 0 if first is None else int(first[b])
            rows = max(0, min(120, n - s))
            for got, x in zip((kc, vc), O.cached(cache, table, b, n)):
                want = x[s:s + rows].transpose(0, 1)             # fp32 product, rounded once more
                assert bool(((got[b, :, :rows].cpu().double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all())
                assert bool((got[b, :, rows:] == 7.0).all())


@pytest.mark.parametrize("kind", KINDS)
def test_append_leaves_out_what_has_no_place(kind):
    KVH, D, page = 2, 128, 32
    cache = poisoned(4, KVH, page, D, kind)
    before = [None if x is None else x.clone() for x in cache]
    table = torch.tensor([[0, 4], [-1, 1]], dtype=torch.int32, device=DEV)
    x = torch.randn(9, KVH, D, device=DEV).to(torch.bfloat16)
    cos, sin = O.tables(60, D, device=DEV)
    seq = torch.tensor([-1, 2, 0, 0, 1, 1, 1, 0, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([0, 0, 40, 64, 3, 60, -1, 2 ** 31 - 1, 63], dtype=torch.int32, device=DEV)
    P.paged_append(x, x, cache, table, seq, pos, cos, sin)
    assert same(cache, before)
    P.paged_append(x, x, cache, table, seq, pos)             # without a rotation only the pages are the limit: positions 60 and 63
    assert not same(cache, before)
    back = [None if y is None else y.view(torch.uint8).clone() for y in cache]
    for y, z in zip(back, before):
        if y is not None:
            y.view(y.shape)[1].copy_(z.view(torch.uint8)[1])
            assert torch.equal(y, z.view(torch.uint8))
    kc = torch.full((2, KVH, 100, D), 7.0, dtype=torch.bfloat16, device=DEV)
    P.paged_read(cache, table, torch.tensor([100, 100], dtype=torch.int32, device=DEV), kc, kc.clone(),
                 start=torch.tensor([32, -5], dtype=torch.int32, device=DEV))
    assert bool((kc[0] == 7).all()) and bool((kc[1, :, :32] == 7).all()) and bool((kc[1, :, 64:] == 7).all())
    assert bool((kc[1, :, 60] == x[5]).all()) if kind == "bf16" else bool(torch.isfinite(kc[1, :, 60]).all())


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_any_pitch_and_extreme_rows(kind):
    KVH, D = 2, 64
    table = torch.zeros((1, 1), dtype=torch.int32, device=DEV)
    rows = torch.randn(6, KVH, D, device=DEV)
    rows[1], rows[2], rows[3] = 0.0, 1e-30, 3e38
    rows[4, :, 1:] *= 1e-4
    rows = rows.to(torch.bfloat16)
    seq, pos = torch.zeros(6, dtype=torch.int32, device=DEV), torch.arange(6, dtype=torch.int32, device=DEV)
    def behind(n):                                           # in a matrix whose first n columns are something else
        return torch.cat([torch.zeros(6, n, dtype=torch.bfloat16, device=DEV), rows.flatten(1)], 1)[:, n:].unflatten(1, (KVH, D))

    views = [rows, torch.stack([rows, rows], 2)[:, :, 0], behind(8), behind(1)]
    got = []
    for x in views:
        cache = P.paged_cache(1, KVH, 32, D, DEV, kind)
        P.paged_append(x, x, cache, table, seq, pos)
        got.append(cache)
        assert same(cache, got[0])
    k, _, _ = O.cached(got[0], table, 0, 6)
    want = rows.cpu().double()
    assert bool(((k - want).abs() <= O.step(kind)(want)).all())


# --------------------------------------------------------------------------- attention of a token
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("QH,KVH", [(12, 4), (32, 8), (3, 3), (16, 1), (20, 2)])
@pytest.mark.parametrize("room", [1, 20])                    # tables of 320 tokens, and of 928: larger clusters
def test_token(kind, D, QH, KVH, room):
    lens = [0, 1, 15, 16, 31, 32, 33, 127, 128, 300, -1]
    cache, table, *_, cos, sin = filled(kind, lens, KVH, D, 32, seed=QH, room=room)
    kqv = (torch.randn(len(lens), (2 * KVH + QH) * D, generator=torch.Generator().manual_seed(1)) * 1.5).to(torch.bfloat16).to(DEV)
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos, sin)
    check_token(cache, table, kqv, o, lens, QH, KVH, D)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mod", ["cap", "far cap", "bias"])
@pytest.mark.parametrize("D", [64, 128])
def test_token_with_modified_scores(kind, mod, D):
    QH, KVH, lens = 12, 4, [700, 5, 64]
    cache, table, *_, cos, sin = filled(kind, lens, KVH, D, 64)
    kqv = (torch.randn(3, (2 * KVH + QH) * D) * 1.5).to(torch.bfloat16).to(DEV)
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / QH) for h in range(QH)], device=DEV) if mod == "bias" else None
    cap = {"cap": 30.0, "far cap": 0.5, "bias": 0.0}[mod]
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos, sin, softcap=cap,
                            slopes=slopes)
    check_token(cache, table, kqv, o, lens, QH, KVH, D, cap, None if slopes is None else slopes.cpu())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,hi,page", [(1, 9000, 128), (3, 4100, 256), (1, 1, 1024), (40, 260, 32), (40, 700, 32), (150, 70, 64),
                                       (700, 40, 1024)])
def test_token_of_long_and_of_many_sequences(kind, B, hi, page):
    QH, KVH, D = 16, 4, 128
    lens = [hi - 61 * b % hi for b in range(B)]
    cache, table, *_, cos, sin = filled(kind, lens, KVH, D, page)
    kqv = (torch.randn(B, (2 * KVH + QH) * D) * 1.5).to(torch.bfloat16).to(DEV)
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos, sin)
    some = sorted({0, 1 % B, B // 2, B - 1})
    check_token(cache, table[some], kqv[some], o[some], [lens[b] for b in some], QH, KVH, D)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
def test_token_in_pieces(kind, D, mod):
    """Few sequences with room for many tokens: empty ones, one that is none, short and long ones; four groups of heads."""
    QH, KVH, lens = 16, 1, [0, 5, -1, 2600]
    cache, table, *_, cos, sin = filled(kind, lens, KVH, D, 64)
    kqv = (torch.randn(4, (2 * KVH + QH) * D, generator=torch.Generator().manual_seed(2)) * 1.5).to(torch.bfloat16).to(DEV)
    slopes = torch.tensor([2.0 ** (-(h + 1) / 2) for h in range(QH)], device=DEV) if mod == "bias" else None
    cap = 20.0 if mod == "cap" else 0.0
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos, sin, softcap=cap,
                            slopes=slopes)
    check_token(cache, table, kqv, o, lens, QH, KVH, D, cap, None if slopes is None else slopes.cpu())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("room", [1, 80])                    # clusters, and pieces that another kernel joins
def test_pages_that_are_not_there(kind, room):
    QH, KVH, D, page, lens = 8, 2, 128, 32, [200, 200, 95, 64]
    cache, table, *_, cos, sin = filled(kind, lens, KVH, D, page, room=room)
    table[0, 1], table[0, 3], table[1, :] = -1, cache.k.shape[0], -7
    table[2, 2] = 2 ** 31 - 1                                # a page that the new token would be written to
    kqv = (torch.randn(4, (2 * KVH + QH) * D) * 1.5).to(torch.bfloat16).to(DEV)
    before = [None if x is None else x.clone() for x in cache]
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos[:64], sin[:64])
    assert same(cache, before)                               # 64 rotary positions: no token is kept
    check_token(cache, table, kqv, o, lens, QH, KVH, D, cos_rows=64)
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos, sin)
    check_token(cache, table, kqv, o, lens, QH, KVH, D)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_queries_of_any_magnitude(kind, size):
    """Scores of 0, or as large as numbers go, where the weight is one token's: the scale brings them back."""
    QH, KVH, D, lens = 4, 1, 128, [70]
    cache, table, *_, cos, sin = filled(kind, lens, KVH, D, 32)
    kqv = torch.randn(1, (2 * KVH + QH) * D, generator=torch.Generator().manual_seed(5))
    kqv[:, KVH * D:(KVH + QH) * D] *= size
    kqv = kqv.to(DEV, torch.bfloat16)
    scale = 1e-18 if size > 1 else 1e18
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos, sin, scale=scale)
    k, v, _ = O.cached(cache, table, 0, 71)
    q = O.rotated(kqv.cpu()[0].view(2 * KVH + QH, D)[KVH:KVH + QH], 70)
    want = O.attend(q, k, v, 70, torch.arange(71), scale)
    x = k[:, 0] @ q.T * scale                                # scores of 10^12 apart from one another, or of nothing
    clear = (x.topk(2, 0).values.diff(dim=0).abs()[0] > 1e-3 * x.abs().max()) | (x.abs().max() < 1e-6)
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -14 * v.abs().max()
    assert bool(torch.isfinite(o).all()) and bool(clear.any())
    assert bool(((o[0].cpu().double() - want).abs() <= tol)[clear].all())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_rows_of_very_different_scales(kind):
    """Sequences in which a few rows of V are 10^6 times the others, or 0, and large queries."""
    QH, KVH, D, lens = 8, 2, 128, [150]
    g = torch.Generator().manual_seed(3)
    table = torch.arange(5, dtype=torch.int32)[None]
    cache = poisoned(5, KVH, 32, D, kind)
    k, v = (torch.randn(150, KVH, D, generator=g) for _ in range(2))
    v[::7] *= 1e6
    v[::5] = 0
    v[1::11] *= 1e-12
    k[3::13] *= 1e-6
    cos, sin = O.tables(160, D, device=DEV)
    seq, pos = torch.zeros(150, dtype=torch.int32, device=DEV), torch.arange(150, dtype=torch.int32, device=DEV)
    P.paged_append(k.to(DEV, torch.bfloat16), v.to(DEV, torch.bfloat16), cache, table.to(DEV), seq, pos, cos, sin)
    kqv = torch.randn(1, (2 * KVH + QH) * D, generator=g)
    kqv[0, KVH * D:(KVH + 4) * D] *= 30
    kqv[0, (KVH + 4) * D:(KVH + 5) * D] = 0
    kqv = kqv.to(DEV, torch.bfloat16)
    o = P.paged_attn_append(kqv, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), QH, KVH, cos, sin)
    check_token(cache, table, kqv, o, lens, QH, KVH, D)


def test_strides_streams_graphs_and_the_general_path(monkeypatch):
    QH, KVH, D, lens = 12, 4, 128, [100, 37]
    cache, table, *_, cos, sin = filled("int8", lens, KVH, D, 32)
    table, n = table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    kqv = torch.randn(2, (2 * KVH + QH) * D, device=DEV).to(torch.bfloat16)
    want = P.paged_attn_append(kqv, cache, table, n, QH, KVH, cos, sin)
    after = [x.clone() for x in cache]
    wide = torch.stack([table, table], 2)[:, :, 0]
    for x in (torch.cat([kqv, kqv], 1)[:, :kqv.shape[1]], torch.cat([kqv[:, :1], kqv], 1)[:, 1:], kqv.t().contiguous().t()):
        assert torch.equal(P.paged_attn_append(x, cache, wide, n, QH, KVH, cos, sin), want)
    with monkeypatch.context() as m:
        m.setattr(native, "host", None)
        assert torch.equal(P.paged_attn_append(kqv, cache, table, n, QH, KVH, cos, sin), want)
        rows = kqv[:, :KVH * D].unflatten(1, (KVH, D))
        seq = torch.arange(2, dtype=torch.int32, device=DEV)
        P.paged_append(rows, kqv[:, (KVH + QH) * D:].unflatten(1, (KVH, D)), cache, table, seq, n, cos, sin)
        assert same(cache, after)                            # the same row from either kernel
        kc, vc = (torch.zeros(2, KVH, 101, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        P.paged_read(cache, table, n + 1, kc, vc)
    k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
    P.paged_read(cache, table, n + 1, k2, v2)
    assert torch.equal(kc, k2) and torch.equal(vc, v2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = P.paged_attn_append(kqv, cache, table, n, QH, KVH, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two captured tokens in a row, replayed with other inputs
    static, length = kqv.clone(), n.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = P.paged_attn_append(static, cache, table, length, QH, KVH, cos, sin)
        length.add_(1)
        b = P.paged_attn_append(static, cache, table, length, QH, KVH, cos, sin)
        P.paged_read(cache, table, length + 1, k2, v2)
    length.copy_(n)
    static.copy_(kqv.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    got_a, got_b = a.clone(), b.clone()
    one = P.paged_attn_append(kqv.flip(0).contiguous(), cache, table, n, QH, KVH, cos, sin)
    two = P.paged_attn_append(kqv.flip(0).contiguous(), cache, table, n + 1, QH, KVH, cos, sin)
    assert torch.equal(got_a, one) and torch.equal(got_b, two)


def test_cuda_refusals():
    cache = P.paged_cache(2, 2, 32, 32, DEV, "int8")
    table, n = torch.zeros((1, 1), dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    cos, sin = O.tables(32, 32, device=DEV)
    x = torch.zeros(1, 2, 32, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        P.paged_append(x, x, cache, table, n, n, cos, sin)   # head dimension 32
    cache = P.paged_cache(2, 2, 32, 64, DEV, "int8")
    x, (cos, sin) = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV), O.tables(32, 64, device=DEV)
    kqv = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(TypeError):
        P.paged_append(x.float(), x.float(), cache, table, n, n, cos, sin)
    with pytest.raises(TypeError):
        P.paged_attn_append(kqv.float(), cache, table, n, 4, 2, cos, sin)
    with pytest.raises(TypeError):
        P.paged_attn_append(kqv, cache, table, n, 4, 2, cos.double(), sin.double())
    with pytest.raises(ValueError):
        P.paged_attn_append(kqv, cache, table.cpu(), n, 4, 2, cos, sin)
    with pytest.raises(ValueError):
        P.paged_attn_append(kqv.cpu(), cache, table, n, 4, 2, cos, sin)
    with pytest.raises(ValueError):
        P.paged_attn_append(kqv, cache, table, n.cpu(), 4, 2, cos, sin)
    with pytest.raises(TypeError):
        P.paged_read(cache, table, n, *(torch.zeros(1, 2, 4, 64, device=DEV) for _ in range(2)))
    off = torch.zeros(1 * 2 * 4 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(1, 2, 4, 64)
    with pytest.raises(ValueError):
        P.paged_read(cache, table, n, off, off)
    with pytest.raises(TypeError):
        P.paged_attn_append(kqv, P.PagedCache(cache.k.float(), cache.v.float()), table, n, 4, 2, cos, sin)


def test_calls_without_rows():
    cache = P.paged_cache(2, 2, 32, 64, DEV, "e4m3")
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    table = torch.zeros((0, 1), dtype=torch.int32, device=DEV)
    cos, sin = O.tables(32, 64, device=DEV)
    kqv = torch.zeros(0, 8 * 64, dtype=torch.bfloat16, device=DEV)
    assert P.paged_attn_append(kqv, cache, table, none, 4, 2, cos, sin).shape == (0, 4, 64)
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    P.paged_append(x, x, cache, table, none, none, cos, sin)
    kc = torch.zeros(0, 2, 5, 64, dtype=torch.bfloat16, device=DEV)
    P.paged_read(cache, table, none, kc, kc.clone())
