"""Span and tree attention kernels against their definitions in fp64, inside the bounds of their roundings (tests/masked_oracle.py)."""
import math
import random

import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A
from create_llm_by_cupy_b200.ops import native
from tests.masked_oracle import span_oracle, tree_oracle, within

pytestmark = pytest.mark.gpu
DEV = "cuda"


def packed(B, T, QH, KVH, D, seed, std=1.5):
    """q, k, v as views of one packed projection [K | Q | V], and an output gradient."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    kqv = (torch.randn(B, T, (2 * KVH + QH) * D, device=DEV, generator=g) * std).to(torch.bfloat16)
    k, q, v = kqv.split([KVH * D, QH * D, KVH * D], 2)
    dout = torch.randn(B, T, QH, D, device=DEV, generator=g).to(torch.bfloat16)
    return q.unflatten(2, (QH, D)), k.unflatten(2, (KVH, D)), v.unflatten(2, (KVH, D)), dout


def documents(B, T, mean, pad, seed):
    rng = random.Random(seed)
    docs, prefix = torch.full((B, T), -1, dtype=torch.int32), torch.zeros(B, T, dtype=torch.bool)
    for b in range(B):
        at, i = 0, 0
        while at < T - pad:
            n = min(T - pad - at, rng.randrange(1, 2 * mean))
            docs[b, at:at + n] = i
            prefix[b, at:at + n // 3] = True
            at, i = at + n, i + 1
    return docs.to(DEV), prefix.to(DEV)


def some_slopes(QH):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / QH) for h in range(QH)], device=DEV)


def check(q, k, v, dout, mask, softcap=0.0, slopes=None, scale=None, train=True):
    sc = 1 / math.sqrt(q.shape[3]) if scale is None else scale
    want = span_oracle(q, k, v, mask.dense(), sc, softcap, slopes, dout if train else None)
    o, lse = A.span_attn_fwd(q, k, v, mask, scale=scale, softcap=softcap, slopes=slopes)
    within(o, want["o"], want["o_b"], "o")
    none = want["lse"].isinf()
    assert torch.equal(lse.isinf(), none) and bool((lse[none] < 0).all())
    # sums of products of bf16 in fp32, and statistics in fp32: 2^-18 of the largest score is 30 times their rounding
    assert bool(((lse.double() - want["lse"])[~none].abs() <= 2 ** -18 * (1 + want["lse"][~none].abs())).all())
    if train:
        grads = A.span_attn_bwd(dout, q, k, v, o, lse, mask, scale=scale, softcap=softcap, slopes=slopes)
        for got, n in zip(grads, ("dq", "dk", "dv")):
            within(got, want[n], want[n + "_b"], n)
    assert native.read_status() == (0, 0)


# --------------------------------------------------------------------------- masks
@pytest.mark.parametrize("T", [1, 127, 128, 129, 1000, 4096, 4099, 9001])
@pytest.mark.parametrize("prefix", [False, True])
def test_span_mask(T, prefix):
    B = 3
    docs, pre = documents(B, T, max(2, T // 5), T // 7, T)
    valid = torch.tensor([T, T // 2, 0], dtype=torch.int32, device=DEV)
    kw = [dict(docs=docs), dict(docs=docs, valid_len=valid), dict(valid_len=valid), {}]
    for k in kw:
        if prefix:
            k = dict(k, prefix=pre)
        got = A.span_mask(B, T, DEV, **k)
        want = A.span_mask(B, T, "cpu", **{n: x.cpu() for n, x in k.items()})
        assert torch.equal(got.spans.cpu(), want.spans)
        again = A.SpanMask.from_spans(want.spans[..., 0].to(DEV).contiguous(), want.spans[..., 1].to(DEV).contiguous())
        assert torch.equal(again.buf, got.buf)
        lo, hi = want.spans.long().unbind(-1)
        nt = (T + 127) // 128
        qtab = got.buf[:4 * B * nt].view(B, nt, 4).cpu()
        ktab = got.buf[4 * B * nt:6 * B * nt].view(B, nt, 2).cpu()
        for b in range(B):
            meets = torch.zeros(nt, nt, dtype=torch.bool)
            for m in range(nt):
                rows = slice(m * 128, min(T, m * 128 + 128))
                some = hi[b, rows] > lo[b, rows]
                if some.any():
                    first, end = int(lo[b, rows][some].min()) // 128, -(-int(hi[b, rows][some].max()) // 128)
                    assert qtab[b, m, :2].tolist() == [first, end]
                    if some.all():
                        assert qtab[b, m, 2:].tolist() == [int(lo[b, rows].max()), int(hi[b, rows].min())]
                    else:
                        assert qtab[b, m, 2] >= T
                    meets[m, first:end] = True
                else:
                    assert qtab[b, m, :2].tolist() == [0, 0]
            for n in range(nt):
                ms = torch.nonzero(meets[:, n]).flatten().tolist()
                assert ktab[b, n].tolist() == ([ms[0], ms[-1] + 1] if ms else [0, 0])


# --------------------------------------------------------------------------- span attention
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
@pytest.mark.parametrize("B,T,QH,KVH,mean,pad", [
    (1, 1, 2, 1, 2, 0), (2, 2, 2, 2, 2, 1), (1, 65, 3, 1, 20, 0), (2, 128, 4, 1, 300, 0), (2, 300, 8, 1, 60, 20), (3, 500, 6, 2, 130, 260),
    (1, 1030, 4, 4, 400, 3)])
@pytest.mark.parametrize("prefix", [False, True])
def test_span_attention(D, mod, B, T, QH, KVH, mean, pad, prefix):
    docs, pre = documents(B, T, mean, pad, T + D)
    mask = A.span_mask(B, T, DEV, docs=docs, prefix=pre if prefix else None)
    check(*packed(B, T, QH, KVH, D, T), mask, 30.0 if mod == "cap" else 0.0, some_slopes(QH) if mod == "bias" else None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("std,cap", [(1.0, 30.0), (2.5, 20.0), (6.0, 20.0), (3.0, 2.0)])
def test_caps_of_every_size(D, std, cap):
    """Scores well inside the cap, up to it and far beyond it, in one row's tiles and over its masked edges."""
    B, T, QH, KVH = 1, 400, 4, 2
    docs, _ = documents(B, T, 150, 10, 4)
    q, k, v, dout = packed(B, T, QH, KVH, D, 9, std)
    q = q * torch.linspace(0.05, 1.0, T, device=DEV, dtype=torch.bfloat16)[None, :, None, None]
    check(q, k, v, dout, A.span_mask(B, T, DEV, docs=docs), cap)


@pytest.mark.parametrize("D", [64, 128])
def test_any_spans(D):
    """Windows, spans with nothing in between, rows that see only later keys, rows that see nothing, spans past the row."""
    B, T = 3, 700
    t = torch.arange(T)
    lo, hi = torch.zeros(B, T, dtype=torch.int32), torch.zeros(B, T, dtype=torch.int32)
    lo[0], hi[0] = (t - 99).clamp_min(-3), t + 1                                   # a window
    far = (t // 128) % 2 == 0                                                      # neighbouring tiles at the two ends
    lo[1], hi[1] = torch.where(far, t * 0 + 640, t * 0 + 3), torch.where(far, t * 0 + 900, t * 0 + 77)
    lo[2], hi[2] = torch.where(t % 3 == 0, t, T - 1 - t), torch.where(t % 5 == 0, t * 0, T - t // 2)
    mask = A.SpanMask.from_spans(lo.to(DEV), hi.to(DEV))
    check(*packed(B, T, 4, 2, D, 3), mask)
    check(*packed(B, T, 4, 2, D, 4), mask, 15.0)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_see_little_after_much_larger_scores(D):
    """A row whose first seen key stands behind tiles of masked, far larger scores; scores of the type's largest magnitudes."""
    B, T, QH, KVH = 1, 384, 2, 1
    q, k, v, dout = packed(B, T, QH, KVH, D, 6)
    k = k.clone()
    k[:, :200] *= 300
    docs = torch.tensor([[0] * 200 + [1] * 184], dtype=torch.int32, device=DEV)
    check(q, k, v, dout, A.span_mask(B, T, DEV, docs=docs))


def test_nothing_to_see():
    q, k, v, dout = packed(2, 200, 4, 2, 64, 1)
    mask = A.span_mask(2, 200, DEV, valid_len=torch.zeros(2, dtype=torch.int32, device=DEV))
    o, lse = A.span_attn_fwd(q, k, v, mask)
    assert not o.any() and bool((lse == -math.inf).all())
    assert not any(g.any() for g in A.span_attn_bwd(dout, q, k, v, o, lse, mask))
    assert native.read_status() == (0, 0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("QH,KVH", [(3, 1), (8, 2), (10, 2), (2, 2)])
def test_heads_shared_by_a_cluster(D, QH, KVH):
    docs, _ = documents(2, 400, 150, 130, 7)
    mask = A.span_mask(2, 400, DEV, docs=docs)
    lib = F._lib()
    q, k, v, dout = packed(2, 400, QH, KVH, D, 2)
    cos, sin = F.rope_table(400, D, 10000.0, DEV)
    o, lse = A.span_attn_fwd(q, k, v, mask)
    rotated = []
    try:
        for n in (1, 2, 3, 4):
            lib.b200_flash_span_split(n)
            check(q, k, v, dout, mask)
            rotated.append(A.span_attn_bwd(dout, q, k, v, o, lse, mask, unrotate=(cos, sin)))
            again = A.span_attn_bwd(dout, q, k, v, o, lse, mask, unrotate=(cos, sin))
            assert all(torch.equal(x, y) for x, y in zip(rotated[-1], again))
    finally:
        lib.b200_flash_span_split(0)
    for r in rotated[1:]:                                  # the order of fp32 sums, then one rounding
        for x, y in zip(r, rotated[0]):
            assert float((x.float() - y.float()).abs().max()) <= 2 ** -7 * float(y.float().abs().max())


def test_unrotated_gradients_in_place():
    B, T, QH, KVH, D = 2, 300, 6, 2, 128
    cos, sin = F.rope_table(T, D, 10000.0, DEV)
    q, k, v, dout = packed(B, T, QH, KVH, D, 5)
    docs, _ = documents(B, T, 100, 0, 1)
    mask = A.span_mask(B, T, DEV, docs=docs)
    o, lse = A.span_attn_fwd(q, k, v, mask)
    want = A.span_attn_bwd(dout.cpu().float(), q.cpu().float(), k.cpu().float(), v.cpu().float(), o.cpu().float(), lse.cpu(),
                           A.span_mask(B, T, "cpu", docs=docs.cpu()), unrotate=(cos.cpu(), sin.cpu()))
    buf = torch.full((B, T, (2 * KVH + QH) * D), math.nan, dtype=torch.bfloat16, device=DEV)
    out = tuple(x.unflatten(2, (-1, D)) for x in buf.split([QH * D, KVH * D, KVH * D], 2))
    A.span_attn_bwd(dout, q, k, v, o, lse, mask, out=out, unrotate=(cos, sin))
    for got, ref in zip(out, want):
        assert float((got.cpu().float() - ref).norm() / ref.norm()) < 1e-2
    with pytest.raises(ValueError):
        A.span_attn_bwd(dout, q, k, v, o, lse, mask, out=(out[0][..., 4:].contiguous(), out[1], out[2]))


@pytest.mark.parametrize("limit", [3 * 4 * 384 * 384 * 2, 2 * 384 * 384 * 2, 1])
def test_backward_in_parts(limit, monkeypatch):
    """Some batch elements, some KV heads, or one KV head at a time."""
    monkeypatch.setattr(F, "FLASH_DQ_GEMM_MAX_BYTES", limit)
    docs, _ = documents(5, 300, 80, 11, 3)
    check(*packed(5, 300, 4, 2, 64, 8), A.span_mask(5, 300, DEV, docs=docs), slopes=some_slopes(4))


def test_layouts():
    """Rows that tiles cannot be copied from are copied first: other orders, odd pitches, odd starts, one head for all (stride 0)."""
    B, T, QH, KVH, D = 2, 150, 4, 2, 64
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(B, QH, T, D, device=DEV, generator=g).to(torch.bfloat16).transpose(1, 2)
    k = torch.randn(B, T, KVH, D + 3, device=DEV, generator=g).to(torch.bfloat16)[..., :D]
    v = torch.randn(B * T * D + 1, device=DEV, generator=g).to(torch.bfloat16)[1:].view(B, T, 1, D).expand(B, T, KVH, D)
    dout = torch.randn(B, T, D, QH, device=DEV, generator=g).to(torch.bfloat16).transpose(2, 3)
    docs, _ = documents(B, T, 40, 5, 2)
    check(q, k, v, dout, A.span_mask(B, T, DEV, docs=docs))


def test_the_two_host_paths_and_streams_agree(monkeypatch):
    q, k, v, dout = packed(2, 260, 6, 2, 64, 3)
    docs, pre = documents(2, 260, 90, 9, 5)
    slopes = some_slopes(6)

    def run():
        m = A.span_mask(2, 260, DEV, docs=docs, prefix=pre)
        o, lse = A.span_attn_fwd(q, k, v, m, slopes=slopes)
        return (m.buf, o, lse, *A.span_attn_bwd(dout, q, k, v, o, lse, m, slopes=slopes))
    first = run()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(run(), first))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(other, first))
    monkeypatch.setattr(native, "host", None)
    assert all(torch.equal(x, y) for x, y in zip(run(), first))


def test_span_refusals_on_the_device():
    q, k, v, dout = packed(1, 64, 2, 1, 32, 1)
    m = A.span_mask(1, 64, DEV)
    with pytest.raises(ValueError):
        A.span_attn_fwd(q, k, v, m)
    with pytest.raises(ValueError):
        A.span_attn_bwd(dout, q, k, v, dout, torch.zeros(1, 2, 64, device=DEV), m)
    q, k, v, _ = packed(1, 64, 2, 1, 64, 1)
    with pytest.raises(TypeError):
        A.span_attn_fwd(q.float(), k.float(), v.float(), m)
    with pytest.raises(ValueError):
        A.span_attn_fwd(q, k, v, A.span_mask(1, 64, "cpu"))
    with pytest.raises(ValueError):
        A.span_mask(1, 64, DEV, docs=torch.zeros(1, 64, dtype=torch.int32))
    for kw in (dict(scale=0.0), dict(softcap=-1.0), dict(slopes=torch.zeros(2)), dict(slopes=torch.zeros(2, device=DEV), softcap=2.0)):
        with pytest.raises(ValueError):
            A.span_attn_fwd(q, k, v, m, **kw)


# --------------------------------------------------------------------------- tree attention
def tree_case(lens, n, QH, KVH, D, Tmax, seed=0, cached_only=False):
    rng, g = random.Random(seed), torch.Generator(device=DEV).manual_seed(seed)
    B = len(lens)
    parents = [[rng.randrange(-1, i) for i in range(n)] for _ in range(B)]
    kqv = (torch.randn(B * n, (2 * KVH + QH) * D, device=DEV, generator=g) * 1.5).to(torch.bfloat16)
    kc, vc = ((torch.randn(B, KVH, Tmax, D, device=DEV, generator=g) * s).to(torch.bfloat16) for s in (1.5, 1.0))
    for b, L in enumerate(lens):                           # what is not cached may hold anything
        kc[b, :, L:], vc[b, :, L:] = math.nan, math.inf
    tree = A.tree_mask(parents, DEV)
    if cached_only:
        for b in range(B):
            parents[b][n - 1] = None
        tree[:, n - 1] = 0
    return kqv, kc, vc, torch.tensor(lens, dtype=torch.int32, device=DEV), tree, parents


def check_tree(lens, n, QH, KVH, D, Tmax, softcap=0.0, bias=False, **kw):
    kqv, kc, vc, lt, tree, parents = tree_case(lens, n, QH, KVH, D, Tmax, **kw)
    slopes = some_slopes(QH) if bias else None
    cos, sin = F.rope_table(Tmax, D, 10000.0, DEV)
    want, bound, kw_, vw = tree_oracle(kqv, kc, vc, lens, parents, QH, KVH, cos, sin, 1 / math.sqrt(D), softcap, slopes)
    got = A.tree_attn_append(kqv, kc, vc, lt, tree, QH, KVH, cos, sin, softcap=softcap, slopes=slopes)
    assert native.read_status() == (0, 0)
    within(got, want, bound, "o")
    for b, L in enumerate(lens):
        assert torch.allclose(kc[b, :, :L + n].double(), kw_[b, :, :L + n], rtol=2 ** -8, atol=1e-5)
        assert torch.equal(vc[b, :, :L + n].double(), vw[b, :, :L + n])
        assert kc[b, :, L + n:].isnan().all() and vc[b, :, L + n:].isinf().all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
@pytest.mark.parametrize("lens,n,QH,KVH", [
    ([0], 1, 2, 1), ([1], 1, 4, 4), ([127, 128, 129], 1, 4, 1), ([5, 0, 300], 7, 6, 2), ([256, 3], 33, 4, 1), ([200, 0, 90], 64, 4, 2),
    ([130], 64, 16, 1), ([70], 43, 3, 1), ([40] * 40, 2, 2, 1), ([1500], 3, 2, 2)])
def test_tree_attention(D, mod, lens, n, QH, KVH):
    check_tree(lens, n, QH, KVH, D, max(lens) + n + 5, 25.0 if mod == "cap" else 0.0, mod == "bias", seed=n)


@pytest.mark.parametrize("D", [64, 128])
def test_full_cache_and_drafts_that_see_the_cache_alone(D):
    check_tree([95, 0], 5, 4, 2, D, 100, cached_only=True)
    kqv, kc, vc, lt, tree, _ = tree_case([98], 5, 4, 2, D, 100)
    cos, sin = F.rope_table(100, D, 10000.0, DEV)
    A.tree_attn_append(kqv, kc, vc, lt, tree, 4, 2, cos, sin)
    rows = kqv.view(5, 8, D)[:2, 6:].transpose(0, 1)
    assert torch.equal(vc[0, :, 98:], rows) and native.read_status() == (0, 0)
    # a tree of nothing over an empty cache: zeros
    kqv, kc, vc, lt, tree, _ = tree_case([0], 3, 4, 2, D, 8)
    assert not A.tree_attn_append(kqv, kc, vc, lt, torch.zeros_like(tree), 4, 2, cos, sin).any()


def test_row_groups_of_every_kind():
    """Rows in a part of one tile, in two, in two groups, in three tiles; sequences cut into pieces and whole ones."""
    for n, QH, KVH in ((64, 2, 2), (64, 6, 2), (50, 12, 2), (64, 128, 1), (5, 100, 1)):
        check_tree([260, 31], n, QH, KVH, 64, 400, seed=n + QH)


def test_pieces_of_long_and_short_sequences():
    """More sequences than pieces, and sequences that many CTAs share; twice the same bits."""
    lens = [3000, 0, 17, 129, 1, 900, 2048]
    check_tree(lens, 4, 4, 2, 128, 3100, seed=2)
    check_tree([9000], 2, 2, 1, 64, 9100, 10.0, seed=3)
    kqv, kc, vc, lt, tree, _ = tree_case(lens, 16, 8, 2, 128, 3100)
    cos, sin = F.rope_table(3100, 128, 10000.0, DEV)
    first = A.tree_attn_append(kqv, kc, vc, lt, tree, 8, 2, cos, sin)
    for _ in range(5):
        assert torch.equal(A.tree_attn_append(kqv, kc, vc, lt, tree, 8, 2, cos, sin), first)


def test_tree_host_paths_streams_and_graphs_agree(monkeypatch):
    kqv, kc, vc, lt, tree, _ = tree_case([500, 20], 9, 6, 2, 128, 600)
    cos, sin = F.rope_table(600, 128, 10000.0, DEV)
    slopes = some_slopes(6)

    def run(x=kqv):
        return A.tree_attn_append(x, kc, vc, lt, tree, 6, 2, cos, sin, slopes=slopes)
    first = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    captured.zero_()
    graph.replay()
    assert torch.equal(captured, first)
    wide = torch.zeros(18, kqv.shape[1] + 5, dtype=torch.bfloat16, device=DEV)     # rows that do not start on 16 bytes
    wide[:, 5:] = kqv
    assert torch.equal(run(wide[:, 5:]), first)
    monkeypatch.setattr(native, "host", None)
    assert torch.equal(run(), first)


def test_caches_beyond_32_bit_offsets():
    """The last KV head of the last sequence starts 2^31 elements behind the cache's start."""
    B, KVH, D, Tmax, n = 2, 3, 128, 3_000_000, 3
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 14 GB")
    kc = torch.zeros(B, KVH, Tmax, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    g = torch.Generator(device=DEV).manual_seed(1)
    kqv = torch.randn(B * n, (2 * KVH + KVH) * D, device=DEV, generator=g).to(torch.bfloat16)
    L = [40, Tmax - 200]
    at = torch.randint(0, Tmax - 200, (4000,), device=DEV, generator=g)
    kc[1, :, at] = (torch.randn(KVH, 4000, D, device=DEV, generator=g) * 3).to(torch.bfloat16)
    vc[1, :, at] = torch.randn(KVH, 4000, D, device=DEV, generator=g).to(torch.bfloat16)
    cos, sin = F.rope_table(Tmax, D, 10000.0, DEV)
    got = A.tree_attn_append(kqv, kc, vc, torch.tensor(L, dtype=torch.int32, device=DEV), A.tree_mask([[-1, 0, 1]] * B, DEV), KVH, KVH,
                             cos, sin)
    assert native.read_status() == (0, 0)
    rows = kqv.view(B, n, 3 * KVH, D)
    assert torch.equal(vc[1, :, L[1]:L[1] + n], rows[1, :, 2 * KVH:].transpose(0, 1))
    h = KVH - 1
    pos = torch.arange(L[1], L[1] + n, device=DEV)
    c, s = cos[pos].double(), sin[pos].double()
    q = rows[1, :, KVH + h].double()
    q = torch.cat([q[:, :64] * c - q[:, 64:] * s, q[:, 64:] * c + q[:, :64] * s], -1).to(torch.bfloat16).double()
    for i in range(n):
        end = L[1] + i + 1
        x = (kc[1, h, :end].float() @ q[i].float()).double() / math.sqrt(D)
        p = torch.softmax(x, 0)
        want = (p.float()[None] @ vc[1, h, :end].float())[0]
        assert float((got[1, i, h].float() - want).norm()) <= 1e-2 * float(want.norm()) + 1e-5


def test_tree_refusals_on_the_device():
    kqv, kc, vc, lt, tree, _ = tree_case([4], 2, 2, 1, 64, 16)
    cos, sin = F.rope_table(16, 64, 10000.0, DEV)
    good = dict(kqv=kqv, kcache=kc, vcache=vc, lens=lt, tree=tree, QH=2, KVH=1, cos=cos, sin=sin)
    for kw in (dict(lens=lt.cpu()), dict(kcache=kc.transpose(2, 3).contiguous().transpose(2, 3)), dict(scale=0.0), dict(softcap=-2.0),
               dict(slopes=torch.zeros(2)), dict(cos=cos[:8], sin=sin[:8]), dict(tree=tree.int())):
        with pytest.raises(ValueError):
            A.tree_attn_append(**{**good, **kw})
    with pytest.raises(TypeError):
        A.tree_attn_append(**{**good, "kqv": kqv.float()})
    with pytest.raises(TypeError):
        A.tree_attn_append(**{**good, "cos": cos.bfloat16(), "sin": sin.bfloat16()})
