"""The paged cache's plain forms on the CPU against the definitions in fp64, and what its functions refuse."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import paged as P

from . import paged_oracle as O

KINDS = ["bf16", "int8", "e4m3"]


def filled(kind, B, lens, KVH, D, page, seed=0, extra=1, device="cpu"):
    """A pool whose pages stand in random order, the table of ``B`` sequences, and the fp32 K and V that went in un-rotated."""
    g = torch.Generator().manual_seed(seed)
    width = max(lens) // page + extra
    pages = B * width + 2
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32)
    cache = P.paged_cache(pages, KVH, page, D, device, kind)
    M = sum(lens)
    k, v = (torch.randn(M, KVH, D, generator=g).to(torch.bfloat16) for _ in range(2))
    seq = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(lens)]) if M else torch.zeros(0, dtype=torch.int32)
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]) if M else torch.zeros(0, dtype=torch.int32)
    cos, sin = O.tables(width * page, D, device=device)
    P.paged_append(k.to(device), v.to(device), cache, table.to(device), seq.to(device), pos.to(device), cos, sin)
    return cache, table, k, v, seq, pos, cos, sin


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens", [[1], [32, 31, 33], [70, 0, 5]])
def test_rows_are_held_as_defined(kind, lens):
    cache, table, k, v, seq, pos, _, _ = filled(kind, len(lens), lens, 2, 16, 32)
    for m in range(len(seq)):
        b, t = int(seq[m]), int(pos[m])
        kk, vv, there = O.cached(cache, table, b, t + 1)
        want = O.rotated(k[m], t)
        assert there[t]
        assert bool(((kk[t] - want).abs() <= O.step(kind)(want)).all())
        assert bool(((vv[t] - v[m].double()).abs() <= O.step(kind)(v[m].double())).all())


@pytest.mark.parametrize("kind", KINDS)
def test_read_gives_back_what_is_held(kind):
    lens = [40, 0, 33]
    cache, table, *_ = filled(kind, 3, lens, 2, 16, 32)
    start = torch.tensor([3, 0, 32], dtype=torch.int32)
    kc, vc = (torch.full((3, 2, 20, 16), 7.0) for _ in range(2))
    assert P.paged_read(cache, table, torch.tensor(lens, dtype=torch.int32), kc, vc, start=start) == (kc, vc)
    for b, n in enumerate(lens):
        k, v, _ = O.cached(cache, table, b, n)
        rows = min(20, max(0, n - int(start[b])))
        for got, x in ((kc, k), (vc, v)):
            assert torch.equal(got[b, :, :rows].double(), x[int(start[b]):int(start[b]) + rows].transpose(0, 1).float().double())
            assert bool((got[b, :, rows:] == 7.0).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
def test_attention_of_a_token(kind, mod):
    lens = [40, 0, 63, -1]
    cache, table, _, _, _, _, cos, sin = filled(kind, 4, [max(n, 0) for n in lens], 2, 16, 32)
    kqv = torch.randn(4, (2 * 2 + 6) * 16, dtype=torch.float32)
    slopes = torch.rand(6) if mod == "bias" else None
    cap = 2.0 if mod == "cap" else 0.0
    before = [None if x is None else x.clone() for x in cache]
    o = P.paged_attn_append(kqv, cache, table, torch.tensor(lens, dtype=torch.int32), 6, 2, cos, sin, softcap=cap, slopes=slopes)
    for b, n in enumerate(lens):
        if n < 0:
            assert bool((o[b] == 0).all())
            continue
        rows = kqv[b].view(10, 16)
        k, v, there = O.cached(cache, table, b, n + 1)
        assert there.all()
        want = O.rotated(rows[:2], n)
        assert bool(((k[n] - want).abs() <= O.step(kind)(want)).all())
        x = O.attend(O.rotated(rows[2:8], n), k, v, n, torch.arange(n + 1), 0.25, cap, slopes)
        assert torch.allclose(o[b].double(), x, atol=2e-5, rtol=2e-5)
    changed = [int((x.float() != y.float()).flatten(3).any(-1).any(1).sum()) for x, y in zip(cache[:2], before[:2])]
    assert changed == [3, 3]                                # the new tokens' rows and no others


@pytest.mark.parametrize("kind", KINDS)
def test_what_is_not_there_is_not_seen_and_not_written(kind):
    cache, table, _, _, _, _, cos, sin = filled(kind, 2, [40, 64], 2, 16, 32, extra=0)
    table[0, 0] = -1                                         # 32 of 40 tokens gone; sequence 1: no room for a token at 64
    kqv = torch.randn(2, 10 * 16)
    before = cache.k.clone()
    o = P.paged_attn_append(kqv, cache, table, torch.tensor([40, 64], dtype=torch.int32), 6, 2, cos, sin)
    k, v, there = O.cached(cache, table, 0, 41)
    want = O.attend(O.rotated(kqv[0].view(10, 16)[2:8], 40), k[32:], v[32:], 40, torch.arange(32, 41), 0.25)
    assert torch.allclose(o[0].double(), want, atol=2e-5)
    k, v, _ = O.cached(cache, table, 1, 64)
    want = O.attend(O.rotated(kqv[1].view(10, 16)[2:8], 63), k, v, 63, torch.arange(64), 0.25)      # the table's last angle
    assert torch.allclose(o[1].double(), want, atol=2e-5)
    assert int((before.float() != cache.k.float()).flatten(3).any(-1).any(1).sum()) == 1
    # rows of other sequences, positions and pages, and behind the rotary tables
    before = cache.k.clone()
    rows = torch.randn(6, 2, 16)
    seq, pos = torch.tensor([-1, 2, 0, 1, 1, 0], dtype=torch.int32), torch.tensor([0, 0, 5, 64, -1, 63], dtype=torch.int32)
    P.paged_append(rows, rows, cache, table, seq, pos, cos[:60], sin[:60])
    assert torch.equal(before.float(), cache.k.float())
    kc, vc = (torch.full((2, 2, 64, 16), 7.0) for _ in range(2))
    P.paged_read(cache, table, torch.tensor([40, 99], dtype=torch.int32), kc, vc)
    assert bool((kc[0, :, :32] == 7).all()) and not bool((kc[0, :, 32:40] == 7).any()) and not bool((kc[1] == 7).any())


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_zeros_and_of_extreme_magnitudes(kind):
    cache = P.paged_cache(1, 1, 32, 16, "cpu", kind)
    rows = torch.zeros(4, 1, 16)
    rows[1], rows[2], rows[3, 0, 0] = 1e-30, 3e38, 1e4
    rows[3, 0, 1:] = 1e-3
    table = torch.zeros((1, 1), dtype=torch.int32)
    P.paged_append(rows, rows, cache, table, torch.zeros(4, dtype=torch.int32), torch.arange(4, dtype=torch.int32))
    k, _, _ = O.cached(cache, table, 0, 4)
    assert bool(torch.isfinite(k).all())
    assert bool(((k - rows.double()).abs() <= O.step(kind)(rows.double())).all())


def test_refusals():
    cache, table, k, v, seq, pos, cos, sin = filled("int8", 2, [3, 4], 2, 16, 32)
    kqv, lens = torch.randn(2, 10 * 16), torch.tensor([3, 4], dtype=torch.int32)
    kc = torch.zeros(2, 2, 8, 16)
    kv = torch.zeros(7, 2, 16)
    for bad in (dict(kind="int4"), dict(page=48), dict(page=16), dict(pages=0), dict(KVH=0)):
        with pytest.raises(ValueError):
            P.paged_cache(**{**dict(pages=2, KVH=2, page=32, D=16, device="cpu", kind="bf16"), **bad})
    bad_caches = [cache._replace(k_scale=None), cache._replace(k_scale=None, v_scale=None), cache._replace(v=cache.v[1:]),
                  cache._replace(k=cache.k.float(), v=cache.v.float()), cache._replace(k_scale=cache.k_scale.double()),
                  cache._replace(k=cache.k.transpose(0, 1), v=cache.v.transpose(0, 1))]
    calls = [lambda c, t: P.paged_append(kv, kv, c, t, seq, pos, cos, sin), lambda c, t: P.paged_read(c, t, lens, kc, kc.clone()),
             lambda c, t: P.paged_attn_append(kqv, c, t, lens, 6, 2, cos, sin)]
    for call in calls:
        call(cache, table)
        for c in bad_caches:
            with pytest.raises((ValueError, TypeError)):
                call(c, table)
        for t in (table.long(), table[0], table[:, :0]):
            with pytest.raises(ValueError):
                call(cache, t)
    with pytest.raises(ValueError):
        P.paged_append(kv, kv, cache, table, seq, pos, cos)
    for args in ((kv[:, :1], kv, seq, pos), (kv, kv, seq[1:], pos), (kv, kv, seq.long(), pos), (kv, kv[:3], seq, pos)):
        with pytest.raises(ValueError):
            P.paged_append(args[0], args[1], cache, table, args[2], args[3], cos, sin)
    with pytest.raises(ValueError):
        P.paged_append(kv, kv, cache, table, seq, pos, cos[:, :4], sin[:, :4])
    for kw in (dict(lens=lens.long()), dict(lens=lens[:1]), dict(kcache=kc[:1], vcache=kc[:1]), dict(start=lens.long()),
               dict(vcache=kc[:, :, :4])):
        with pytest.raises(ValueError):
            P.paged_read(**{**dict(cache=cache, table=table, lens=lens, kcache=kc, vcache=kc.clone()), **kw})
    for kw in (dict(QH=5), dict(KVH=1), dict(lens=lens.long()), dict(cos=cos[:0], sin=sin[:0]), dict(softcap=-1.0),
               dict(softcap=1.0, slopes=torch.ones(6)), dict(slopes=torch.ones(2)), dict(scale=0.0), dict(kqv=kqv[:1])):
        with pytest.raises(ValueError):
            P.paged_attn_append(**{**dict(kqv=kqv, cache=cache, table=table, lens=lens, QH=6, KVH=2, cos=cos, sin=sin), **kw})
