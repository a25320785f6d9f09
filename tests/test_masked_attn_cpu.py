"""Span masks, span attention and tree attention on the CPU: definitions, gradients against differences, refusals."""
import math
import random

import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A
from tests.masked_oracle import span_oracle, tree_oracle


def seen_by_definition(B, T, docs, prefix, valid_len):
    """Token by token, with none of the module's scans."""
    out = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        n = T if valid_len is None else min(max(int(valid_len[b]), 0), T)
        starts, s = [], 0
        for t in range(T):
            if t > 0 and docs is not None and docs[b, t] != docs[b, t - 1]:
                s = t
            starts.append(s)
        for t in range(n):
            if docs is not None and docs[b, t] < 0:
                continue
            lead = starts[t]                               # end of the leading flagged run of t's document
            while prefix is not None and lead < T and prefix[b, lead] and starts[lead] == starts[t]:
                lead += 1
            end = max(t + 1, lead if t < lead else 0)
            out[b, t, starts[t]:min(end, n)] = True
    return out


@pytest.mark.parametrize("T", [1, 2, 7, 64, 130])
@pytest.mark.parametrize("use", ["none", "docs", "prefix", "docs+prefix", "valid", "all"])
def test_span_mask_is_the_definition(T, use):
    g = torch.Generator().manual_seed(T)
    B = 3
    docs = torch.randint(-1, 3, (B, T), generator=g).sort(1).values.to(torch.int32) if use in ("docs", "docs+prefix", "all") else None
    prefix = torch.rand(B, T, generator=g) < 0.7 if "prefix" in use or use == "all" else None
    valid = torch.tensor([0, T // 2, T], dtype=torch.int32) if use in ("valid", "all") else None
    got = A.span_mask(B, T, "cpu", docs=docs, prefix=prefix, valid_len=valid)
    assert torch.equal(got.dense(), seen_by_definition(B, T, docs, prefix, valid))


def test_spans_are_cut_to_the_row():
    lo = torch.tensor([[-5, 2, 3, 1]], dtype=torch.int32)
    hi = torch.tensor([[1, 2, 99, 0]], dtype=torch.int32)
    assert A.SpanMask.from_spans(lo, hi).spans.tolist() == [[[0, 1], [0, 0], [3, 4], [0, 0]]]


@pytest.mark.parametrize("softcap,bias", [(0.0, False), (3.0, False), (0.0, True)])
def test_span_attention_and_its_gradient(softcap, bias):
    """Against the definition, and every gradient against differences of the sum of o dout, in fp64."""
    g = torch.Generator().manual_seed(5)
    B, T, QH, KVH, D = 2, 7, 4, 2, 4
    q, k, v = (torch.randn(B, T, h, D, generator=g, dtype=torch.float64) * 1.5 for h in (QH, KVH, KVH))
    dout = torch.randn(B, T, QH, D, generator=g, dtype=torch.float64)
    docs = torch.tensor([[0, 0, 0, 1, 1, 1, -1], [0] * 7], dtype=torch.int32)
    prefix = torch.tensor([[1, 1, 0, 1, 0, 0, 0], [1, 1, 1, 0, 0, 0, 0]], dtype=torch.bool)
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625]) if bias else None
    mask = A.span_mask(B, T, "cpu", docs=docs, prefix=prefix)
    kw = dict(softcap=softcap, slopes=slopes)
    o, lse = A.span_attn_fwd(q, k, v, mask, **kw)
    want = span_oracle(q, k, v, mask.dense(), 1 / math.sqrt(D), softcap, slopes, dout)
    assert torch.allclose(o, want["o"], atol=1e-12)
    assert torch.equal(lse.isinf(), want["lse"].isinf()) and torch.allclose(lse[~lse.isinf()], want["lse"][~lse.isinf()], atol=1e-12)
    assert lse[0, :, 6].isinf().all() and not o[0, 6].any()
    grads = A.span_attn_bwd(dout, q, k, v, o, lse, mask, **kw)
    for got, n in zip(grads, ("dq", "dk", "dv")):
        assert torch.allclose(got, want[n], atol=1e-11), n
    rng, eps = random.Random(0), 1e-6
    for x, got in zip((q, k, v), grads):
        for _ in range(24):
            i = tuple(rng.randrange(n) for n in x.shape)
            keep = float(x[i])
            f = []
            for s in (eps, -eps):
                x[i] = keep + s
                f.append(float((A.span_attn_fwd(q, k, v, mask, **kw)[0] * dout).sum()))
            x[i] = keep
            assert abs((f[0] - f[1]) / (2 * eps) - float(got[i])) < 1e-6


def test_causal_rows_are_the_plain_attention():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(2, 9, h, 8, generator=g) for h in (4, 2, 2))
    n = torch.tensor([9, 5], dtype=torch.int32)
    o, lse = A.span_attn_fwd(q, k, v, A.span_mask(2, 9, "cpu", valid_len=n))
    ref, ref_lse = F.flash_attn_fwd(q, k, v, valid_len=n)
    for b in range(2):                                     # rows of padding differ: here they see nothing
        assert torch.allclose(o[b, :n[b]], ref[b, :n[b]], atol=1e-6) and torch.allclose(lse[b, :, :n[b]], ref_lse[b, :, :n[b]], atol=1e-5)
    assert not o[1, 5:].any()


def test_rotated_gradients():
    """``unrotate`` gives the gradients of the un-rotated tensors, ``out`` is written in place."""
    g = torch.Generator().manual_seed(2)
    B, T, QH, KVH, D = 1, 6, 2, 1, 8
    cos, sin = F.rope_table(T, D, 100.0, "cpu")
    q, k, v, do = (torch.randn(B, T, h, D, generator=g) for h in (QH, KVH, KVH, QH))
    mask = A.span_mask(B, T, "cpu")

    def rot(x, inverse=False):
        y = x.reshape(B * T, -1).clone()
        F.rope_inplace(y, cos, sin, T, x.shape[2], D, inverse=inverse)
        return y.view(x.shape)
    qr, kr = rot(q), rot(k)
    o, lse = A.span_attn_fwd(qr, kr, v, mask)
    plain = A.span_attn_bwd(do, qr, kr, v, o, lse, mask)
    out = tuple(torch.empty_like(x) for x in (q, k, v))
    got = A.span_attn_bwd(do, qr, kr, v, o, lse, mask, out=out, unrotate=(cos, sin))
    assert all(x is y for x, y in zip(got, out))
    for x, y in zip(got, (rot(plain[0], True), rot(plain[1], True), plain[2])):
        assert torch.allclose(x, y, atol=1e-5)


# --------------------------------------------------------------------------- trees
def some_parents(rng, n):
    return [rng.randrange(-1, i) for i in range(n)]


@pytest.mark.parametrize("lens,n,softcap,bias", [([5, 0], 1, 0.0, False), ([3, 11], 6, 4.0, False), ([0, 2], 9, 0.0, True)])
def test_tree_attention(lens, n, softcap, bias):
    rng, g = random.Random(n), torch.Generator().manual_seed(n)
    B, QH, KVH, D, Tmax = 2, 4, 2, 8, 24
    parents = [some_parents(rng, n) for _ in range(B)]
    kqv = torch.randn(B * n, (2 * KVH + QH) * D, generator=g).to(torch.bfloat16)
    kc, vc = (torch.randn(B, KVH, Tmax, D, generator=g).to(torch.bfloat16) for _ in range(2))
    for b, L in enumerate(lens):
        kc[b, :, L:], vc[b, :, L:] = math.nan, math.inf
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(QH)]) if bias else None
    cos, sin = F.rope_table(Tmax, D, 10000.0, "cpu")
    want, bound, kw, vw = tree_oracle(kqv, kc, vc, lens, parents, QH, KVH, cos, sin, 1 / math.sqrt(D), softcap, slopes)
    got = A.tree_attn_append(kqv, kc, vc, torch.tensor(lens, dtype=torch.int32), A.tree_mask(parents, "cpu"), QH, KVH, cos, sin,
                             softcap=softcap, slopes=slopes)
    assert ((got.double() - want).abs() <= bound + 1e-6).all()
    for b, L in enumerate(lens):
        assert torch.allclose(kc[b, :, :L + n].double(), kw[b, :, :L + n], rtol=2 ** -8, atol=1e-6)
        assert torch.equal(vc[b, :, :L + n].double(), vw[b, :, :L + n])
        assert kc[b, :, L + n:].isnan().all() and vc[b, :, L + n:].isinf().all()


def test_a_chain_is_token_by_token_decoding():
    """n drafts in a chain are n decoded tokens, one after the other."""
    g = torch.Generator().manual_seed(3)
    QH, KVH, D, Tmax, n = 4, 2, 8, 16, 5
    cos, sin = F.rope_table(Tmax, D, 10000.0, "cpu")
    kqv = torch.randn(n, (2 * KVH + QH) * D, generator=g)
    kc, vc = (torch.zeros(1, KVH, Tmax, D) for _ in range(2))
    kc1, vc1 = kc.clone(), vc.clone()
    chain = A.tree_attn_append(kqv, kc, vc, torch.zeros(1, dtype=torch.int32), A.tree_mask([range(-1, n - 1)], "cpu"), QH, KVH, cos, sin)
    for i in range(n):
        one = A.tree_attn_append(kqv[i:i + 1], kc1, vc1, torch.tensor([i], dtype=torch.int32), A.tree_mask([[-1]], "cpu"), QH, KVH, cos, sin)
        assert torch.allclose(one[0, 0], chain[0, i], atol=1e-6)
    assert torch.equal(kc, kc1) and torch.equal(vc, vc1)


def test_drafts_past_the_end_are_not_kept():
    QH, KVH, D, Tmax = 2, 1, 8, 4
    cos, sin = F.rope_table(Tmax, D, 10000.0, "cpu")
    kc, vc = (torch.zeros(1, KVH, Tmax, D) for _ in range(2))
    A.tree_attn_append(torch.ones(3, 4 * D), kc, vc, torch.tensor([3], dtype=torch.int32), A.tree_mask([[-1, 0, 1]], "cpu"), QH, KVH, cos, sin)
    assert vc[0, 0, 3].eq(1).all() and not vc[0, 0, :3].any()


def test_tree_mask():
    assert A.tree_mask([[-1, 0, 0, 2]], "cpu").tolist() == [[1, 3, 5, 13]]
    chain = A.tree_mask([list(range(-1, 63))], "cpu")
    assert chain[0, 63] == -1 and chain[0, 62] == (1 << 63) - 1
    for bad in ([[0]], [[-1, 1]], [[-2]], [list(range(-1, 64))]):
        with pytest.raises(ValueError):
            A.tree_mask(bad, "cpu")


# --------------------------------------------------------------------------- refusals
def test_span_refusals():
    q, k = torch.zeros(2, 4, 4, 8), torch.zeros(2, 4, 2, 8)
    m = A.span_mask(2, 4, "cpu")
    lse = torch.zeros(2, 4, 4)
    for bad in (dict(docs=torch.zeros(2, 4)), dict(docs=torch.zeros(2, 5, dtype=torch.int32)), dict(prefix=torch.zeros(2, 4)),
                dict(valid_len=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            A.span_mask(2, 4, "cpu", **bad)
    with pytest.raises(ValueError):
        A.span_mask(-1, 4, "cpu")
    with pytest.raises(ValueError):
        A.span_mask(1, 512001, "cpu")
    with pytest.raises(ValueError):
        A.SpanMask.from_spans(torch.zeros(2, 4), torch.zeros(2, 4))
    with pytest.raises(TypeError):
        A.span_attn_fwd(q, k, k, m.dense())
    for args, kw in (((q, k[:, :, :, :4], k), {}), ((q[:, :3], k, k), {}), ((q[:, :, :3], k, k), {}), ((q, k, k[:, :, :1]), {}),
                     ((q, k, k), dict(scale=0.0)), ((q, k, k), dict(scale=math.inf)), ((q, k, k), dict(softcap=-1.0)),
                     ((q, k, k), dict(softcap=math.nan)), ((q, k, k), dict(slopes=torch.zeros(3))),
                     ((q, k, k), dict(slopes=torch.zeros(4), softcap=1.0))):
        with pytest.raises(ValueError):
            A.span_attn_fwd(*args, m, **kw)
    with pytest.raises(ValueError):
        A.span_attn_fwd(q, k, k, A.span_mask(2, 5, "cpu"))
    for kw in (dict(dout=q[:, :3]), dict(o=q[:1]), dict(lse=lse[:1]), dict(unrotate=(torch.zeros(3, 4), torch.zeros(3, 4)))):
        a = dict(dout=q, q=q, k=k, v=k, o=q, lse=lse, mask=m)
        a.update(kw)
        with pytest.raises(ValueError):
            A.span_attn_bwd(**a)


def test_tree_refusals():
    QH, KVH, D, Tmax, B, n = 4, 2, 8, 16, 2, 3
    cos, sin = F.rope_table(Tmax, D, 10000.0, "cpu")
    good = dict(kqv=torch.zeros(B * n, 8 * D), kcache=torch.zeros(B, KVH, Tmax, D), vcache=torch.zeros(B, KVH, Tmax, D),
                lens=torch.zeros(B, dtype=torch.int32), tree=torch.ones(B, n, dtype=torch.int64), QH=QH, KVH=KVH, cos=cos, sin=sin)
    A.tree_attn_append(**good)
    for kw in (dict(kqv=torch.zeros(B * n, 7 * D)), dict(kqv=torch.zeros(B * n - 1, 8 * D)), dict(vcache=torch.zeros(B, KVH, Tmax + 1, D)),
               dict(lens=torch.zeros(B)), dict(lens=torch.zeros(B + 1, dtype=torch.int32)), dict(tree=torch.ones(B, n, dtype=torch.int32)),
               dict(QH=3), dict(cos=cos[:8], sin=sin[:8]), dict(sin=sin[:, :2]), dict(scale=-1.0), dict(softcap=math.inf),
               dict(slopes=torch.zeros(2)), dict(tree=torch.ones(B, 0, dtype=torch.int64), kqv=torch.zeros(0, 8 * D))):
        with pytest.raises(ValueError):
            A.tree_attn_append(**{**good, **kw})
