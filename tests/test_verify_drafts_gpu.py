"""Verification of drafted tokens on the GPU: whole numbers, equal to the definition's. (Both sides decide in 64 bits; a number falls
within their rounding, 10^-12, of a border between two tokens once in 10^7 draws at these sizes. The seeds are fixed.)"""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops import native
from create_llm_by_cupy_b200.ops.drafts import verify_drafts

from . import paged_oracle as O
from .test_verify_drafts_cpu import check, tree

pytestmark = pytest.mark.gpu


def run(logits, tokens, parents, u, q=None, accept=None, **kw):
    more = dict(draft_probs=q.cuda(), accept=accept.cuda()) if q is not None else {}
    return verify_drafts(logits.cuda(), tokens.cuda(), parents.cuda(), u.cuda(), **more, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temp", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("top", [1.0, 0.9, 0.3, 1e-9])
@pytest.mark.parametrize("drawn", [False, True])
def test_against_the_definition(dtype, temp, top, drawn):
    for seed, (B, n, V) in enumerate([(1, 1, 1), (3, 2, 127), (5, 9, 130), (2, 64, 1000), (3, 5, 4099)]):
        x, tokens, parents, u, q, accept = tree(B, n, V, seed, dtype=dtype)
        check(run(x, tokens, parents, u, q if drawn else None, accept, temp=temp, top=top),
              O.verify(x, tokens, parents, u, temp, top, q if drawn else None, accept))


@pytest.mark.parametrize("temp", [1e-6, 1e-3, 50.0, 1e6])
def test_extreme_temperatures(temp):
    """From the largest logit alone to all tokens alike, with logits that are far apart and large."""
    x, tokens, parents, u, q, accept = tree(3, 5, 900, 4, spread=30.0)
    x[1] += 1e4
    for top in (1.0, 0.7):
        check(run(x, tokens, parents, u, temp=temp, top=top), O.verify(x, tokens, parents, u, temp, top))
        check(run(x, tokens, parents, u, q, accept, temp=temp, top=top), O.verify(x, tokens, parents, u, temp, top, q, accept))


@pytest.mark.parametrize("V", [32000, 60001, 120000, 8 * 376 * 128])
@pytest.mark.parametrize("top", [1.0, 0.9])
@pytest.mark.parametrize("drawn", [False, True])
def test_large_vocabularies(V, top, drawn):
    x, tokens, parents, u, q, accept = tree(2, 3, V, V, spread=4.0)
    check(run(x, tokens, parents, u, q if drawn else None, accept, temp=0.8, top=top),
          O.verify(x, tokens, parents, u, 0.8, top, q if drawn else None, accept))


@pytest.mark.parametrize("B,n", [(300, 3), (40, 33), (1, 64)])
def test_many_rows(B, n):
    x, tokens, parents, u, q, accept = tree(B, n, 600, B)
    check(run(x, tokens, parents, u, temp=0.9, top=0.7), O.verify(x, tokens, parents, u, 0.9, 0.7))
    check(run(x, tokens, parents, u, q, accept), O.verify(x, tokens, parents, u, 1.0, 1.0, q, accept))


@pytest.mark.parametrize("top", [1.0, 0.5, 0.26])
def test_ties_and_rows_of_nothing(top):
    """Equal logits everywhere, in blocks, and next to -infinity, NaN and infinity: what is kept goes by the index."""
    V = 700
    x = torch.zeros(6, 1, V)
    x[1, 0, ::2] = -1.0
    x[2] = -math.inf
    x[3, 0, 5:] = -math.inf
    x[4, 0, :3] = torch.tensor([math.nan, math.inf, math.inf])
    x[5] = math.nan
    none = torch.zeros(6, 1, dtype=torch.int32)
    for r in (0.0, 0.2, 0.77, 1.0 - 2.0 ** -24):
        u = torch.full((6, 1), r)
        for temp in (0.0, 1.0, 3.0):
            check(run(x, none, none - 1, u, temp=temp, top=top), O.verify(x, none, none - 1, u, temp, top))


def test_equal_siblings_and_drafts_that_are_none():
    V, n = 50, 6
    x, *_ = tree(1, n, V, 3)
    tokens = torch.tensor([[0, 7, 7, -1, V, 7]], dtype=torch.int32)
    parents = torch.tensor([[-1, 0, 0, 0, 0, 5]], dtype=torch.int32)      # the last one's parent does not stand before it
    q = torch.softmax(x + 1, -1)
    q[0, 0] = 0
    q[0, 0, 7] = 1.0
    for r in (0.0, 0.3, 0.6, 0.9):
        u, a = torch.full((1, n), r), torch.tensor([[0.0, 0.999, 0.0, 0.0, 0.0, 0.0]])
        check(run(x, tokens, parents, u), O.verify(x, tokens, parents, u, 1.0, 1.0))
        check(run(x, tokens, parents, u, q, a), O.verify(x, tokens, parents, u, 1.0, 1.0, q, a))


def test_paths_streams_and_graphs(monkeypatch):
    x, tokens, parents, u, q, a = tree(4, 12, 900, 9)
    want = run(x, tokens, parents, u, q, a, temp=0.7, top=0.95)
    with monkeypatch.context() as m:
        m.setattr(native, "host", None)
        for got, w in zip(run(x, tokens, parents, u, q, a, temp=0.7, top=0.95), want):
            assert torch.equal(got, w)
    big = torch.stack([x.cuda(), x.cuda()], 3)[..., 0]                    # a view that is not contiguous
    more = dict(temp=0.7, top=0.95, draft_probs=q.cuda(), accept=a.cuda())
    for got, w in zip(verify_drafts(big, tokens.cuda(), parents.cuda(), u.cuda(), **more), want):
        assert torch.equal(got, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, tokens, parents, u, q, a, temp=0.7, top=0.95)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(y, w) for y, w in zip(got, want))
    args = [t.cuda() for t in (x, tokens, parents, u, q, a)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verify_drafts(*args[:4], temp=0.7, top=0.95, draft_probs=args[4], accept=args[5])
    other = torch.rand(4, 12)
    args[3].copy_(other)
    graph.replay()
    check(got, O.verify(x, tokens, parents, other, 0.7, 0.95, q, a))
