"""Verification where there are more nodes than clusters and a row is shared by several CTAs: which nodes are passed over depends on the
time, what comes out does not, token for token (the seeds are fixed; see ``test_verify_drafts_gpu``)."""
import pytest
import torch

from . import paged_oracle as O
from .test_verify_drafts_cpu import check, tree
from .test_verify_drafts_gpu import run

pytestmark = pytest.mark.gpu


def on_the_way(B, n, V, seed):
    """A batch of trees that texts go down far: drafts hold what their parents' rows are likely to draw."""
    x, tokens, parents, u, q, accept = tree(B, n, V, seed, spread=9.0)
    return x, tokens, parents, u, q, accept


# rows shared by two, four and eight CTAs, with at most 148, 74 and 37 clusters at a time
@pytest.mark.parametrize("B,n,V", [(8, 32, 32000), (75, 2, 17000), (3, 50, 17000), (4, 40, 60001), (2, 64, 140000)])
@pytest.mark.parametrize("top", [1.0, 0.9])
@pytest.mark.parametrize("drawn", [False, True])
def test_rows_in_clusters(B, n, V, top, drawn):
    x, tokens, parents, u, q, accept = on_the_way(B, n, V, B)
    want = O.verify(x, tokens, parents, u, 0.8, top, q if drawn else None, accept)
    assert sum(len(path) for _, path in want) >= (B + 1) // 2            # some texts get to their later nodes
    args = [t.cuda() for t in (x, tokens, parents, u)] + ([q.cuda(), accept.cuda()] if drawn else [])
    for _ in range(5):
        check(run(*args, temp=0.8, top=top), want)


def test_calls_one_behind_the_other():
    """Workspaces that the allocator hands on: what a call leaves in its own decides nothing in the next."""
    several = [on_the_way(6, 40, 17000, seed) for seed in range(3)]
    cases = [([t.cuda() for t in (x, tok, par, u)], O.verify(x, tok, par, u, 0.7, 0.9)) for x, tok, par, u, _, _ in several]
    got = [(run(*args, temp=0.7, top=0.9), want) for _ in range(4) for args, want in cases]
    for g, want in got:
        check(g, want)


# vocabularies whose slices leave room for more CTAs on an SM than its registers do: between one wave of nodes and the next
@pytest.mark.parametrize("B,n", [(9, 33), (8, 63), (37, 16)])
@pytest.mark.parametrize("V", [600, 4000])
def test_more_nodes_than_places_in_small_vocabularies(B, n, V):
    x, tokens, parents, u, q, accept = on_the_way(B, n, V, n)
    check(run(x, tokens, parents, u, temp=0.7, top=0.9), O.verify(x, tokens, parents, u, 0.7, 0.9))
    check(run(x, tokens, parents, u, q, accept), O.verify(x, tokens, parents, u, 1.0, 1.0, q, accept))
