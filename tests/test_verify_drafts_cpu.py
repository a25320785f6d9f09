"""Verification of drafted tokens: the plain form against the definition, what it refuses, and that what is kept is distributed as the
target's own text is."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops.drafts import verify_drafts

from . import paged_oracle as O


def tree(B, n, V, seed, width=3, spread=2.0, dtype=torch.float32):
    """Random logits, parents (absent drafts among them), drafts that are often right, and numbers."""
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B, n, V, generator=g) * spread).to(dtype)
    parents = torch.full((B, n), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(1, n):
            parents[b, i] = int(torch.randint(max(0, i - width), i, (1,), generator=g)) if torch.rand(1, generator=g) > 0.1 else -1
    probs = torch.softmax(logits.float() + 0.3 * torch.randn(B, n, V, generator=g), -1)
    tokens = torch.multinomial(probs.view(-1, V), n, replacement=True, generator=g).view(B, n, n)
    of_parent = torch.gather(tokens, 1, parents.clamp_min(0).long()[..., None].expand(B, n, n))
    tokens = of_parent[:, torch.arange(n), torch.arange(n)].to(torch.int32)
    return logits, tokens, parents, torch.rand(B, n, generator=g), probs, torch.rand(B, n, generator=g)


def check(got, want):
    tokens, path, count = (x.cpu() for x in got)
    for b, (t, p) in enumerate(want):
        n = tokens.shape[1]
        assert int(count[b]) == len(p)
        assert tokens[b].tolist() == t + [-1] * (n - len(t))
        assert path[b].tolist() == p + [-1] * (n - len(p))


@pytest.mark.parametrize("temp", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("top", [1.0, 0.8, 1e-9])
@pytest.mark.parametrize("drawn", [False, True])
def test_against_the_definition(temp, top, drawn):
    for seed, (B, n, V) in enumerate([(1, 1, 1), (3, 1, 40), (4, 9, 17), (2, 64, 33)]):
        logits, tokens, parents, u, q, accept = tree(B, n, V, seed)
        kw = dict(draft_probs=q, accept=accept) if drawn else {}
        check(verify_drafts(logits, tokens, parents, u, temp=temp, top=top, **kw),
              O.verify(logits, tokens, parents, u, temp, top, q if drawn else None, accept))


def test_ties_and_rows_of_nothing():
    logits = torch.zeros(1, 2, 8)
    tokens, parents = torch.tensor([[0, 3]], dtype=torch.int32), torch.tensor([[-1, 0]], dtype=torch.int32)
    u = torch.tensor([[0.9, 0.1]])
    # eight equal tokens: the nucleus of half the mass is the first four
    check(verify_drafts(logits, tokens, parents, u, top=0.5), [([3, 0], [1])])
    check(verify_drafts(logits, tokens, parents, u, temp=0.0), [([0], [])])
    logits[0, 1] = -math.inf
    check(verify_drafts(logits, tokens, parents, u, top=0.5), [([3, -1], [1])])
    logits[0, 0] = torch.tensor([math.nan, -math.inf, math.inf, math.inf, 5.0, 0.0, 0.0, 0.0])
    check(verify_drafts(logits, tokens, parents, u), [([3, -1], [1])])
    check(verify_drafts(logits, tokens, parents, u, temp=0.0), [([2], [])])


def test_kept_text_is_distributed_as_the_targets():
    """Two tokens from a chain of drafts: counts of every pair against the product of the target's probabilities. 40000 texts, 9 pairs:
    a count's standard deviation is at most 100; six of them."""
    N, V = 40000, 3
    g = torch.Generator().manual_seed(5)
    target = torch.randn(1, V, V, generator=g)                   # behind the root, and behind each first token
    p0, p1 = torch.softmax(target[0, 0], 0), torch.softmax(torch.randn(V, V, generator=g), -1)
    q0 = torch.softmax(torch.randn(V, generator=g), 0)
    first = torch.multinomial(q0, N * 2, replacement=True, generator=g).view(N, 2)        # two children of the root
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32).expand(N, 3).contiguous()
    tokens = torch.cat([torch.zeros(N, 1, dtype=torch.long), first], 1).to(torch.int32)
    logits = torch.stack([p0.log().expand(N, V), p1[first[:, 0]].log(), p1[first[:, 1]].log()], 1).contiguous()
    u, a = torch.rand(N, 3, generator=g), torch.rand(N, 3, generator=g)
    for kw in (dict(draft_probs=q0.expand(N, 3, V).contiguous(), accept=a), {}):
        tok, _, count = verify_drafts(logits, tokens, parents, u, **kw)
        for x in range(V):
            assert abs(int((tok[:, 0] == x).sum()) - N * float(p0[x])) < 600
            for y in range(V):                                   # behind a kept draft
                there = (tok[:, 0] == x) & (count > 0)
                n = int(there.sum())
                assert abs(int((there & (tok[:, 1] == y)).sum()) - n * float(p1[x, y])) < 600


def test_refusals():
    logits, tokens, parents, u, q, a = tree(2, 4, 9, 0)
    good = dict(logits=logits, tokens=tokens, parents=parents, u=u, temp=1.0, top=1.0)
    verify_drafts(**good)
    for bad in (dict(logits=logits[0]), dict(logits=logits[:, :, :0]), dict(tokens=tokens.long()), dict(parents=parents[:1]),
                dict(u=u.double()), dict(temp=-1.0), dict(temp=math.nan), dict(temp=math.inf), dict(temp=1e-9), dict(temp=2e6),
                dict(top=0.0), dict(top=math.nan),
                dict(draft_probs=q), dict(accept=a), dict(draft_probs=q.double(), accept=a), dict(draft_probs=q, accept=a[:, :2])):
        with pytest.raises(ValueError):
            verify_drafts(**{**good, **bad})
    with pytest.raises(TypeError):
        verify_drafts(**{**good, "logits": logits.half()})
    many = torch.zeros(1, 65, 2)
    with pytest.raises(ValueError):
        verify_drafts(many, torch.zeros(1, 65, dtype=torch.int32), torch.zeros(1, 65, dtype=torch.int32), torch.zeros(1, 65))
    out = verify_drafts(logits[:0], tokens[:0], parents[:0], u[:0])
    assert [tuple(x.shape) for x in out] == [(0, 4), (0, 4), (0,)]
