"""A model's generation over paged caches, and drawn text from drafted tokens, on the kernels."""
import pytest
import torch

from create_llm_by_cupy_b200.models.model import Cupa_ver4
from create_llm_by_cupy_b200.ops import native
from create_llm_by_cupy_b200.ops.masked_attn import span_mask
from tests.test_masked_model_gpu import cfg

pytestmark = pytest.mark.gpu
DEV = "cuda"
PROMPTS = [list(range(5, 205)), [7], list(range(30, 93)), list(range(100, 140))]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache,near", [("bf16", 0.02), ("int8", 0.03), ("e4m3", 0.1)])
@pytest.mark.parametrize("kw", [{}, dict(attn_softcap=20.0), dict(attn_distance_bias=True)])
def test_batches(D, cache, near, kw):
    """Every chosen token has the largest logit of the full sequence, or one that bf16 (2 % of the largest, as for a single sequence) and
    the cache's half step, 0.4 % or 6 % of its rows, cannot tell from it."""
    m = Cupa_ver4(cfg(D, **kw), device=DEV)
    outs = m.generate_batch(PROMPTS, greedy=True, max_new_tokens=16, cache=cache, prefix=20 if kw else 0)
    for p, out in zip(PROMPTS, outs):
        n = len(p) + len(out)
        mask = span_mask(1, n, DEV, prefix=(torch.arange(n, device=DEV) < min(20, len(p)))[None]) if kw else None
        logits = m.logits(torch.tensor([p + out], device=DEV), x_pa=mask)[0]
        assert len(out) == 16
        logits[:, 511] = -1e30
        for i, tok in enumerate(out):
            row = logits[len(p) + i - 1]
            assert float(row.max() - row[tok]) <= near * float(row.abs()[:511].max())
    assert native.read_status() == (0, 0)


def test_drawn_batches_and_drafts():
    m = Cupa_ver4(cfg(128), device=DEV)
    a = m.generate_batch(PROMPTS, seed=1, max_new_tokens=12, cache="int8")
    assert a == m.generate_batch(PROMPTS, seed=1, max_new_tokens=12, cache="int8")
    assert all(len(x) == 12 and 511 not in x for x in a)
    calls = []
    greedy = m.generate(PROMPTS[2], greedy=True, max_new_tokens=24)

    def draft(tokens):
        calls.append(len(tokens))
        ahead = greedy[len(tokens) - 63:][:6]
        q = torch.full((len(ahead) + 1, 512), 1e-3)
        for i, t in enumerate(ahead):
            q[i, t] = 1.0
        return [(t, i - 1) for i, t in enumerate(ahead)], q / q.sum(-1, keepdim=True)

    # a temperature near 0: the greedy text, most of it from drafts
    out = m.generate_drafted(PROMPTS[2], draft, max_new_tokens=24, temp=1e-3, top=1.0, seed=0)
    logits = m.logits(torch.tensor([PROMPTS[2] + out], device=DEV))[0]
    logits[:, 511] = -1e30
    for i, tok in enumerate(out):
        row = logits[63 + i - 1]
        assert float(row.max() - row[tok]) <= 2e-2 * float(row.abs()[:511].max())
    assert len(out) == 24 and len(calls) < 24
    twice = [m.generate_drafted(PROMPTS[2], draft, max_new_tokens=9, temp=1.0, seed=3) for _ in range(2)]
    assert twice[0] == twice[1]
    assert native.read_status() == (0, 0)
