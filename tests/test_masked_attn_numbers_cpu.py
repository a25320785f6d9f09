"""Caps and scales that fp32 arithmetic has no room for are refused; those at the edge are what they are."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A

WRONG = [dict(softcap=1e-46), dict(softcap=1e-19), dict(softcap=1e39), dict(softcap=1e19), dict(scale=1e-46), dict(scale=1e-19),
         dict(scale=1e39), dict(scale=1e19)]


@pytest.mark.parametrize("kw", WRONG)
def test_refused(kw):
    q = torch.zeros(1, 4, 2, 8)
    m = A.span_mask(1, 4, "cpu")
    with pytest.raises(ValueError):
        A.span_attn_fwd(q, q, q, m, **kw)
    with pytest.raises(ValueError):
        A.span_attn_bwd(q, q, q, q, q, torch.zeros(1, 2, 4), m, **kw)
    cos, sin = F.rope_table(8, 8, 10000.0, "cpu")
    with pytest.raises(ValueError):
        A.tree_attn_append(torch.zeros(1, 6 * 8), torch.zeros(1, 2, 8, 8), torch.zeros(1, 2, 8, 8), torch.zeros(1, dtype=torch.int32),
                           torch.ones(1, 1, dtype=torch.int64), 2, 2, cos, sin, **kw)


@pytest.mark.parametrize("softcap", [1e-18, 1e18])
def test_taken(softcap):
    q = torch.randn(1, 4, 2, 8, dtype=torch.float64)
    o, lse = A.span_attn_fwd(q, q, q, A.span_mask(1, 4, "cpu"), softcap=softcap)
    assert bool(torch.isfinite(o).all() and torch.isfinite(lse).all())
    if softcap < 1:                                        # no score differs from another: the mean of what is seen
        assert torch.allclose(o, q.cumsum(1) / torch.arange(1, 5)[None, :, None, None]) and abs(float(lse[0, 0, 3]) - math.log(4)) < 1e-12
