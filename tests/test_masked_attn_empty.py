"""Calls without sequences, without tokens and without heads: the same on the CPU and on the kernels' side."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def zeros(dev, *shape):
    return torch.zeros(*shape, dtype=torch.bfloat16, device=dev)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("B,T", [(0, 5), (2, 0), (0, 0)])
def test_no_tokens(dev, B, T):
    q, k = zeros(dev, B, T, 4, 64), zeros(dev, B, T, 2, 64)
    m = A.span_mask(B, T, dev, docs=torch.zeros(B, T, dtype=torch.int32, device=dev))
    o, lse = A.span_attn_fwd(q, k, k, m)
    assert o.shape == q.shape and lse.shape == (B, 4, T)
    grads = A.span_attn_bwd(q, q, k, k, o, lse, m)
    assert [g.shape for g in grads] == [q.shape, k.shape, k.shape]


@pytest.mark.parametrize("dev", DEVICES)
def test_no_sequences_of_drafts(dev):
    cos, sin = F.rope_table(8, 64, 10000.0, dev)
    c = zeros(dev, 0, 1, 8, 64)
    o = A.tree_attn_append(zeros(dev, 0, 4 * 64), c, c.clone(), torch.zeros(0, dtype=torch.int32, device=dev),
                           torch.zeros(0, 3, dtype=torch.int64, device=dev), 2, 1, cos, sin)
    assert o.shape == (0, 3, 2, 64)


@pytest.mark.parametrize("dev", DEVICES)
def test_no_heads_are_refused(dev):
    m = A.span_mask(1, 3, dev)
    for qh, kvh in ((0, 1), (1, 0), (0, 0)):
        q, k = zeros(dev, 1, 3, qh, 64), zeros(dev, 1, 3, kvh, 64)
        with pytest.raises(ValueError):
            A.span_attn_fwd(q, k, k, m)
