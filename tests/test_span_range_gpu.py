"""Span attention where the grid, the walk of the batch and the sequences are long: units that CTAs take over from one another, batches
whose K and V are walked in parts, key tiles in every number of CTAs that the rule gives, thousands of tokens."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import masked_attn as A
from tests.test_masked_attn_gpu import DEV, check, documents, packed, some_slopes

pytestmark = pytest.mark.gpu


def modifier(mod, QH):
    return dict(softcap=20.0 if mod == "cap" else 0.0, slopes=some_slopes(QH) if mod == "bias" else None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
def test_more_units_than_ctas(D, mod):
    """576 units of head_dim 128, 1152 of 64, where 148 and 296 CTAs are resident; a row of padding alone, rows that end in it; 288 key
    tiles of four query heads: two CTAs to a tile."""
    B, T, QH, KVH = 6, 700, 32, 8
    docs, prefix = documents(B, T, 150, 40, 1)
    docs[2] = -1
    docs[4, 100:] = -1
    mask = A.span_mask(B, T, DEV, docs=docs, prefix=prefix)
    check(*packed(B, T, QH, KVH, D, 2), mask, **modifier(mod, QH))


@pytest.mark.parametrize("mod", ["", "cap"])
def test_batches_in_parts(mod):
    """K and V of four batch elements are walked together in the forward, of two in the backward: the last part is smaller."""
    B, T, H = 5, 512, 64
    docs, _ = documents(B, T, 120, 30, 3)
    docs[3] = -1
    check(*packed(B, T, H, H, 128, 4), A.span_mask(B, T, DEV, docs=docs), **modifier(mod, H))


def test_key_tiles_of_a_cta_each():
    """576 key tiles of four query heads: more than three rounds of the SMs."""
    B, T, QH, KVH = 6, 700, 64, 16
    docs, _ = documents(B, T, 200, 0, 5)
    check(*packed(B, T, QH, KVH, 64, 6), A.span_mask(B, T, DEV, docs=docs))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
@pytest.mark.parametrize("T,mean", [(2049, 0), (4100, 0), (4100, 900)])
def test_thousands_of_tokens(D, mod, T, mean):
    docs = documents(1, T, mean, 60, 7)[0] if mean else None
    check(*packed(1, T, 2, 1, D, 8), A.span_mask(1, T, DEV, docs=docs), **modifier(mod, 2))


@pytest.mark.parametrize("D", [64, 128])
def test_windows_over_thousands_of_tokens(D):
    """Every query sees 300 keys up to itself: tiles that none of a pair of query tiles sees in between, and long walks of short spans."""
    T = 3000
    t = torch.arange(T, dtype=torch.int32, device=DEV)
    lo, hi = (t - 299).clamp_min(0), t + 1
    far = t // 128 % 4 == 3                                # every fourth tile: the first keys
    lo, hi = torch.where(far, 0 * t, lo), torch.where(far, 0 * t + 5, hi)
    check(*packed(1, T, 4, 2, D, 9), A.SpanMask.from_spans(lo[None].contiguous(), hi[None].contiguous()))
