"""Drafts that do not fit behind the cached tokens: neither kept nor seen, in the kernels as in the plain restatement."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A
from create_llm_by_cupy_b200.ops import native
from tests.test_masked_attn_gpu import some_slopes, tree_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
# Weights and results of the kernels are bf16, of which each leaves at most 2^-8 of the sum of p |v|; the restatement on the CPU (from the
# same bf16 inputs, in fp32) rounds its result to bf16 too, and the rotated K that both caches hold may differ by a unit of bf16.
LIMIT = 2.0 ** -6


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
@pytest.mark.parametrize("lens,n,QH,KVH,Tmax", [
    ([6], 4, 2, 1, 8), ([8], 1, 4, 2, 8), ([98, 100, 40], 5, 4, 2, 100), ([128, 120], 1, 8, 1, 128), ([250, 256], 64, 8, 1, 256),
    ([1], 9, 2, 2, 1), ([0], 3, 4, 1, 1)])
def test_drafts_behind_the_end(D, mod, lens, n, QH, KVH, Tmax):
    kqv, kc, vc, lt, tree, _ = tree_case(lens, n, QH, KVH, D, Tmax, seed=n)
    cos, sin = F.rope_table(Tmax + n, D, 10000.0, DEV)
    kw = dict(softcap=25.0 if mod == "cap" else 0.0)
    slopes = some_slopes(QH) if mod == "bias" else None
    kc1, vc1 = kc.cpu(), vc.cpu()
    want = A.tree_attn_append(kqv.cpu(), kc1, vc1, lt.cpu(), tree.cpu(), QH, KVH, cos.cpu(), sin.cpu(),
                              slopes=None if slopes is None else slopes.cpu(), **kw).float()
    got = A.tree_attn_append(kqv, kc, vc, lt, tree, QH, KVH, cos, sin, slopes=slopes, **kw).float().cpu()
    assert native.read_status() == (0, 0)
    most = float(torch.where(vc1.isfinite(), vc1, torch.zeros_like(vc1)).float().abs().max())
    assert bool(torch.isfinite(got).all()) and float((got - want).abs().max()) <= LIMIT * most
    assert float((got - want).norm()) <= LIMIT * float(want.norm())
    assert torch.equal(vc.cpu().nan_to_num(posinf=7.0), vc1.nan_to_num(posinf=7.0))


@pytest.mark.parametrize("D", [64, 128])
def test_nothing_cached_and_nothing_kept(D):
    """A draft that sees none but drafts that were not kept has nothing to attend to: zeros."""
    kqv, kc, vc, lt, tree, _ = tree_case([0], 3, 4, 2, D, 1)
    cos, sin = F.rope_table(4, D, 10000.0, DEV)
    tree[0] = torch.tensor([1, 2, 6])                      # the last two see themselves and one another alone
    o = A.tree_attn_append(kqv, kc, vc, lt, tree, 4, 2, cos, sin)
    assert not o[0, 1:].any() and not math.isnan(float(o.sum()))
    v = kqv.view(3, 8, D)[0, 6:].repeat_interleave(2, 0)   # the first sees itself: its own values
    assert torch.equal(o[0, 0], v) and native.read_status() == (0, 0)
