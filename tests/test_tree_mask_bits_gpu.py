"""Bits of a draft's mask behind the drafts that there are: nobody to see, and no step of depth either."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A
from create_llm_by_cupy_b200.ops import native
from tests.test_masked_attn_gpu import some_slopes, tree_case

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n", [1, 5, 63, 64])
def test_bits_of_drafts_that_are_not_there(D, bias, n):
    kqv, kc, vc, lt, tree, _ = tree_case([90, 3], n, 4, 2, D, 200, seed=n)
    cos, sin = F.rope_table(300, D, 10000.0, DEV)
    slopes = some_slopes(4) if bias else None
    more = 0 if n == 64 else -1 << n                       # every bit from n on
    kc1, vc1 = kc.clone(), vc.clone()
    want = A.tree_attn_append(kqv, kc1, vc1, lt, tree, 4, 2, cos, sin, slopes=slopes)
    got = A.tree_attn_append(kqv, kc, vc, lt, tree | more, 4, 2, cos, sin, slopes=slopes)
    assert torch.equal(got, want) and native.read_status() == (0, 0)
    for b, L in enumerate((90, 3)):
        assert torch.equal(kc[b, :, :L + n], kc1[b, :, :L + n]) and torch.equal(vc[b, :, :L + n], vc1[b, :, :L + n])
