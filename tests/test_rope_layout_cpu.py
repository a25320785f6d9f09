"""The kernels' layout of rotary tables follows the tables."""
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops.gemm import rope_tables_transposed


def test_tables_that_are_changed_in_place():
    cos, sin = (x.clone() for x in F.rope_table(6, 8, 100.0, "cpu"))
    first = rope_tables_transposed(cos, sin)
    assert rope_tables_transposed(cos, sin)[0] is first[0]                # laid out once
    for x in (cos, sin):
        x.mul_(-0.5)
        c, s = rope_tables_transposed(cos, sin)[:2]
        assert torch.equal(c, cos.t()) and torch.equal(s, sin.t())


def test_tables_of_inference_mode():
    with torch.inference_mode():
        cos, sin = torch.ones(5, 4), torch.zeros(5, 4)
        first = rope_tables_transposed(cos, sin)
        assert torch.equal(first[0], cos.t()) and rope_tables_transposed(cos, sin)[0] is first[0]
