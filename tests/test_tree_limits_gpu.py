"""Tree attention kernels inside limits that a cap, a key or half of the queries' bits cannot be missing in (tests/tree_limits.py)."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import masked_attn as A
from create_llm_by_cupy_b200.ops import native
from tests.tree_limits import CASES, attention, good, make, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("path", ["host", "python"])
@pytest.mark.parametrize("name", list(CASES))
def test_tree_attention(name, path, monkeypatch):
    if path == "python":
        monkeypatch.setattr(native, "host", None)
    a, parents = make(name, "cuda")
    before = a["kcache"].clone(), a["vcache"].clone()
    got = A.tree_attn_append(**a)
    assert native.read_status() == (0, 0)
    n = a["tree"].shape[1]
    for b, L in enumerate(CASES[name][0]):
        _, k, v, _, _, _ = rows_of(a, parents, b)
        for cache, rows, old in ((a["kcache"], k, before[0]), (a["vcache"], v, before[1])):
            # rotated in fp32 (2^-22 of the larger of the two terms) and rounded to bf16
            assert torch.allclose(cache[b, :, L:L + n].double(), rows.transpose(0, 1), rtol=2.0 ** -8, atol=1e-5)
            assert torch.equal(cache[b, :, :L], old[b, :, :L])
            assert torch.equal(cache[b, :, L + n:].nan_to_num(9.0, 7.0), old[b, :, L + n:].nan_to_num(9.0, 7.0))
        assert torch.equal(a["vcache"][b, :, L:L + n].double(), v.transpose(0, 1))
    want, bound = attention(a, parents)
    off = got.double() - want
    assert good(got, want, bound), (float((off.abs() / bound).max()), float(off.norm() / want.norm()))
