"""The limits of tests/tree_limits.py: the roundings that the kernel makes keep them, and mistakes do not."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import masked_attn as A
from tests.tree_limits import CASES, attention, good, make


def bf16(x):
    return x.to(torch.float32).to(torch.bfloat16).double()


def two_parts(q):
    return bf16(q) + bf16(q - bf16(q))


@pytest.fixture(scope="module", params=list(CASES))
def case(request):
    a, parents = make(request.param, "cpu")
    A.tree_attn_append(**a)                                # appends the drafts' rows
    return request.param, a, parents, attention(a, parents)


def kernel(a, parents, **mistake):
    """What the kernel's roundings make of it, with a mistake or without."""
    return bf16(attention(a, parents, **{**dict(q_of=two_parts, p_of=bf16), **mistake})[0])


def test_the_kernels_roundings_keep_the_limits(case):
    _, a, parents, want = case
    assert good(kernel(a, parents), *want)


def test_a_cap_that_is_not_taken_is_noticed(case):
    _, a, parents, want = case
    if a["softcap"] == 0.0:
        pytest.skip("no cap")
    assert not good(kernel(a, parents, cap=0.0), *want)
    assert not good(kernel(a, parents, cap=1.05 * a["softcap"]), *want)


def test_a_lost_key_is_noticed(case):
    """The first, one in the middle, those on both sides of a tile's edge, the last cached one; of the longest sequence."""
    name, a, parents, want = case
    if "large scores" in name or name == "biased":
        pytest.skip("most keys weigh next to nothing")
    L = int(a["lens"].max())
    for at in (0, L // 2, 127, 128, (L - 1) // 128 * 128, L - 1):
        if len(CASES[name][0]) == 1:
            assert not good(kernel(a, parents, lost=at), *want), at


def test_queries_in_one_part_are_noticed(case):
    name, a, parents, want = case
    if "large scores" not in name and name != "two row tiles, capped":
        pytest.skip("scores so small that 8 bits of the queries are enough")
    assert not good(kernel(a, parents, q_of=bf16), *want)
