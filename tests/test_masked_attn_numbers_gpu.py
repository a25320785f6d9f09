"""Caps far below the scores, where the polynomials' coefficients leave fp32, and at both ends of what is taken; scores of 0 among them."""
import math
import random

import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A
from create_llm_by_cupy_b200.ops import native
from tests.masked_oracle import span_oracle, within
from tests.test_masked_attn_cpu import some_parents
from tests.test_masked_attn_gpu import packed
from tests.test_masked_attn_numbers_cpu import WRONG

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [1e-18, 1e-8, 1e-6, 1e-4, 1e-2, 1e18])
@pytest.mark.parametrize("zero", ["none", "half", "all"])
def test_span_attention(D, cap, zero):
    T = 200
    q, k, v, dout = packed(1, T, 2, 1, D, 3)
    q = q.clone()
    if zero != "none":
        q[:, :T // 2 if zero == "half" else T] = 0         # (whole warps of rows whose scores are all 0)
    mask = A.span_mask(1, T, DEV)
    want = span_oracle(q, k, v, mask.dense(), 1 / math.sqrt(D), cap, None, dout)
    o, lse = A.span_attn_fwd(q, k, v, mask, softcap=cap)
    within(o, want["o"], want["o_b"], "o")
    assert bool(((lse.double() - want["lse"]).abs() <= 2 ** -18 * (1 + want["lse"].abs())).all())
    # dq and dk are scaled by 1 - tanh^2, which fp32 has as 2^-23 of 1 at best where the scores are far beyond the cap
    grads = A.span_attn_bwd(dout, q, k, v, o, lse, mask, softcap=cap)
    slack = 2.0 ** -22 * T * D * 64
    for got, n in zip(grads, ("dq", "dk", "dv")):
        within(got, want[n], want[n + "_b"] + (slack if n != "dv" else 0.0), n)
    assert native.read_status() == (0, 0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [1e-18, 1e-8, 1e-4])
def test_tree_attention_of_scores_that_are_all_alike(D, cap):
    """Under a cap of next to nothing every key that is seen weighs the same: the mean of their values."""
    n, L, QH, KVH, Tmax = 5, 140, 4, 2, 160
    g = torch.Generator(device=DEV).manual_seed(1)
    parents = some_parents(random.Random(1), n)
    for std in (0.0, 1.5):
        kqv = (torch.randn(n, (2 * KVH + QH) * D, device=DEV, generator=g) * std).to(torch.bfloat16)
        kc, vc = (torch.randn(1, KVH, Tmax, D, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
        cos, sin = F.rope_table(Tmax, D, 10000.0, DEV)
        got = A.tree_attn_append(kqv, kc, vc, torch.tensor([L], dtype=torch.int32, device=DEV), A.tree_mask([parents], DEV), QH, KVH,
                                 cos, sin, softcap=cap)
        assert native.read_status() == (0, 0)
        for i in range(n):
            at, j = list(range(L)) + [L + i], parents[i]
            while j >= 0:
                at, j = at + [L + j], parents[j]
            mean = vc[0, :, at].double().mean(1).repeat_interleave(QH // KVH, 0)
            # weights within exp(2 cap) of one another, a bf16 each; the result a bf16
            limit = (2 * 2.0 ** -8 + 4 * cap) * vc[0, :, at].double().abs().mean(1).repeat_interleave(QH // KVH, 0)
            assert bool(((got[0, i].double() - mean).abs() <= limit).all())


@pytest.mark.parametrize("path", ["host", "python"])
@pytest.mark.parametrize("kw", WRONG)
def test_refused(kw, path, monkeypatch):
    if path == "python":
        monkeypatch.setattr(native, "host", None)
    q, k, v, dout = packed(1, 64, 2, 1, 64, 1)
    m = A.span_mask(1, 64, DEV)
    with pytest.raises(ValueError):
        A.span_attn_fwd(q, k, v, m, **kw)
    with pytest.raises(ValueError):
        A.span_attn_bwd(dout, q, k, v, dout, torch.zeros(1, 2, 64, device=DEV), m, **kw)
    cos, sin = F.rope_table(16, 64, 10000.0, DEV)
    c = torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        A.tree_attn_append(torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device=DEV), c, c.clone(),
                           torch.zeros(1, dtype=torch.int32, device=DEV), torch.ones(1, 1, dtype=torch.int64, device=DEV), 2, 1, cos, sin,
                           **kw)
