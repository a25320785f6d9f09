"""How many bits the gradients of span attention keep: no more is lost than by the roundings that the kernels are meant to make.

Those are made here in fp64: P to bf16 for dV, dS to bf16 for dQ and dK, delta from an output that is bf16, and the results. The error of
the kernels' gradients, root mean square, may be 8 % more than that (another draw of the same roundings, over more than 10^5 elements, and
fp32 sums); P kept as bf16 for dS as well would make it 12 to 17 % more."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.ops import masked_attn as A
from create_llm_by_cupy_b200.ops import native
from tests.test_masked_attn_gpu import DEV, documents, packed, some_slopes

pytestmark = pytest.mark.gpu


def bf16(x):
    return x.to(torch.bfloat16).double()


def gradients(q, k, v, dout, seen, softcap, slopes, keep_p=lambda p: p):
    """(exact, with the kernels' roundings): dq, dk, dv of each, fp64."""
    T, QH, D = q.shape[1:]
    KVH = k.shape[2]
    t = torch.arange(T, device=q.device)
    both = [[torch.zeros(T, h, D, dtype=torch.float64, device=q.device) for h in (QH, KVH, KVH)] for _ in range(2)]
    for h in range(QH):
        g = h // (QH // KVH)
        qq, kk, vv, do = q[0, :, h].double(), k[0, :, g].double(), v[0, :, g].double(), dout[0, :, h].double()
        x, one = qq @ kk.T / math.sqrt(D), 1.0
        if softcap:
            th = torch.tanh(x / softcap)
            x, one = softcap * th, 1 - th * th
        if slopes is not None:
            x = x - float(slopes[h]) * (t[:, None] - t[None]).abs()
        p = torch.softmax(x.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
        dp, o = do @ vv.T, p @ vv
        for (dq, dk, dv), rounded in zip(both, (False, True)):
            to = bf16 if rounded else (lambda y: y)
            kept = keep_p(p * one) if rounded else p * one
            ds = to(kept * (dp - (do * to(o)).sum(-1, keepdim=True)) / math.sqrt(D))
            dq[:, h] = ds @ kk
            dk[:, g] += ds.T @ qq
            dv[:, g] += to(p).T @ do
    return both[0], [bf16(x) for x in both[1]]


def error(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mod", ["", "cap", "bias"])
@pytest.mark.parametrize("T,mean", [(700, 150), (1500, 0)])
def test_gradients(D, mod, T, mean):
    q, k, v, dout = packed(1, T, 4, 2, D, T)
    cap, slopes = 30.0 if mod == "cap" else 0.0, some_slopes(4) if mod == "bias" else None
    mask = A.span_mask(1, T, DEV, docs=documents(1, T, mean, 0, 1)[0] if mean else None)
    o, lse = A.span_attn_fwd(q, k, v, mask, softcap=cap, slopes=slopes)
    got = A.span_attn_bwd(dout, q, k, v, o, lse, mask, softcap=cap, slopes=slopes)
    want, rounded = gradients(q, k, v, dout, mask.dense()[0], cap, slopes)
    assert native.read_status() == (0, 0)
    for name, x, w, r in zip(("dq", "dk", "dv"), got, want, rounded):
        assert error(x[0], w) <= 1.08 * error(r, w), (name, error(x[0], w), error(r, w))
    # the limit is one that a rounding more would not keep
    for w, r, one_more in zip(want[:2], rounded, gradients(q, k, v, dout, mask.dense()[0], cap, slopes, keep_p=bf16)[1]):
        assert error(one_more, w) > 1.08 * error(r, w)
