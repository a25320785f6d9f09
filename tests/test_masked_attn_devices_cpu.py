"""Tensors of one call stand on one device: whatever does not is refused before its address goes anywhere."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import masked_attn as A

B, T, QH, KVH, D = 1, 6, 2, 1, 8
META = torch.device("meta")                                # (a device without memory, in place of another GPU)


def call():
    q, k, v = (torch.zeros(B, T, h, D) for h in (QH, KVH, KVH))
    m = A.span_mask(B, T, "cpu")
    o, lse = A.span_attn_fwd(q, k, v, m)
    return dict(dout=q, q=q, k=k, v=v, o=o, lse=lse, mask=m)


@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_forward(name):
    a = call()
    kw = {n: a[n] for n in ("q", "k", "v", "mask")}
    kw[name] = kw[name].to(META)
    with pytest.raises(ValueError):
        A.span_attn_fwd(**kw)


@pytest.mark.parametrize("name", ["dout", "k", "v", "o", "lse", "delta", "unrotate", "out"])
def test_backward(name):
    kw = call()
    if name == "delta":
        kw["delta"] = torch.zeros(B, QH, T, device=META)
    elif name == "unrotate":
        kw["unrotate"] = (torch.ones(T, D // 2), torch.zeros(T, D // 2, device=META))
    elif name == "out":
        kw["out"] = (torch.zeros(B, T, QH, D), torch.zeros(B, T, KVH, D), torch.zeros(B, T, KVH, D, device=META))
    else:
        kw[name] = kw[name].to(META)
    with pytest.raises(ValueError):
        A.span_attn_bwd(**kw)


def test_shapes_of_what_is_given_beside_the_tensors():
    kw = call()
    for more in (dict(delta=torch.zeros(B, QH, T + 1)), dict(out=(torch.zeros(B, T, QH, D), torch.zeros(B, T, KVH, D))),
                 dict(out=(torch.zeros(B, T, QH, D), torch.zeros(B, T, KVH, D), torch.zeros(B, T + 1, KVH, D)))):
        with pytest.raises(ValueError):
            A.span_attn_bwd(**kw, **more)
