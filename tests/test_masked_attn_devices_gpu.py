"""Tensors of another device or type beside those of the call are refused, on both host paths."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import functional as F
from create_llm_by_cupy_b200.ops import masked_attn as A
from create_llm_by_cupy_b200.ops import native
from tests.test_masked_attn_gpu import packed

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=["host", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(native, "host", None)


def test_span_attention(path):
    T, D = 70, 64
    q, k, v, dout = packed(1, T, 4, 2, D, 1)
    m = A.span_mask(1, T, DEV)
    o, lse = A.span_attn_fwd(q, k, v, m)
    for kw in (dict(k=k.cpu()), dict(v=v.cpu()), dict(q=q.cpu())):
        with pytest.raises(ValueError):
            A.span_attn_fwd(**{**dict(q=q, k=k, v=v, mask=m), **kw})
    good = dict(dout=dout, q=q, k=k, v=v, o=o, lse=lse, mask=m)
    cos, sin = F.rope_table(T, D, 10000.0, DEV)
    grads = A.span_attn_bwd(**good)
    for kw in (dict(dout=dout.cpu()), dict(k=k.cpu()), dict(v=v.cpu()), dict(o=o.cpu()), dict(lse=lse.cpu()),
               dict(delta=torch.zeros(1, 4, T)), dict(unrotate=(cos, sin.cpu())), dict(out=(grads[0], grads[1], grads[2].cpu()))):
        with pytest.raises(ValueError):
            A.span_attn_bwd(**{**good, **kw})
    for kw in (dict(unrotate=(cos.bfloat16(), sin.bfloat16())), dict(unrotate=(cos, sin.double())), dict(lse=lse.double())):
        with pytest.raises(TypeError):
            A.span_attn_bwd(**{**good, **kw})
    assert native.read_status() == (0, 0)


def test_the_mask_is_made_where_it_was_asked_for(path):
    docs = torch.zeros(1, 64, dtype=torch.int32, device=DEV)
    for device in (DEV, torch.device(DEV), torch.device(DEV, torch.cuda.current_device())):
        assert A.span_mask(1, 64, device, docs=docs).device == docs.device
    for device in ("cpu", torch.device(DEV, torch.cuda.current_device() + 1)):
        with pytest.raises(ValueError):
            A.span_mask(1, 64, device, docs=docs)
    with pytest.raises(ValueError):
        A.span_mask(1, 64, DEV, docs=docs, valid_len=torch.tensor([3], dtype=torch.int32))
