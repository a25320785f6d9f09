"""A pool that the kernels write and one that the plain form writes in fp32 are the same bit for bit: rows, and scales."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import paged as P

from . import paged_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def written(kind, D, device, k, v, cos, sin):
    M, KVH, _ = k.shape
    cache = P.paged_cache(M // 64, KVH, 64, D, device, kind)
    table = torch.arange(M // 64, dtype=torch.int32, device=device)[None]
    seq, pos = torch.zeros(M, dtype=torch.int32, device=device), torch.arange(M, dtype=torch.int32, device=device)
    P.paged_append(k.to(device), v.to(device), cache, table, seq, pos, cos.to(device), sin.to(device))
    return cache


@pytest.mark.parametrize("kind", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_and_scales(kind, D):
    M, KVH, QH = 2048, 3, 6
    g = torch.Generator().manual_seed(D)
    k, v = (torch.randn(M, KVH, D, generator=g) * torch.exp2(torch.randint(-30, 30, (M, KVH, 1), generator=g).float()) for _ in range(2))
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    v[5], v[6, :, 3:] = 0, 0
    cos, sin = O.tables(M, D)
    here, there = written(kind, D, DEV, k, v, cos, sin), written(kind, D, "cpu", k, v, cos, sin)
    # and a decoded token, in the place of the last row
    kqv, n = torch.randn(1, (2 * KVH + QH) * D, generator=g).to(torch.bfloat16), torch.tensor([M - 1], dtype=torch.int32)
    table = torch.arange(M // 64, dtype=torch.int32)[None]
    for cache, dev in ((here, DEV), (there, "cpu")):
        P.paged_attn_append(kqv.to(dev), cache, table.to(dev), n.to(dev), QH, KVH, cos.to(dev), sin.to(dev))
    for a, b in zip(here, there):
        assert (a is None) == (b is None)
        if a is not None:
            assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
