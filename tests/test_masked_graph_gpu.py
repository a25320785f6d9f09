"""Packed documents in the whole-step CUDA graph: every replay reads the documents of its own batch."""
import pytest
import torch

from create_llm_by_cupy_b200.ops import native
from create_llm_by_cupy_b200.ops.masked_attn import span_mask
from create_llm_by_cupy_b200.parallel.trainer import Trainer
from tests.test_masked_model_gpu import cfg

pytestmark = pytest.mark.gpu
DEV = "cuda"


def batches(n, kinds):
    g = torch.Generator().manual_seed(0)
    for i in range(n):
        x = torch.randint(0, 500, (2, 640), generator=g)
        t = torch.roll(x, -1, 1)
        if kinds[i % len(kinds)] == "lengths":
            yield x.to(DEV), t.to(DEV), torch.tensor([640, 300 + i], dtype=torch.int32, device=DEV)
            continue
        ids = (torch.arange(640) // (40 + 97 * i)).to(torch.int32).expand(2, 640).clone()
        ids[1, 640 - 50 * i:] = -1
        t[ids < 0] = 511
        yield x.to(DEV), t.to(DEV), span_mask(2, 640, DEV, docs=ids.to(DEV))


def losses(kinds, softcap, **kw):
    tr = Trainer(cfg(64, attn_softcap=softcap), device="cuda:0", accum_step=1, lr_max=2e-3, **kw)
    return tr, [float(tr.train_step([b])["loss"]) for b in batches(7, kinds)]


@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("kinds", [["documents"], ["documents", "lengths"], ["lengths", "lengths", "lengths", "documents"]])
def test_replayed_steps_are_the_eager_steps(kinds, softcap):
    """Losses of seven steps on seven batches: a mask that a replay did not take over would put them far apart."""
    _, want = losses(kinds, softcap)
    tr, got = losses(kinds, softcap, cuda_graph=True)
    assert tr._graph is not None and native.read_status() == (0, 0)
    assert max(abs(a - b) for a, b in zip(got, want)) < 2e-3, (got, want)
