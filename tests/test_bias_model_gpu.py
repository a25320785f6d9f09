"""The model with a distance bias in place of a rotation, on the span and tree kernels."""
import pytest
import torch

from create_llm_by_cupy_b200.models.model import Cupa_ver4
from create_llm_by_cupy_b200.ops import native
from create_llm_by_cupy_b200.ops.masked_attn import span_mask
from create_llm_by_cupy_b200.parallel.trainer import Trainer
from tests.test_masked_model_gpu import cfg

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 128])
def test_loss_and_gradients_of_the_plain_restatement(D):
    """The same weights on the CPU, in fp32."""
    m = Cupa_ver4(cfg(D, attn_distance_bias=True), device=DEV)
    ref = Cupa_ver4(cfg(D, attn_distance_bias=True, dtype="fp32"), device="cpu")
    for a, b in zip(ref.params, m.params):
        a.copy_(b.float().cpu())
    g = torch.Generator().manual_seed(0)
    x = torch.randint(0, 500, (2, 300), generator=g)
    t = torch.roll(x, -1, 1)
    docs = (torch.arange(300) // 130).to(torch.int32).expand(2, 300).contiguous()
    loss = m.forward(x.to(DEV), t.to(DEV), span_mask(2, 300, DEV, docs=docs.to(DEV)))
    m.backward(1.0)
    want = ref.forward(x, t, span_mask(2, 300, "cpu", docs=docs))
    ref.backward(1.0)
    assert abs(float(loss) - float(want)) < 5e-3
    for got, w in zip(m.grads, ref.grads):                 # a bf16 pass beside an fp32 one
        assert float((got.float().cpu() - w).norm() / w.norm()) < 3e-2
    assert native.read_status() == (0, 0)


def test_generation_and_drafts():
    """Every chosen token has the largest logit of the full sequence, or one that bf16 cannot tell from it."""
    m = Cupa_ver4(cfg(64, attn_distance_bias=True), device=DEV)
    prompt = list(range(5, 40))
    greedy = m.generate(prompt, greedy=True, max_new_tokens=24)
    drafted = m.generate_drafted(prompt, lambda toks: [(t, i - 1) for i, t in enumerate(greedy[len(toks) - len(prompt):][:8])],
                                 max_new_tokens=24)
    for out in (greedy, drafted):
        assert len(out) == 24
        logits = m.logits(torch.tensor([prompt + out], device=DEV))[0]
        logits[:, 511] = -1e30
        for i, tok in enumerate(out):
            row = logits[len(prompt) + i - 1]
            assert float(row.max() - row[tok]) <= 2e-2 * float(row.abs()[:511].max())
    assert native.read_status() == (0, 0)


def test_training_steps():
    tr = Trainer(cfg(128, attn_distance_bias=True), device="cuda:0", zero_stage="3", accum_step=1, lr_max=2e-3)
    g = torch.Generator().manual_seed(0)
    x = torch.randint(0, 500, (2, 640), generator=g)
    t = torch.roll(x, -1, 1)
    n = torch.tensor([640, 500], dtype=torch.int32)
    t[1, 500:] = 511
    losses = [float(tr.train_step([(x.to(DEV), t.to(DEV), n.to(DEV))])["loss"]) for _ in range(12)]
    assert losses[-1] < losses[0] - 0.5 and native.read_status() == (0, 0)
