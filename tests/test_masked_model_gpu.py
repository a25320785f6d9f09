"""The model on packed documents, with capped scores, and with drafted tokens, on the span and tree kernels."""
import pytest
import torch

from create_llm_by_cupy_b200.models.model import Cupa_ver4
from create_llm_by_cupy_b200.ops import native
from create_llm_by_cupy_b200.ops.masked_attn import span_mask, tree_mask
from create_llm_by_cupy_b200.parallel.trainer import Trainer

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cfg(D, **kw):
    return dict(layer_num=2, time_size=640, hidden_size=4 * D, vocab_size=512, kv_head=2, q_head=4, ffn_size=512, padding_id=511, seed=3,
                init_std=0.05, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_packed_documents_are_separate_documents(D, softcap):
    m = Cupa_ver4(cfg(D, attn_softcap=softcap), device=DEV)
    g = torch.Generator().manual_seed(0)
    sizes = [200, 31, 300]
    docs = [torch.randint(0, 500, (n + 1,), generator=g) for n in sizes]
    x, t, ids = torch.full((1, 640), 511), torch.full((1, 640), 511), torch.full((1, 640), -1, dtype=torch.int32)
    at = 0
    for i, d in enumerate(docs):
        n = len(d) - 1
        x[0, at:at + n], t[0, at:at + n], ids[0, at:at + n] = d[:-1], d[1:], i
        at += n

    def run(x, t, mask):
        loss = m.forward(x.to(DEV), t.to(DEV), mask)
        m.backward(1.0)
        return float(loss), [p.float().clone() for p in m.grads]
    loss, grads = run(x, t, span_mask(1, 640, DEV, docs=ids.to(DEV)))
    want, total = [torch.zeros_like(p, dtype=torch.float32) for p in m.params], 0.0
    for d in docs:
        n = len(d) - 1
        part, gs = run(d[None, :-1], d[None, 1:], None)
        total += part * n / sum(sizes)
        for w, p in zip(want, gs):
            w += p * (n / sum(sizes))
    assert native.read_status() == (0, 0)
    assert abs(loss - total) < 5e-3
    for got, w in zip(grads, want):                        # two bf16 passes of different shapes
        assert float((got - w).norm() / w.norm()) < 3e-2


@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_drafted_tokens_see_what_the_sequence_sees(softcap):
    """Hidden states of two branches of drafts against those of the two sequences, through a whole block."""
    m = Cupa_ver4(cfg(64, attn_softcap=softcap), device=DEV)
    gqa, _, norm, _ = m.block_modules(0)
    g = torch.Generator(device=DEV).manual_seed(1)
    h = torch.randn(300, 256, device=DEV, generator=g).to(torch.bfloat16)
    left, right = (torch.randn(3, 256, device=DEV, generator=g).to(torch.bfloat16) for _ in range(2))
    kc, vc = (torch.zeros(1, 2, 640, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    gqa.prefill(norm.forward(h, False), 1, 300, kc, vc)
    drafts = torch.stack([left[0], right[0], left[1], right[1], left[2], right[2]])
    tree = tree_mask([[-1, -1, 0, 1, 2, 3]], DEV)
    got = gqa.decode_drafts(norm.forward(drafts, False), tree, kc, vc, torch.tensor([300], dtype=torch.int32, device=DEV))
    for branch, rows in ((left, got[0::2]), (right, got[1::2])):
        full = torch.cat([h, branch])
        want = gqa.forward(norm.forward(full, False), 1, 303, None, train_flg=False)[300:]
        assert float((rows.float() - want.float()).norm() / want.float().norm()) < 2e-2
    assert native.read_status() == (0, 0)


@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_drafted_generation(softcap):
    """Every chosen token has the largest logit of the full sequence, or one that bf16 cannot tell from it."""
    m = Cupa_ver4(cfg(64, attn_softcap=softcap), device=DEV)
    prompt = list(range(5, 40))
    greedy = m.generate(prompt, greedy=True, max_new_tokens=24)
    calls = []

    def draft(tokens):
        calls.append(len(tokens))
        ahead = greedy[len(tokens) - len(prompt):][:8]
        return [x for i, t in enumerate(ahead) for x in (((t + 1) % 500, 2 * i - 1), (t, 2 * i - 1))]
    out = m.generate_drafted(prompt, draft, max_new_tokens=24)
    assert len(out) == 24 and len(calls) < 24
    logits = m.logits(torch.tensor([prompt + out], device=DEV))[0]
    logits[:, 511] = -1e30
    for i, tok in enumerate(out):
        row = logits[len(prompt) + i - 1]
        assert float(row.max() - row[tok]) <= 2e-2 * float(row.abs()[:511].max())
    assert native.read_status() == (0, 0)


def test_training_steps_on_packed_documents():
    """Through the trainer: the loss of a memorised batch falls, documents and padding in its rows, capped scores."""
    tr = Trainer(cfg(128, attn_softcap=30.0), device="cuda:0", zero_stage="3", accum_step=1, lr_max=2e-3)
    g = torch.Generator().manual_seed(0)
    x = torch.randint(0, 500, (2, 640), generator=g)
    ids = (torch.arange(640) // 150).to(torch.int32).expand(2, 640).clone()
    ids[:, 600:] = -1
    t = torch.roll(x, -1, 1)
    t[ids < 0] = 511
    mask = span_mask(2, 640, DEV, docs=ids.to(DEV))
    losses = [float(tr.train_step([(x.to(DEV), t.to(DEV), mask)])["loss"]) for _ in range(12)]
    assert losses[-1] < losses[0] - 0.5 and native.read_status() == (0, 0)
