"""The model on packed documents, with capped scores, and its greedy decoding with drafted tokens (CPU restatements)."""
import random

import pytest
import torch

from create_llm_by_cupy_b200.models.layers import GroupedQueryAttention
from create_llm_by_cupy_b200.models.model import Cupa_ver4
from create_llm_by_cupy_b200.ops.masked_attn import span_mask

CFG = dict(layer_num=2, time_size=24, hidden_size=32, vocab_size=40, kv_head=2, q_head=4, ffn_size=48, padding_id=39, seed=3, init_std=0.3,
           dtype="fp32")


def model(**kw):
    return Cupa_ver4({**CFG, **kw}, device="cpu")


def grads_of(m, x, t, x_pa):
    loss = m.forward(x, t, x_pa)
    m.backward(1.0)
    return float(loss), [g.clone() for g in m.grads]


@pytest.mark.parametrize("softcap", [0.0, 2.0])
def test_packed_documents_are_separate_documents(softcap):
    """One row of three documents and padding: the mean loss and the gradients of the documents in rows of their own."""
    g = torch.Generator().manual_seed(0)
    sizes = [5, 9, 7]
    docs = [torch.randint(0, 38, (n + 1,), generator=g) for n in sizes]
    x, t, ids = torch.full((1, 24), 39), torch.full((1, 24), 39), torch.full((1, 24), -1, dtype=torch.int32)
    at = 0
    for i, d in enumerate(docs):
        n = len(d) - 1
        x[0, at:at + n], t[0, at:at + n], ids[0, at:at + n] = d[:-1], d[1:], i
        at += n
    m = model(attn_softcap=softcap)
    loss, grads = grads_of(m, x, t, span_mask(1, 24, "cpu", docs=ids))
    want, total = [torch.zeros_like(p) for p in m.params], 0.0
    for d in docs:
        n = len(d) - 1
        part, gs = grads_of(m, d[None, :-1], d[None, 1:], None)
        total += part * n / sum(sizes)
        for w, p in zip(want, gs):
            w += p * (n / sum(sizes))
    assert abs(loss - total) < 1e-5
    for got, w in zip(grads, want):
        assert torch.allclose(got, w, atol=2e-5, rtol=1e-3)


@pytest.mark.parametrize("keep", [True, False])
def test_capped_model_backward_by_differences(keep):
    """d loss along the gradient, from two losses; also with the recompute switches."""
    g = torch.Generator().manual_seed(1)
    x = torch.randint(0, 38, (2, 12), generator=g)
    t = torch.randint(0, 38, (2, 12), generator=g)
    n = torch.tensor([12, 7], dtype=torch.int32)
    m = model(attn_softcap=1.5, gqa_cache_out_value=keep, gqa_cache_kqv=keep)
    _, grads = grads_of(m, x, t, n)
    for i in (0, 1, 4):                                    # K | Q | V, the output projection, a norm
        d = grads[i] / grads[i].norm()
        eps, f = 2e-2, []
        for s in (eps, -eps):
            m.params[i].add_(d, alpha=s)
            f.append(float(m.forward(x, t, n, train_flg=False)))
            m.params[i].add_(d, alpha=-s)
        assert abs((f[0] - f[1]) / (2 * eps) - float(grads[i].norm())) < 2e-2 * float(grads[i].norm()) + 1e-4


@pytest.mark.parametrize("softcap", [0.0, 2.0])
def test_generation_reads_the_same_attention(softcap):
    """Greedy decoding chooses what the full-sequence logits say."""
    m = model(attn_softcap=softcap, padding_id=-1)
    prompt = [3, 17, 8]
    out = m.generate(prompt, greedy=True, max_new_tokens=10)
    for i, tok in enumerate(out):
        logits = m.logits(torch.tensor([prompt + out[:i]]))[0, -1]
        assert int(logits.argmax()) == tok


@pytest.mark.parametrize("softcap", [0.0, 2.0])
@pytest.mark.parametrize("kind", ["none", "right", "wrong", "mixed", "branches"])
def test_drafted_generation_is_greedy_generation(softcap, kind):
    m = model(attn_softcap=softcap)
    prompt = [3, 17, 8]
    want = m.generate(prompt, greedy=True)
    rng, calls = random.Random(0), []

    def draft(tokens):
        calls.append(len(tokens))
        ahead = want[len(tokens) - len(prompt):]
        if kind == "none":
            return []
        if kind == "right":
            return [(t, i - 1) for i, t in enumerate(ahead[:6])]
        if kind == "wrong":
            return [((t + 1) % 39, i - 1) for i, t in enumerate(ahead[:6])]
        if kind == "mixed":
            return [(t if rng.random() < 0.7 else (t + 5) % 39, i - 1) for i, t in enumerate(ahead[:6])]
        tree, last = [], -1                                # a wrong sibling before every right one
        for t in ahead[:8]:
            tree.append(((t + 1) % 39, last))
            tree.append((t, last))
            last = len(tree) - 1
        return tree
    assert m.generate_drafted(prompt, draft) == want
    if kind in ("right", "branches"):
        assert len(calls) <= -(-len(want) // 6) + 1
    if kind in ("none", "wrong"):
        assert len(calls) == len(want) - 1
    assert m.generate_drafted(prompt, draft, max_new_tokens=4) == want[:4]
    end = want[5]
    assert m.generate_drafted(prompt, draft, end_id=end) == m.generate(prompt, greedy=True, end_id=end)


def test_refusals():
    m = model()
    with pytest.raises(ValueError):
        m.generate_drafted([], lambda t: [])
    with pytest.raises(ValueError):
        m.generate_drafted([1, 2], lambda t: [(3, 0)])
    gqa = GroupedQueryAttention(32, 8, 4, 2, 1, dropout_rate=0.1, dtype=torch.float32, softcap=2.0)
    with pytest.raises(ValueError):
        gqa.forward(torch.zeros(8, 32), 1, 8)
