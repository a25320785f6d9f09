"""A model under prefixes and documents: its logits, and generation behind a prompt that sees itself whole (CPU restatements)."""
import pytest
import torch

from create_llm_by_cupy_b200.ops.masked_attn import span_mask
from tests.test_masked_model_cpu import model


@pytest.mark.parametrize("kw", [{}, dict(attn_softcap=2.0), dict(attn_distance_bias=True)])
def test_logits_are_those_of_the_loss(kw):
    g = torch.Generator().manual_seed(0)
    x, t = (torch.randint(0, 38, (2, 20), generator=g) for _ in range(2))
    docs = torch.tensor([[0] * 8 + [1] * 12, [0] * 20], dtype=torch.int32)
    prefix = torch.zeros(2, 20, dtype=torch.bool)
    prefix[0, 8:13] = prefix[1, :7] = True
    m = model(**kw)
    for x_pa in (None, torch.tensor([20, 20], dtype=torch.int32), span_mask(2, 20, "cpu", docs=docs, prefix=prefix)):
        loss = torch.nn.functional.cross_entropy(m.logits(x, x_pa=x_pa).reshape(40, -1), t.reshape(-1))
        assert abs(float(loss) - float(m.predict(x, t, x_pa))) < 1e-5
    whole = m.logits(x, x_pa=span_mask(2, 20, "cpu", docs=docs, prefix=prefix))
    plain = m.logits(x)
    assert torch.allclose(whole[0, :8], plain[0, :8], atol=1e-5)                      # the first document has no prefix
    assert not torch.allclose(whole[1, 0], plain[1, 0], atol=1e-3)                    # the first token of a prefix sees the last


@pytest.mark.parametrize("kw", [{}, dict(attn_softcap=2.0), dict(attn_distance_bias=True)])
def test_generation_behind_a_prefix(kw):
    """Every chosen token is the one that the full sequence's logits say, the prompt's start seeing itself whole."""
    m = model(**kw)
    prompt, prefix = [3, 17, 8, 25, 9, 30], 5
    out = m.generate(prompt, greedy=True, max_new_tokens=10, prefix=prefix)
    for i, tok in enumerate(out):
        n = len(prompt) + i
        flags = (torch.arange(n) < prefix)[None]
        logits = m.logits(torch.tensor([prompt + out[:i]]), x_pa=span_mask(1, n, "cpu", prefix=flags))[0, -1]
        logits[39] = -1e30                                 # (padding is never chosen)
        assert int(logits.argmax()) == tok
    if not kw:                                             # (a prefix need not change the choices; of this model it does)
        assert out != m.generate(prompt, greedy=True, max_new_tokens=10)
    draft = [[(t, i - 1) for i, t in enumerate(out[j:j + 4])] for j in range(len(out) + 1)]
    assert m.generate_drafted(prompt, lambda toks: draft[len(toks) - len(prompt)], max_new_tokens=10, prefix=prefix) == out
