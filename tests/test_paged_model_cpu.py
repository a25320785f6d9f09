"""Generation over paged caches, and drawn text from drafted tokens (CPU restatements)."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.models.model import Cupa_ver4
from create_llm_by_cupy_b200.ops.drafts import target_probs

CFG = dict(layer_num=2, time_size=48, hidden_size=32, vocab_size=40, kv_head=2, q_head=4, ffn_size=48, padding_id=39, seed=3, init_std=0.3,
           dtype="fp32")
PROMPTS = [[3, 17, 8], [5] * 33, [1, 2, 4, 6, 9, 30, 31]]


def model(**kw):
    return Cupa_ver4({**CFG, **kw}, device="cpu")


@pytest.mark.parametrize("kw", [{}, dict(attn_softcap=2.0), dict(attn_distance_bias=True)])
@pytest.mark.parametrize("prefix", [0, 5])
def test_a_batch_is_its_sequences(kw, prefix):
    m = model(**kw)
    for limit in (None, 9):
        want = [m.generate(p, greedy=True, max_new_tokens=limit, prefix=prefix) for p in PROMPTS]
        assert m.generate_batch(PROMPTS, greedy=True, max_new_tokens=limit, page=32, prefix=prefix) == want
    end = want[0][4]
    want = [m.generate(p, start_id=7, end_id=end, greedy=True, prefix=prefix) for p in PROMPTS]
    assert m.generate_batch(PROMPTS, start_id=7, end_id=end, greedy=True, page=32, prefix=prefix) == want


@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_eight_bit_caches(cache):
    """The chosen token has the largest logit of the full sequence, or one near it: the cache is off by half a step, 0.4 % (int8) or 6 %
    (e4m3) of its rows; a tenth of the largest logit holds both."""
    m = model()
    for p, out in zip(PROMPTS, m.generate_batch(PROMPTS, greedy=True, max_new_tokens=10, cache=cache, page=32)):
        assert len(out) == 10
        logits = m.logits(torch.tensor([p + out]))[0, :, :39]
        for i, t in enumerate(out):
            row = logits[len(p) + i - 1]
            assert float(row.max() - row[t]) <= 0.1 * float(row.abs().max())


def test_drawn_batches():
    m = model()
    a = m.generate_batch(PROMPTS, seed=1, max_new_tokens=12)
    assert a == m.generate_batch(PROMPTS, seed=1, max_new_tokens=12) != m.generate_batch(PROMPTS, seed=2, max_new_tokens=12)
    assert all(len(x) == 12 and 39 not in x for x in a)
    assert m.generate_batch([], seed=1) == [] and m.generate_batch([[1]], max_new_tokens=0) == [[]]
    # almost no temperature, and almost no nucleus, is greedy decoding
    want = [m.generate(p, greedy=True, max_new_tokens=8) for p in PROMPTS]
    assert m.generate_batch(PROMPTS, temp=1e-6, penalty=1.0, max_new_tokens=8) == want
    assert m.generate_batch(PROMPTS, top=1e-9, penalty=1.0, max_new_tokens=8) == want
    with pytest.raises(ValueError):
        m.generate_batch([[1], []])
    with pytest.raises(ValueError):
        m.generate_batch([[1]], cache="int4")
    with pytest.raises(ValueError):
        m.generate_batch([[1]], page=17)


def test_repetition_penalty_as_in_generate():
    """Greedy in all but name: with a nucleus of one token the penalised choices of a sequence are those of the batch."""
    m = model()
    want = [m.generate(p, top=1e-9, penalty=1.5, max_new_tokens=10) for p in PROMPTS]
    assert m.generate_batch(PROMPTS, top=1e-9, penalty=1.5, max_new_tokens=10) == want


@pytest.mark.parametrize("with_probs", [False, True])
def test_drafts_do_not_change_what_is_drawn(with_probs):
    """Pairs of drawn tokens behind a prompt, with drafts of two branches: counts against the target's probabilities. 1500 texts; a count's
    standard deviation is at most 19.4, of which five are allowed."""
    m = model(vocab_size=6, padding_id=-1, init_std=0.5)
    prompt, N, temp, top = [1, 2], 1500, 0.9, 0.95
    g = torch.Generator().manual_seed(0)
    q = torch.tensor([0.3, 0.3, 0.1, 0.1, 0.1, 0.1])

    def draft(tokens):
        a, b, c = (int(x) for x in torch.multinomial(q, 3, replacement=True, generator=g))
        pairs = [(a, -1), (b, -1), (c, 0)]
        return (pairs, q.expand(4, 6)) if with_probs else pairs

    p0 = target_probs(m.logits(torch.tensor([prompt]))[0, -1], temp, top)
    counts = torch.zeros(6, 6)
    for i in range(N):
        # the first token comes from the prefill, drafts begin behind it
        _, x, y = m.generate_drafted(prompt, draft, max_new_tokens=3, temp=temp, top=top, seed=i)
        counts[x, y] += 1
    want = torch.zeros(6, 6)
    for z in range(6):
        p1 = target_probs(m.logits(torch.tensor([prompt + [z]]))[0, -1], temp, top)
        for x in range(6):
            want[x] += float(p0[z] * p1[x]) * target_probs(m.logits(torch.tensor([prompt + [z, x]]))[0, -1], temp, top).float()
    assert float((counts - N * want).abs().max()) <= 97 and math.isclose(float(want.sum()), 1.0, rel_tol=1e-5)


def test_drawn_drafts_refusals():
    m = model()
    q = torch.full((2, 40), 1 / 40)
    with pytest.raises(ValueError):
        m.generate_drafted([1, 2], lambda t: ([(3, -1)], q))                 # greedy
    with pytest.raises(ValueError):
        m.generate_drafted([1, 2], lambda t: ([(3, -1)], q[:1]), temp=1.0)
    out = m.generate_drafted([1, 2], lambda t: ([(3, -1)], q), temp=1.0, seed=0)
    assert len(out) == 46 and out == m.generate_drafted([1, 2], lambda t: ([(3, -1)], q), temp=1.0, seed=0)
    assert m.generate_drafted([1, 2], lambda t: [(5, -1)], temp=0.0) == m.generate([1, 2], greedy=True)
