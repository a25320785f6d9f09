"""The model whose scores lose a slope times the distance in place of a rotation: training, scoring and generation (CPU restatements)."""
import math

import pytest
import torch

from create_llm_by_cupy_b200.models.layers import GroupedQueryAttention
from create_llm_by_cupy_b200.ops.masked_attn import span_mask
from tests.test_masked_model_cpu import grads_of, model


def test_the_layer_is_the_definition():
    """No rotation, slope[head] * distance taken from the scores, documents apart."""
    g = torch.Generator().manual_seed(0)
    H, QH, KVH, T = 24, 6, 2, 9
    D, R = H // QH, QH // KVH
    gqa = GroupedQueryAttention(H, 16, QH, KVH, 1, dtype=torch.float32, generator=g, distance_bias=True)
    x = torch.randn(2 * T, H, generator=g)
    docs = torch.tensor([[0] * T, [0] * 4 + [1] * 5], dtype=torch.int32)
    got = gqa.forward(x, 2, T, span_mask(2, T, "cpu", docs=docs), train_flg=False)
    k, q, v = (x.double() @ gqa.params[0].double()).view(2, T, -1).split([KVH * D, H, KVH * D], 2)
    t = torch.arange(T)
    o = torch.zeros(2, T, QH, D, dtype=torch.float64)
    for h in range(QH):
        qh, kh, vh = q.view(2, T, QH, D)[:, :, h], k.view(2, T, KVH, D)[:, :, h // R], v.view(2, T, KVH, D)[:, :, h // R]
        s = qh @ kh.transpose(1, 2) / math.sqrt(D) - 2.0 ** (-8 * (h + 1) / QH) * (t[:, None] - t[None])
        s = s.masked_fill((t[None] > t[:, None]) | (docs[:, :, None] != docs[:, None]), -math.inf)
        o[:, :, h] = torch.softmax(s, -1) @ vh
    assert torch.allclose(got.double(), o.reshape(2 * T, H) @ gqa.params[1].double(), atol=1e-5)


@pytest.mark.parametrize("keep", [True, False])
def test_backward_by_differences(keep):
    """d loss along the gradient, from differences of losses; also with the recompute switches."""
    g = torch.Generator().manual_seed(1)
    x, t = (torch.randint(0, 38, (2, 12), generator=g) for _ in range(2))
    n = torch.tensor([12, 7], dtype=torch.int32)
    m = model(attn_distance_bias=True, gqa_cache_out_value=keep, gqa_cache_kqv=keep)
    _, grads = grads_of(m, x, t, n)
    for i in (0, 1, 4):                                    # K | Q | V, the output projection, a norm
        d = grads[i] / grads[i].norm()
        slope = []
        for eps in (2e-2, 1e-2):                           # two step widths: what a difference is off by falls with their square
            f = []
            for s in (eps, -eps):
                m.params[i].add_(d, alpha=s)
                f.append(float(m.forward(x, t, n, train_flg=False)))
                m.params[i].add_(d, alpha=-s)
            slope.append((f[0] - f[1]) / (2 * eps))
        assert abs((4 * slope[1] - slope[0]) / 3 - float(grads[i].norm())) < 2e-2 * float(grads[i].norm()) + 1e-4


def test_generation_reads_the_same_attention():
    m = model(attn_distance_bias=True, padding_id=-1)
    prompt = [3, 17, 8]
    out = m.generate(prompt, greedy=True, max_new_tokens=10)
    for i, tok in enumerate(out):
        assert int(m.logits(torch.tensor([prompt + out[:i]]))[0, -1].argmax()) == tok
    m = model(attn_distance_bias=True)
    want = m.generate(prompt, greedy=True)
    drafts = [[(t, i - 1) for i, t in enumerate(want[j:j + 5])] for j in range(len(want) + 1)]
    assert m.generate_drafted(prompt, lambda toks: drafts[len(toks) - len(prompt)]) == want


def test_capped_and_biased_is_refused():
    with pytest.raises(ValueError):
        model(attn_distance_bias=True, attn_softcap=3.0)
