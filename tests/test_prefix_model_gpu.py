"""A model under prefixes on the kernels: logits, and generation behind a prompt that sees itself whole."""
import pytest
import torch

from create_llm_by_cupy_b200.models.model import Cupa_ver4
from create_llm_by_cupy_b200.ops import native
from create_llm_by_cupy_b200.ops.masked_attn import span_mask
from tests.test_masked_model_gpu import cfg

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [{}, dict(attn_softcap=20.0), dict(attn_distance_bias=True)])
def test_generation_behind_a_prefix(D, kw):
    """Every chosen token has the largest logit of the full sequence under the prefix, or one that bf16 cannot tell from it."""
    m = Cupa_ver4(cfg(D, **kw), device=DEV)
    prompt, prefix = list(range(5, 205)), 170
    out = m.generate(prompt, greedy=True, max_new_tokens=12, prefix=prefix)
    drafted = m.generate_drafted(prompt, lambda toks: [(t, i - 1) for i, t in enumerate(out[len(toks) - len(prompt):][:5])],
                                 max_new_tokens=12, prefix=prefix)
    for toks in (out, drafted):
        n = len(prompt) + len(toks)
        flags = (torch.arange(n, device=DEV) < prefix)[None]
        x = torch.tensor([prompt + toks], device=DEV)
        logits = m.logits(x, x_pa=span_mask(1, n, DEV, prefix=flags))[0]
        plain = m.logits(x)[0]
        assert float((logits[:prefix - 1] - plain[:prefix - 1]).norm()) > 0.05 * float(plain[:prefix - 1].norm())
        logits[:, 511] = -1e30
        for i, tok in enumerate(toks):
            row = logits[len(prompt) + i - 1]
            assert float(row.max() - row[tok]) <= 2e-2 * float(row.abs()[:511].max())
    assert native.read_status() == (0, 0)


def test_logits_are_those_of_the_loss():
    m = Cupa_ver4(cfg(128), device=DEV)
    g = torch.Generator().manual_seed(0)
    x, t = (torch.randint(0, 500, (2, 300), generator=g).to(DEV) for _ in range(2))
    docs = (torch.arange(300, device=DEV) // 130).to(torch.int32).expand(2, 300).contiguous()
    for x_pa in (None, torch.tensor([300, 300], dtype=torch.int32, device=DEV), span_mask(2, 300, DEV, docs=docs)):
        loss = torch.nn.functional.cross_entropy(m.logits(x, x_pa=x_pa).reshape(600, -1), t.reshape(-1))
        assert abs(float(loss) - float(m.predict(x, t, x_pa))) < 5e-3
    assert native.read_status() == (0, 0)
