"""What generation of batches and from drafts takes beside ``generate``: temperatures, nuclei and proposals of any kind (CPU forms)."""
import numpy as np
import pytest
import torch

from create_llm_by_cupy_b200.models import model as M

from .test_paged_model_cpu import PROMPTS, model


@pytest.mark.parametrize("top", [0.0, -1.0, 0])
def test_a_nucleus_of_nothing_is_the_likeliest_token(top):
    m = model()
    want = [m.generate(p, top=top, penalty=1.3, max_new_tokens=7) for p in PROMPTS]
    assert m.generate_batch(PROMPTS, top=top, penalty=1.3, max_new_tokens=7) == want
    greedy = [m.generate(p, greedy=True, max_new_tokens=7) for p in PROMPTS]
    assert m.generate_batch(PROMPTS, greedy=True, top=top, max_new_tokens=7) == greedy


@pytest.mark.parametrize("temp", [0.0, -1.0, 1e-9])
def test_temperatures_of_nothing(temp):
    m = model()
    want = [m.generate(p, temp=temp, penalty=1.3, max_new_tokens=7) for p in PROMPTS]
    assert m.generate_batch(PROMPTS, temp=temp, penalty=1.3, max_new_tokens=7) == want


def test_very_high_temperatures():
    """All tokens but the padding are alike: 322 draws of 39 tokens miss one with a probability of at most 39 (38 / 39)^322 = 0.009 (the
    seed is fixed)."""
    m = model()
    for temp in (1e6, 1e7, 1e30, float("inf")):
        outs = m.generate_batch([[1, 2]] * 7, temp=temp, top=1.0, penalty=1.0, seed=5)
        assert all(len(x) == 46 and 39 not in x for x in outs) and len({t for x in outs for t in x}) == 39


def test_numbers_are_checked_first(monkeypatch):
    m = model()
    monkeypatch.setattr(type(m), "_rows_mask", lambda *a, **k: pytest.fail("a pass was begun"))
    for kw in (dict(temp=float("nan")), dict(top=float("nan"))):
        with pytest.raises(ValueError):
            m.generate_batch(PROMPTS, **kw)


@pytest.mark.parametrize("temp,top", [(1e-9, 0.9), (-1.0, 0.9), (1e-7, 1.0), (0.0, 0.5), (1.0, 0.0), (0.7, -2.0)])
def test_drafts_with_nothing_to_draw_are_greedy(temp, top):
    m = model()
    want = m.generate([1, 2], greedy=True)
    assert m.generate_drafted([1, 2], lambda t: [(want[len(t) - 2], -1), (5, 0)], temp=temp, top=top) == want


def test_drafts_at_very_high_temperatures_and_numbers_that_are_none(monkeypatch):
    m = model()
    assert len(m.generate_drafted([1, 2], lambda t: [(5, -1)], temp=1e9, seed=0)) == 46
    monkeypatch.setattr(type(m), "_rows_mask", lambda *a, **k: pytest.fail("a pass was begun"))
    for kw in (dict(temp=float("nan")), dict(temp=1.0, top=float("nan"))):
        with pytest.raises(ValueError):
            m.generate_drafted([1, 2], lambda t: [], **kw)


@pytest.mark.parametrize("pack", [np.array, torch.tensor, tuple, list])
@pytest.mark.parametrize("outer", [tuple, list])
@pytest.mark.parametrize("temp", [None, 1e-6])
def test_two_proposals_in_any_container(pack, outer, temp):
    """Two pairs that are arrays, in a tuple, are two proposals, not proposals and their probabilities."""
    m = model()
    want, calls = m.generate([1, 2], greedy=True), []

    def draft(tokens):
        calls.append(len(tokens))
        ahead = (want + [0, 0])[len(tokens) - 2:][:2]
        return outer([pack([ahead[0], -1]), pack([ahead[1], 0])])

    assert m.generate_drafted([1, 2], draft, temp=temp, top=1.0) == want and len(calls) <= 16


def test_probabilities_that_are_no_rows_are_refused():
    m = model()
    for q in (torch.full((40,), 1 / 40), torch.full((1, 2, 40), 1 / 40), torch.tensor(1.0)):
        with pytest.raises(ValueError):
            m.generate_drafted([1, 2], lambda t: ([(3, -1)], q), temp=1.0)


def test_models_that_the_kernels_do_not_take_are_refused_first(monkeypatch):
    """Before any pool is made: head dimensions other than 64 and 128 on CUDA, vocabularies that the verification has no room for."""
    monkeypatch.setattr(M, "paged_cache", lambda *a, **k: pytest.fail("a pool was made"))
    m = model()
    m.device = torch.device("cuda")                          # head dimension 8
    with pytest.raises(ValueError, match="head dimension"):
        m.generate_batch(PROMPTS)
    m = model()
    m.vocab_size = 8 * 376 * 128 + 1
    for greedy in (False, True):
        with pytest.raises(ValueError, match="vocabularies"):
            m.generate_batch(PROMPTS, greedy=greedy)
    monkeypatch.setattr(type(m), "_rows_mask", lambda *a, **k: pytest.fail("a pass was begun"))
    with pytest.raises(ValueError, match="vocabularies"):
        m.generate_drafted([1, 2], lambda t: [], temp=1.0)
