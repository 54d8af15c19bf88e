"""speculative_generate when pages are scarce, and with prompts on the GPU."""

import importlib

import numpy as np
import pytest
import torch

from test_gpu_speculative import small_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(jsx, ref, cuda):
    return small_model(jsx, ref)[0]


def prompts(B, S):
    return np.random.default_rng(11).integers(0, 1000, (B, S))


KW = dict(max_new_tokens=40, temperature=0.9, page_tokens=16, draft_tokens=0)


def ending(model, jsx, **kw):
    """Prompts of 16 tokens, an EOS id that ends the first sequence within its second page and
    never comes up in the second, and the text (which depends on the number of drafts: so do the
    uniforms)."""
    p, kw = prompts(2, 16), dict(KW, **kw)
    for seed in range(20):
        text = jsx.speculative_generate(model, p, seed=seed, **kw)
        for at in range(2, 12):
            eos = int(text[0, 16 + at])
            if eos not in text[0, 16:16 + at] and eos not in text[1, 16:]:
                return p, seed, eos, jsx.speculative_generate(model, p, seed=seed, eos_token_id=eos, **kw)
    raise AssertionError("no such text")


def test_a_finished_sequence_gives_its_pages_back(jsx, model):
    """56 tokens of one sequence need 4 pages of 16; the other one's two must be free by then."""
    p, seed, eos, want = ending(model, jsx)
    got = jsx.speculative_generate(model, p, seed=seed, eos_token_id=eos, num_pages=4, **KW)
    assert torch.equal(got, want)
    # the same with drafts, all of them refused
    kw = dict(draft_tokens=3, draft=lambda history, n: [(history[-1] + 1) % 1000] * n)
    p, seed, eos, want = ending(model, jsx, **kw)
    assert torch.equal(jsx.speculative_generate(model, p, seed=seed, eos_token_id=eos, num_pages=5, **dict(KW, **kw)), want)


def test_cache_of_finished_sequences_is_empty(jsx, model, monkeypatch):
    """After a sequence's end the steps hold no page for it."""
    sp = importlib.import_module("e2e-jaxscale_b200.speculative")
    p, seed, eos, _ = ending(model, jsx)
    seen, real = [], sp.step
    monkeypatch.setattr(sp, "step", lambda m, st, *a: seen.append((st.count.tolist(), st.cache.held.tolist())) or real(m, st, *a))
    jsx.speculative_generate(model, p, seed=seed, eos_token_id=eos, **KW)
    assert any(count[0] == 0 for count, _ in seen)
    assert all(held[0] == 0 for count, held in seen if count[0] == 0)


def test_the_text_survives_a_pool_that_runs_out(jsx, model):
    p = prompts(2, 16)
    whole = jsx.speculative_generate(model, p, seed=3, **KW)
    with pytest.raises(RuntimeError, match="pages missing") as e:
        jsx.speculative_generate(model, p, seed=3, num_pages=5, **KW)
    text = e.value.tokens                          # 5 pages: 32 tokens of both are stored
    assert text.shape == whole.shape and text.dtype == torch.int32
    assert torch.equal(text[:, :33], whole[:, :33]) and (text[:, 33:] == -1).all()
    with pytest.raises(RuntimeError) as e:         # not even the prompt fits
        jsx.speculative_generate(model, p, num_pages=1, **KW)
    assert torch.equal(e.value.tokens[:, :16], torch.as_tensor(p, dtype=torch.int32)) and (e.value.tokens[:, 16:] == -1).all()


def test_prompts_on_the_gpu(jsx, model):
    p = torch.from_numpy(prompts(2, 9)).int()
    a = jsx.speculative_generate(model, p, max_new_tokens=6)
    b = jsx.speculative_generate(model, p.cuda(), max_new_tokens=6)
    assert not b.is_cuda and torch.equal(a, b)
