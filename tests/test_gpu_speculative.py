"""Drafted generation over the paged 4-bit cache (speculative.py, layers/paged_cache.py)."""

import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def small_model(jsx, ref, seed=0, layers=2):
    rc = ref.GLMConfig(hidden_size=256, num_hidden_layers=layers, num_attention_heads=4, num_key_value_heads=2,
                       head_dim=128, intermediate_size=384, vocab_size=1000)
    model = jsx.GLM4ForCausalLM(jsx.ModelConfig(hidden_size=256, num_hidden_layers=layers, num_attention_heads=4,
                                                num_key_value_heads=2, head_dim=128, intermediate_size=384,
                                                vocab_size=1000), jsx.create_mesh(1))
    model.load_state(ref.init_params(rc, seed=seed))
    return model, rc


def test_pages_answer_as_the_static_cache_of_their_values(jsx, cuda):
    """Attention over the pages against jsx_attn_decode over the same values read back as bf16.
    Both round their output to bf16 and their weights to 8 (bf16) or 11 (f16) bits, so outputs
    differ by at most 2^-8 |o| + (2^-9 + 2^-11) V, V the largest |v|."""
    K = jsx.kernels
    B, nq, nkv, hd, L = 3, 32, 2, 128, 700
    cache = jsx.PagedKV4Cache(1, B, L, nkv, hd, page_tokens=32)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    assert int(cache.reserve(zero, torch.full_like(zero, L))) == 0
    g = torch.Generator("cuda").manual_seed(1)
    k, v = (torch.randn(B, L, nkv, hd, generator=g, device="cuda").to(torch.bfloat16) for _ in "kv")
    cache.append(0, k, v, zero, tokens_per_seq=L)
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    cache.read(0, zero, kb, vb, tokens_per_seq=L)
    q = torch.randn(B, nq * hd, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.tensor([699, 0, 350], dtype=torch.int32, device="cuda")
    a = cache.attend(0, q, pos, hd ** -0.5)
    b = torch.empty_like(q)
    K.attn_decode(q, kb, vb, b, pos, hd ** -0.5, K.attn_workspace(B, nq, nkv, hd, L, q.device))
    bound = 2.0 ** -8 * b.float().abs() + (2.0 ** -9 + 2.0 ** -11) * vb.float().abs().max()
    assert ((a.float() - b.float()).abs() <= bound).all()


def test_cache_fork_write_release(jsx, cuda):
    """A fork reads its parent's rows, writes its own, and gives everything back."""
    B, L, hd = 3, 200, 64
    cache = jsx.PagedKV4Cache(2, B, L, 1, hd, page_tokens=16, num_pages=30)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    assert int(cache.reserve(i32(0, 0, 0), i32(100, 0, 0))) == 0
    rows = torch.randn(B, L, 1, hd, device="cuda").to(torch.bfloat16)
    for layer in range(2):
        cache.append(layer, rows, rows, i32(0, 0, 0), tokens_per_seq=100, n_tokens=i32(100, 0, 0))
    cache.fork(i32(0, 0, -1))
    assert cache.free_pages() == 23
    assert int(cache.reserve(i32(100, 100, 0), i32(101, 110, 0))) == 0
    assert cache.free_pages() == 23 - 2 + 1       # both write into page 6: both get a copy, and it is free again
    other = torch.randn(B, L, 1, hd, device="cuda").to(torch.bfloat16)
    cache.append(1, other, other, i32(100, 100, 0), tokens_per_seq=10, n_tokens=i32(1, 10, 0))
    out, out2 = torch.zeros_like(rows), torch.zeros_like(rows)
    cache.read(1, i32(0, 0, 0), out, out2, tokens_per_seq=110, n_tokens=i32(101, 110, 0))
    want = torch.zeros_like(rows)
    ref = importlib.import_module("oracle.paged_ref")
    stored = lambda t: torch.from_numpy(ref.stored(t.double().cpu().numpy())).to("cuda", torch.bfloat16)  # noqa: E731
    want[0, :100], want[1, :100] = stored(rows[0, :100]), stored(rows[0, :100])
    want[0, 100], want[1, 100:110] = stored(other[0, 100]), stored(other[1, 100:110])
    assert torch.equal(out, want) and torch.equal(out2, want)
    remap = cache.compact()
    assert int(cache.table.max()) < 9 and int((remap >= 0).sum()) == 8
    out.zero_()
    cache.read(1, i32(0, 0, 0), out, out2, tokens_per_seq=110, n_tokens=i32(101, 110, 0))
    assert torch.equal(out, want)
    assert int(cache.reserve(i32(0, 0, 0), i32(200, 200, 200))) > 0   # 39 pages of 30: nothing happens
    assert cache.free_pages() == 22
    cache.reserve(i32(0, 0, 0), i32(0, 0, 0))
    assert cache.free_pages() == 30


@pytest.mark.parametrize("window,sinks", [(0, 0), (16, 2)])
def test_greedy_drafts_do_not_change_the_text(jsx, ref, cuda, window, sinks):
    """Temperature 0: with drafts (good ones, bad ones, none) and without them the same tokens."""
    model, rc = small_model(jsx, ref)
    rng = np.random.default_rng(3)
    prompt = rng.integers(0, rc.vocab_size, (3, 37))
    prompt[:, 20:] = prompt[:, 3:20]               # repeats itself, so that lookup finds something
    kw = dict(max_new_tokens=24, window=window, sinks=sinks, page_tokens=16)
    plain = jsx.speculative_generate(model, prompt, draft_tokens=0, **kw)
    assert plain.shape == (3, 61)
    stats = {}
    looked = jsx.speculative_generate(model, prompt, draft_tokens=4, stats=stats, **kw)
    truth = [r.tolist() for r in plain]

    def oracle(history, count):                     # what will come, with a mistake now and then
        b = next(i for i in range(3) if truth[i][:len(history)] == history)
        t = truth[b][len(history):len(history) + count]
        return [(x + (len(history) + i) % 5 // 4) % 1000 for i, x in enumerate(t)]

    good = {}
    drafted = jsx.speculative_generate(model, prompt, draft_tokens=5, draft=oracle, stats=good, **kw)
    bad = jsx.speculative_generate(model, prompt, draft_tokens=3, draft=lambda h, n: [(h[-1] + 1) % 1000] * n, **kw)
    for other in (looked, drafted, bad):
        assert torch.equal(plain, other)
    assert good["accepted"] > 0.5 * good["drafted"] and good["steps"] < 24
    assert jsx.kernels.device_error() == 0


def test_first_logits_match_the_bf16_cache(jsx, ref, cuda):
    """The prompt's logits do not depend on the cache's bits: the same as the model's own forward."""
    model, rc = small_model(jsx, ref)
    from importlib import import_module
    sp = import_module("e2e-jaxscale_b200.speculative")
    prompt = torch.from_numpy(np.random.default_rng(5).integers(0, rc.vocab_size, (2, 40))).int().cuda()
    st = sp.DraftedState(model, 2, 1, 64, page_tokens=16)
    got = sp.prefill(model, st, prompt)
    want, _ = model(prompt, torch.arange(40, dtype=torch.int32).expand(2, 40))
    err = (got.float() - want[:, -1].float()).abs().max() / want[:, -1].float().abs().max()
    assert err < 2e-2


def test_sampling_ends_and_seeds(jsx, ref, cuda):
    model, rc = small_model(jsx, ref)
    prompt = np.random.default_rng(7).integers(0, rc.vocab_size, (2, 9))
    a = jsx.speculative_generate(model, prompt, max_new_tokens=12, temperature=0.9, seed=1)
    b = jsx.speculative_generate(model, prompt, max_new_tokens=12, temperature=0.9, seed=1)
    c = jsx.speculative_generate(model, prompt, max_new_tokens=12, temperature=0.9, seed=2)
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert ((a >= 0) & (a < 1000)).all()
    eos = int(a[0, 9 + 4])
    d = jsx.speculative_generate(model, prompt, max_new_tokens=12, temperature=0.9, seed=1, eos_token_id=eos)
    stop = a[0, 9:].tolist().index(eos)
    assert d[0, 9 + stop:].eq(eos).all()
    with pytest.raises(RuntimeError):
        jsx.speculative_generate(model, prompt, max_new_tokens=12, num_pages=1, page_tokens=16)


def test_prompt_lookup(jsx):
    f = importlib.import_module("e2e-jaxscale_b200.speculative").prompt_lookup
    assert f([1, 2, 3, 4, 1, 2, 3], 2) == [4, 1]
    assert f([5, 6, 5, 7, 5], 3) == [7, 5]
    assert f([1, 2, 3], 4) == [] and f([1], 4) == [] and f([9, 9], 4) == [9]
