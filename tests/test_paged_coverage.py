"""The attention over 4-bit pages and the verification where their other tests are thin: head_dim 64
at long contexts, a windowed prompt in the 128-row kernel, and verifications whose every sequence
is compared.  Bounds of the attention as in test_gpu_kv4.py."""

import importlib

import numpy as np
import pytest
import torch

from test_gpu_kv4 import attn_case
from test_gpu_speculative import small_model
from test_gpu_verify import make

pytestmark = pytest.mark.gpu

R = importlib.import_module("oracle.paged_ref")


@pytest.mark.parametrize("B,T,nq,nkv,pt,L,window,sinks", [
    (1, 1, 32, 2, 64, 20001, 0, 0), (3, 5, 32, 2, 32, 6000, 0, 0), (2, 16, 16, 1, 64, 9001, 0, 0), (40, 1, 8, 1, 16, 1500, 0, 0),
    (4, 1, 8, 1, 32, 12001, 4096, 4), (1, 64, 12, 4, 128, 2000, 300, 3)])
def test_attention_head_dim_64_long(jsx, cuda, B, T, nq, nkv, pt, L, window, sinks):
    rng = np.random.default_rng(B * T + nq)
    positions = [L - T] + [int(x) for x in rng.integers(0, L - T, B - 1)]
    attn_case(jsx, rng, B, T, nq, nkv, 64, pt, positions, window=window, sinks=sinks)


def test_a_windowed_prompt_in_one_call(jsx, ref, cuda, monkeypatch):
    """A windowed prefill's attention, all of a prompt's tokens in one call, against the same queries
    eight tokens at a time (the 16-row kernel: 2 heads x 8 tokens).  Each is within
    2^-8 |o| + 2^-9 V of the definition, so they are within twice that of each other."""
    model, rc = small_model(jsx, ref)
    sp = importlib.import_module("e2e-jaxscale_b200.speculative")
    K = jsx.kernels
    B, S, window, sinks, nq, nkv, hd = 3, 1100, 200, 3, 4, 2, 128
    calls, real = [], K.kv4_attn

    def spy(q, pool, table, positions, head_dim, ws, **kw):
        o = real(q, pool, table, positions, head_dim, ws, **kw)
        calls.append((q.clone(), pool, table, o.clone(), kw))
        return o
    prompt = torch.from_numpy(np.random.default_rng(5).integers(0, rc.vocab_size, (B, S))).int().cuda()
    st = sp.DraftedState(model, B, 1, S + 8, page_tokens=32)
    monkeypatch.setattr(K, "kv4_attn", spy)
    logits = sp.prefill(model, st, prompt, window, sinks)
    monkeypatch.undo()
    assert torch.isfinite(logits.float()).all() and len(calls) == 2
    for q, pool, table, o, kw in calls:
        assert kw["tokens_per_seq"] == S and kw["window"] == window and kw["sinks"] == sinks
        T = 8
        ws = K.kv4_attn_workspace(B, T, nq, nkv, hd, q.device)
        want = torch.zeros_like(o).view(B, S, -1)
        for at in range(0, S, T):
            n = min(T, S - at)
            part = q.view(B, S, -1)[:, at:at + n].reshape(B * n, -1).contiguous()
            pos = torch.full((B,), at, dtype=torch.int32, device="cuda")
            want[:, at:at + n] = real(part, pool, table, pos, hd, ws, scale=kw["scale"], tokens_per_seq=n, window=window, sinks=sinks).view(B, n, -1)
        _, v = R.unpack_pool(pool.cpu().numpy(), hd)
        bound = 2 * (2.0 ** -8 * want.float().abs() + 2.0 ** -9 * float(np.abs(v).max()))
        assert ((o.view(B, S, -1).float() - want.float()).abs() <= bound).all()
    assert K.device_error() == 0


@pytest.mark.parametrize("B,T,V,f32,probs,temperature,share", [
    (24, 2, 9001, False, True, 1.0, 0.9), (24, 0, 9001, True, False, 0.7, 0.9), (60, 3, 61, False, True, 1.3, 1.0), (60, 2, 300, True, False, 1.0, 0.99),
    (12, 1, 151552, False, False, 1.0, 0.5), (16, 4, 32003, False, False, 0.0, 1.0)])
def test_every_sequence_of_a_verification(jsx, cuda, B, T, V, f32, probs, temperature, share):
    """Most sequences are clear of a boundary by 1e-6 of the total, and equal the oracle's.  (Of V entries
    with mass, a share of about 2e-6 V of the uniforms is not.)  The others accept one draft more or
    less at most, or draw an entry whose running sum is that near."""
    rng = np.random.default_rng(B + V)
    x, ids, u, q = make(rng, B, T, V, f32, probs=probs, temperature=temperature)
    acc, tok, _ = jsx.kernels.verify_drafts(x, ids, u, jsx.kernels.verify_workspace(B, T, V, x.device), draft_probs=q, temperature=temperature)
    f = lambda t: None if t is None else t.float().cpu().numpy()  # noqa: E731
    wa, wt, _, margin = R.verify(f(x), ids.cpu().numpy(), f(u), f(q), None, temperature)
    acc, tok, clear = acc.cpu().numpy(), tok.cpu().numpy(), margin > 1e-6
    assert clear.mean() >= share
    assert np.array_equal(acc[clear], wa[clear]) and np.array_equal(tok[clear], wt[clear])
    for b in np.nonzero(~clear)[0]:
        if acc[b] != wa[b]:
            continue                                # an acceptance at its boundary: the rest follows from another row
        n = acc[b]
        assert np.array_equal(tok[b, :n], wt[b, :n]) and (tok[b, n + 1:] == -1).all()
        w = R._weights(f(x)[b, n], np.float32(1) / np.float32(temperature))
        if n < T:                                   # what is left after a refusal
            if q is None:
                w[ids[b, n].item()] = 0
            else:
                d = w / w.sum() - f(q)[b, n].astype(np.float64)
                w = np.floor(np.where(d > 0, d, 0) * 2.0 ** 40)
        run = np.cumsum(w) / w.sum()
        at = float(u[b, T])
        lo, hi = np.searchsorted(run, at - 2e-6), np.searchsorted(run, at + 2e-6)
        assert lo <= tok[b, n] <= hi and w[tok[b, n]] > 0
