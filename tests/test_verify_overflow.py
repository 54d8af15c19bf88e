"""Verification where a row's largest logit is finite but its quotient by the temperature is not: a
row that a mask left empty by the type's lowest value, logits near the type's largest, temperatures
near zero.  Against softmax in 64 bits, where nothing overflows.

The quotients of two different logits of such a row differ by more than 2^100, so a probability is
0 or 1 / (number of maxima), and both are exact in fp32 up to the division's rounding: 2^-23."""

import importlib

import numpy as np
import pytest
import torch

R = importlib.import_module("oracle.paged_ref")
BF = torch.bfloat16


def softmax64(x, temperature):
    x = x.astype(np.float64) / np.float64(np.float32(temperature))
    w = np.exp(x - x.max(-1, keepdims=True))
    return w / w.sum(-1, keepdims=True)


def rows(f32, V):
    """[4, 2, V] logits, and the temperature that makes their quotients overflow."""
    low, top = (torch.finfo(torch.float32 if f32 else BF).min, torch.finfo(torch.float32 if f32 else BF).max)
    x = torch.randn(4, 2, V, generator=torch.Generator().manual_seed(V))
    x[0, 0] = low                                   # nothing left by the mask
    x[1, 0] = low
    x[1, 0, [3, V // 2, V - 1]] = low / 2           # three left, all very low
    x[2, 0, [0, V - 2]] = top                       # two maxima among ordinary logits
    x[3, 0, 5] = float("-inf")
    x[3, 0, 7] = top                                # one, beside a banned one
    x[3, 0, 9] = float("nan")
    return x if f32 else x.to(BF)


def ordinary(f32, V):
    x = torch.randn(4, 2, V, generator=torch.Generator().manual_seed(V)) * 3
    x[:, 0, V // 3], x[:, 0, V // 2] = 40.0, 40.0
    return x if f32 else x.to(BF)


def test_the_oracle_is_softmax():
    for x, t in ((rows(True, 100), 0.5), (rows(False, 100), 0.9), (ordinary(True, 100), 1e-37)):
        x = x.double().numpy()
        want = softmax64(np.where(np.isnan(x), -np.inf, x), t)
        for b in range(4):
            w = R._weights(x[b, 0].astype(np.float32), np.float32(1) / np.float32(t))
            assert w is not None and np.allclose(w / w.sum(), want[b, 0], atol=1e-11)


@pytest.mark.gpu
@pytest.mark.parametrize("f32,V,make,temperature", [(True, 64, rows, 0.5), (False, 301, rows, 0.7), (False, 70001, rows, 0.99),
                                                    (True, 4099, ordinary, 1e-37), (False, 1000, ordinary, 2e-38)])
@pytest.mark.parametrize("probs", [False, True])
def test_quotients_that_overflow(jsx, cuda, f32, V, make, temperature, probs):
    x = make(f32, V)
    x64 = x.double().numpy()
    p = softmax64(np.where(np.isnan(x64), -np.inf, x64), temperature)[:, 0]
    for b in range(4):                              # (the inputs are what this file says)
        assert set(np.unique(p[b])) <= {0.0, p[b].max()}
    first = [int(np.argmax(r)) for r in p]
    last = [int(V - 1 - np.argmax(r[::-1])) for r in p]
    dev = lambda t, d=torch.int32: torch.as_tensor(t).to("cuda", d)  # noqa: E731
    q = torch.full((4, 1, V), 1.0 / V, device="cuda") if probs else None
    ws = jsx.kernels.verify_workspace(4, 1, V, "cuda")
    # the first maximum as a draft: p(x) / q(x), q(x) = 1 for a certain draft
    u = torch.zeros(4, 2, device="cuda")
    acc, tok, pr = jsx.kernels.verify_drafts(x.cuda(), dev(first)[:, None], u, ws, draft_probs=q, temperature=temperature)
    want = np.minimum(1, np.array([p[b, first[b]] for b in range(4)]) / (float(np.float32(1 / V)) if probs else 1.0))
    assert np.allclose(pr[:, 0].cpu().numpy(), want, rtol=2.0 ** -22)
    assert acc.tolist() == [1] * 4 and tok[:, 0].tolist() == first
    # without drafts: the first and the last of the maxima by u
    none = torch.zeros(4, 0, dtype=torch.int32, device="cuda")
    for uniform, at in ((0.0, first), (1 - 2.0 ** -24, last)):
        _, tok, _ = jsx.kernels.verify_drafts(x[:, :1].cuda(), none, torch.full((4, 1), uniform, device="cuda"), ws, temperature=temperature)
        assert tok[:, 0].tolist() == at
    # a draft without mass is refused, and the token comes from the maxima
    bad = [int(np.argmin(r)) for r in p]
    _, tok, pr = jsx.kernels.verify_drafts(x.cuda(), dev(bad)[:, None], u, ws, draft_probs=q, temperature=temperature)
    for b in range(4):
        if p[b, bad[b]] == 0:
            assert pr[b, 0] == 0 and int(tok[b, 0]) == first[b]


@pytest.mark.gpu
def test_rows_without_a_finite_maximum_still_have_no_token(jsx, cuda):
    x = torch.zeros(3, 1, 50, device="cuda")
    x[0], x[1], x[2, 0, 4] = float("-inf"), float("nan"), float("inf")
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    for t in (0.5, 1e-37, 1.0):
        _, tok, _ = jsx.kernels.verify_drafts(x, none, torch.full((3, 1), 0.5, device="cuda"), jsx.kernels.verify_workspace(3, 0, 50, "cuda"), temperature=t)
        assert tok[:, 0].tolist() == [-1] * 3
