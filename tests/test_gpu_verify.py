"""Verification of drafted tokens (jsx_verify_drafts) against the 64-bit oracle
(oracle/paged_ref.py verify): accepted counts and tokens are equal wherever the oracle's own
decisions are not within 1e-6 of a boundary; acceptance probabilities within 2e-6 relative
(fp32 exponentials of 2^-22 each, V 2^-41 of floors)."""

import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

R = importlib.import_module("oracle.paged_ref")


def make(rng, B, T, V, f32=False, spread=2.5, probs=True, temperature=1.0):
    x = torch.from_numpy((rng.standard_normal((B, T + 1, V)) * spread).astype(np.float32)).cuda()
    x = x if f32 else x.to(torch.bfloat16)
    near = x[:, :T].float() + 0.5 * torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32)).cuda()
    q = torch.softmax(near / (temperature or 1.0), -1)
    if T and probs:
        ids = torch.multinomial(q.view(B * T, V), 1, generator=torch.Generator("cuda").manual_seed(int(rng.integers(1 << 30)))).view(B, T)
    else:
        ids = x[:, :T].float().argmax(-1)
        ids = torch.where(torch.from_numpy(rng.random((B, T)) < 0.3).cuda(), (ids + 1) % V, ids)
    u = torch.from_numpy(rng.random((B, T + 1), dtype=np.float32)).cuda()
    return x, ids.to(torch.int32), u, q.contiguous() if probs else None


def check(jsx, x, ids, u, q=None, n_draft=None, temperature=1.0):
    B, T1, V = x.shape
    nd = None if n_draft is None else torch.as_tensor(n_draft, dtype=torch.int32, device="cuda")
    ws = jsx.kernels.verify_workspace(B, T1 - 1, V, x.device)
    acc, tok, pr = jsx.kernels.verify_drafts(x, ids, u, ws, draft_probs=q, n_draft=nd, temperature=temperature)
    f = lambda t: None if t is None else t.float().cpu().numpy()  # noqa: E731
    wa, wt, wp, margin = R.verify(f(x), ids.cpu().numpy(), f(u), f(q), n_draft, temperature)
    clear = margin > 1e-6
    assert np.array_equal(acc.cpu().numpy()[clear], wa[clear])
    assert np.array_equal(tok.cpu().numpy()[clear], wt[clear])
    assert np.allclose(pr.cpu().numpy(), wp, rtol=2e-6, atol=1e-9)
    again = jsx.kernels.verify_drafts(x, ids, u, ws, draft_probs=q, n_draft=nd, temperature=temperature)
    for a, b in zip((acc, tok, pr), again):
        assert torch.equal(a, b)
    return int(clear.sum())


@pytest.mark.parametrize("B,T,V,f32,probs,temperature", [
    (1, 4, 151552, False, False, 1.0), (6, 3, 151552, False, True, 0.7), (3, 1, 32003, True, True, 1.3), (9, 8, 1000, False, True, 1.0),
    (5, 2, 4099, True, False, 0.5), (2, 31, 257, False, True, 1.0), (4, 0, 999, False, False, 1.0), (3, 2, 1, False, True, 1.0), (7, 2, 7, True, True, 2.0),
    (3, 5, 70001, False, False, 0.0), (4, 3, 513, True, False, 0.0)])
def test_verify(jsx, cuda, B, T, V, f32, probs, temperature):
    rng = np.random.default_rng(V + T)
    clear = 0
    for trial in range(3):
        x, ids, u, q = make(rng, B, T, V, f32, probs=probs, temperature=temperature)
        nd = None if trial < 2 else rng.integers(0, T + 1, B)
        clear += check(jsx, x, ids, u, q, nd, temperature)
    assert clear >= 1


@pytest.mark.parametrize("probs", [True, False])
def test_output_follows_the_target(jsx, cuda, probs):
    """First tokens over many sequences are distributed as the target's: the total variation
    distance of n = 20000 draws over 6 outcomes is below 4 sqrt(6 / n) / 2."""
    rng = np.random.default_rng(7)
    n, V = 20000, 6
    lg = torch.tensor([0.3, -1.0, 1.2, 0.0, -3.0, 0.9])
    x = lg.to(torch.bfloat16).float().expand(n, 2, V).contiguous().cuda()
    d = torch.softmax(torch.tensor([1.0, 0.5, -0.5, 0.2, 0.0, -1.0]), 0)
    ids = torch.multinomial(d, n, replacement=True, generator=torch.Generator().manual_seed(3)).to(torch.int32)[:, None]
    if not probs:
        ids = torch.full_like(ids, 2)
    q = d.expand(n, 1, V).contiguous().cuda() if probs else None
    u = torch.from_numpy(rng.random((n, 2), dtype=np.float32)).cuda()
    acc, tok, _ = jsx.kernels.verify_drafts(x, ids.cuda().contiguous(), u, jsx.kernels.verify_workspace(n, 1, V, "cuda"), draft_probs=q)
    p = torch.softmax(lg.to(torch.bfloat16).double(), 0).numpy()
    got = np.bincount(tok[:, 0].cpu().numpy(), minlength=V) / n
    assert 0.5 * np.abs(got - p).sum() < 2 * np.sqrt(V / n)
    second = tok[:, 1][acc == 1].cpu().numpy()   # after an accepted draft: a draw from the next row
    got = np.bincount(second, minlength=V) / len(second)
    assert 0.5 * np.abs(got - p).sum() < 2 * np.sqrt(V / len(second))


def test_bounds_of_the_draw(jsx, cuda):
    """Uniforms of 0, just below 1, 1 and NaN give the first and the last token with mass."""
    V = 300
    x = torch.full((4, 1, V), float("-inf"), device="cuda")
    x[:, 0, 17], x[:, 0, 250] = 0.0, -1.0
    u = torch.tensor([[0.0], [1.0 - 2.0 ** -24], [1.0], [float("nan")]], device="cuda")
    none = torch.zeros(4, 0, dtype=torch.int32, device="cuda")
    ws = jsx.kernels.verify_workspace(4, 0, V, "cuda")
    acc, tok, pr = jsx.kernels.verify_drafts(x, none, u, ws)
    assert tok[:, 0].tolist() == [17, 250, 250, 17] and acc.tolist() == [0] * 4 and pr.numel() == 0


def test_rows_without_a_distribution_and_odd_ids(jsx, cuda):
    V, inf, nan = 64, float("inf"), float("nan")
    x = torch.zeros(6, 2, V, device="cuda")
    x[0, 0] = -inf                     # no mass: nothing accepted, no token
    x[1, 0] = nan
    x[2, 0, 5] = inf                   # no finite maximum
    x[3, 0, :] = nan
    x[3, 0, 9] = 2.0                   # NaN has no mass: 9 is certain
    ids = torch.tensor([[1], [1], [5], [9], [-1], [V]], dtype=torch.int32, device="cuda")
    u = torch.full((6, 2), 0.5, device="cuda")
    ws = jsx.kernels.verify_workspace(6, 1, V, "cuda")
    acc, tok, pr = jsx.kernels.verify_drafts(x, ids, u, ws)
    assert acc.tolist() == [0, 0, 0, 1, 0, 0]
    assert tok[:3, 0].tolist() == [-1, -1, -1] and tok[3, 0] == 9 and tok[3, 1] == 32
    assert tok[4:, 0].tolist() == [32, 32] and pr[:, 0].tolist() == [0, 0, 0, 1, 0, 0]
    g = jsx.kernels.verify_drafts(x, ids, None, ws, temperature=0.0)
    assert g[0].tolist() == [0, 0, 1, 1, 0, 0] and g[1][:, 0].tolist() == [-1, -1, 5, 9, 0, 0]


def test_a_draft_of_the_target_itself_is_always_accepted(jsx, cuda):
    """q = p up to fp32: refused with a probability of a few 2^-24; an empty residual draws from p."""
    rng = np.random.default_rng(1)
    x, ids, u, _ = make(rng, 16, 4, 5000, f32=True)
    q = torch.softmax(x[:, :4].double(), -1).float().contiguous()
    ids = torch.multinomial(q.view(64, -1), 1).view(16, 4).to(torch.int32)
    acc, tok, pr = jsx.kernels.verify_drafts(x, ids, u, jsx.kernels.verify_workspace(16, 4, 5000, "cuda"), draft_probs=q)
    assert (acc == 4).all() and (pr > 1 - 1e-5).all()
    one = torch.ones(16, 4, 5000, device="cuda")   # q above p everywhere: refused, and the residual is empty
    acc, tok, _ = jsx.kernels.verify_drafts(x, ids, torch.full_like(u, 0.999), jsx.kernels.verify_workspace(16, 4, 5000, "cuda"), draft_probs=one)
    assert (acc == 0).all() and (tok[:, 0] >= 0).all()


def test_strided_rows_of_logits(jsx, cuda):
    rng = np.random.default_rng(2)
    x, ids, u, q = make(rng, 3, 2, 1001)
    wide = torch.zeros(3, 3, 1500, dtype=x.dtype, device="cuda")
    wide[..., 3:1004] = x                # odd offset and row length: unaligned rows
    ws = jsx.kernels.verify_workspace(3, 2, 1001, "cuda")
    a = jsx.kernels.verify_drafts(x, ids, u, ws, draft_probs=q)
    b = jsx.kernels.verify_drafts(wide[..., 3:1004], ids, u, ws, draft_probs=q)
    for s, t in zip(a, b):
        assert torch.equal(s, t)


def test_one_workspace_for_calls_of_several_shapes(jsx, cuda):
    """Records of one shape lie where another shape keeps its sums: every call leaves zeros."""
    rng = np.random.default_rng(31)
    shapes = [(2, 31, 257), (40, 0, 9001), (9, 4, 3001), (2, 31, 257), (1, 2, 151552), (40, 0, 9001)]
    size = max(jsx.kernels.verify_workspace(B, T, V, torch.device("cuda")).numel() for B, T, V in shapes)
    shared = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for B, T, V in shapes:
        for temperature in (1.0, 0.0):
            x, ids, u, q = make(rng, B, T, V, probs=T > 2, temperature=temperature)
            own = jsx.kernels.verify_workspace(B, T, V, x.device)
            a = jsx.kernels.verify_drafts(x, ids, u, own, draft_probs=q, temperature=temperature)
            b = jsx.kernels.verify_drafts(x, ids, u, shared, draft_probs=q, temperature=temperature)
            assert all(torch.equal(y, z) for y, z in zip(a, b))
            assert not shared.any()


@pytest.mark.parametrize("f32", [False, True])
def test_greedy_takes_the_first_of_equals(jsx, cuda, f32):
    """Equal maxima in one vector, in several and in several slices; +0 and -0 are equal."""
    V = 40000
    x = torch.full((4, 2, V), -1.0, device="cuda", dtype=torch.float32 if f32 else torch.bfloat16)
    x[0, :, [9001, 9002, 30000]] = 2.0
    x[1, :, 17], x[1, :, 39999] = -0.0, 0.0
    x[2, :, 39998], x[2, :, 23] = -0.0, 0.0
    x[3] = float("nan")
    x[3, :, 5], x[3, :, 20000] = float("inf"), float("inf")
    want = torch.tensor([9001, 17, 23, 5], dtype=torch.int32, device="cuda")
    ws = jsx.kernels.verify_workspace(4, 1, V, x.device)
    acc, tok, pr = jsx.kernels.verify_drafts(x, want.view(4, 1), None, ws, temperature=0.0)
    assert (acc == 1).all() and (pr == 1).all() and torch.equal(tok, want.view(4, 1).expand(4, 2))
    acc, tok, pr = jsx.kernels.verify_drafts(x, (want + 1).view(4, 1), None, ws, temperature=0.0)
    assert (acc == 0).all() and (pr == 0).all() and torch.equal(tok[:, 0], want) and (tok[:, 1] == -1).all()


def test_refusals(jsx, cuda):
    K = jsx.kernels
    x = torch.zeros(2, 3, 100, device="cuda")
    ids, u = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda")
    ws = K.verify_workspace(2, 2, 100, "cuda")
    for bad in (lambda: K.verify_drafts(x.half(), ids, u, ws), lambda: K.verify_drafts(x, ids.long(), u, ws),
                lambda: K.verify_drafts(x, ids[:1], u, ws), lambda: K.verify_drafts(x, ids, u[:, :2].contiguous(), ws),
                lambda: K.verify_drafts(x, ids, u, ws, draft_probs=torch.zeros(2, 2, 99, device="cuda"))):
        with pytest.raises((ValueError, TypeError)):
            bad()
    for bad in (lambda: K.verify_drafts(x, ids, None, ws), lambda: K.verify_drafts(x, ids, u, ws[:16]),
                lambda: K.verify_drafts(x, ids, u, ws, temperature=-1.0), lambda: K.verify_drafts(x, ids, u, ws, temperature=float("nan"))):
        with pytest.raises(jsx._lib.JsxError) as e:
            bad()
        assert e.value.status == jsx._lib.JSX_EINVAL
