"""Sharing, resizing and compacting pages (jsx_pages_*) against the sequential oracle
(oracle/paged_ref.py): tables, counts and moved bytes are equal exactly."""

import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

R = importlib.import_module("oracle.paged_ref")


def dev(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def host(t):
    return t.cpu().numpy()


def state(rng, S, slots, P, fill=0.6):
    """Rows that hold some pages, some of them shared, on a scattered part of the pool."""
    free = list(rng.permutation(P))
    table, held, refs = np.full((S, slots), -1, np.int32), np.zeros(S, np.int32), np.zeros(P, np.int32)
    for b in range(S):
        if b and rng.random() < 0.4:      # shares the first pages of an earlier row
            src = int(rng.integers(0, b))
            n = int(rng.integers(0, held[src] + 1))
            table[b, :n] = table[src, :n]
            held[b] = n
        want = int(rng.integers(0, slots + 1))
        while held[b] < want and len(free) > (1 - fill) * P:
            table[b, held[b]] = free.pop()
            held[b] += 1
        refs += np.bincount(table[b, :held[b]], minlength=P).astype(np.int32)
    return table, held, refs


def pool_of(rng, layers, P, nbytes):
    return torch.from_numpy(rng.integers(0, 256, (layers, P, 1, nbytes), dtype=np.uint8)).cuda()


@pytest.mark.parametrize("S,slots,P", [(1, 1, 1), (3, 4, 16), (40, 9, 300), (300, 33, 9001), (1500, 5, 4000)])
def test_fork(jsx, cuda, S, slots, P):
    rng = np.random.default_rng(S)
    table, held, refs = state(rng, S, slots, P)
    refs[rng.integers(0, P)] += 1         # a hold of someone else's
    for parent in (np.arange(S), rng.integers(-1, S, S), np.zeros(S), np.full(S, -1), np.full(S, S + 5)):
        parent = parent.astype(np.int32)
        want = R.pages_fork(table, held, refs, parent)
        got = jsx.kernels.pages_fork(dev(table), dev(held), dev(refs), dev(parent))
        for w, g in zip(want, got):
            assert np.array_equal(w, host(g))
    r = dev(refs)                          # counts in place
    got = jsx.kernels.pages_fork(dev(table), dev(held), r, dev(parent), refs_out=r)
    assert np.array_equal(host(r), want[2])


@pytest.mark.parametrize("S,slots,P,pt,layers,nbytes", [
    (1, 1, 2, 16, 1, 16), (4, 6, 64, 16, 3, 144), (33, 20, 900, 64, 2, 4608), (200, 70, 20011, 32, 1, 48), (1100, 4, 9000, 128, 2, 16)])
def test_resize(jsx, cuda, S, slots, P, pt, layers, nbytes):
    rng = np.random.default_rng(S + slots)
    for trial in range(3):
        table, held, refs = state(rng, S, slots, P, fill=0.3)
        keep = np.array([rng.integers(0, h * pt + 1) for h in held], np.int32)
        need = np.minimum(keep + rng.integers(-pt, 3 * pt, S), slots * pt).astype(np.int32)
        if trial == 1:
            need[rng.random(S) < 0.5] = 0      # freed
        if trial == 2:
            keep, need = held * pt, held * pt  # nothing to do
        pool = pool_of(rng, layers, P, nbytes)
        want_pool = pool.clone()
        t, h, r, copies, missing = R.pages_resize(table, held, refs, keep, need, pt)
        for a, b in copies:
            want_pool[:, b] = pool[:, a]
        dt, dh, dr = dev(table), dev(held), dev(refs)
        ws = jsx.kernels.pages_workspace(S, slots, P, "cuda")
        m = jsx.kernels.pages_resize(dt, dh, dr, dev(keep), dev(need), pool, pt, ws)
        assert int(m) == missing
        assert np.array_equal(host(dt), t) and np.array_equal(host(dh), h) and np.array_equal(host(dr), r)
        assert torch.equal(pool, want_pool)


def test_resize_copies_shared_last_pages_once_per_writer(jsx, cuda):
    """Four rows on one prompt of 2.5 pages: each gets a copy of the third page and shares the first two."""
    pt, slots, P = 16, 5, 32
    table, held, refs = np.full((4, slots), -1, np.int32), np.array([3, 0, 0, 0], np.int32), np.zeros(P, np.int32)
    table[0, :3] = [7, 3, 9]
    refs[[7, 3, 9]] = 1
    pool = pool_of(np.random.default_rng(0), 2, P, 32)
    t, h, r = jsx.kernels.pages_fork(dev(table), dev(held), dev(refs), dev([0, 0, 0, 0]))
    assert host(r)[[7, 3, 9]].tolist() == [4, 4, 4]
    ws = jsx.kernels.pages_workspace(4, slots, P, "cuda")
    keep, need = dev([40] * 4), dev([49, 41, 40, 48])     # row 2 writes nothing, yet its partial page becomes its own
    assert int(jsx.kernels.pages_resize(t, h, r, keep, need, pool, pt, ws)) == 0
    tt = host(t)
    assert tt[:, :2].tolist() == [[7, 3]] * 4
    assert tt[:, 2:4].tolist() == [[0, 1], [2, -1], [4, -1], [5, -1]]
    assert host(r)[[7, 3, 9, 0, 1, 2, 4, 5]].tolist() == [4, 4, 0, 1, 1, 1, 1, 1]
    for p in (0, 2, 4, 5):
        assert torch.equal(pool[:, p], pool[:, 9])
    # given back: everything becomes free again
    zero = dev([0] * 4)
    assert int(jsx.kernels.pages_resize(t, h, r, zero, zero, pool, pt, ws)) == 0
    assert not host(r).any() and (host(t) == -1).all() and not host(h).any()


def test_resize_is_all_or_nothing(jsx, cuda):
    pt, slots, P = 16, 4, 6
    table, held, refs = np.full((3, slots), -1, np.int32), np.array([2, 1, 0], np.int32), np.zeros(P, np.int32)
    table[0, :2], table[1, 0] = [5, 0], 2
    refs[[5, 0, 2]] = 1
    ws = jsx.kernels.pages_workspace(3, slots, P, "cuda")
    pool = pool_of(np.random.default_rng(0), 1, P, 16)
    for need, missing in (([64, 32, 32], 2), ([100, 16, 0], 2 + 3 - 3), ([2 ** 31 - 1, 0, 0], None)):
        t, h, r = dev(table), dev(held), dev(refs)
        m = int(jsx.kernels.pages_resize(t, h, r, dev([32, 16, 0]), dev(need), pool, pt, ws))
        want = R.pages_resize(table, held, refs, np.array([32, 16, 0]), np.array(need), pt)
        if missing is None:
            assert m > 0
        else:
            assert m == want[4]
        if m:
            assert np.array_equal(host(t), table) and np.array_equal(host(h), held) and np.array_equal(host(r), refs)
        else:
            assert np.array_equal(host(t), want[0])


@pytest.mark.parametrize("S,slots,P,layers,nbytes", [(1, 1, 1, 1, 16), (5, 7, 50, 2, 32), (64, 20, 3000, 3, 4608), (30, 400, 40000, 1, 16)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(jsx, cuda, S, slots, P, layers, nbytes, in_place):
    rng = np.random.default_rng(P)
    for fill in (0.5, 1.0, 0.0):
        table, held, refs = state(rng, S, slots, P, fill)
        if fill == 0.0:                    # nothing live but one page that only an outside holder has
            table[:], held[:], refs[:] = -1, 0, 0
            refs[P - 1] = 2
        pool = pool_of(rng, layers, P, nbytes)
        want_pool = pool.clone()
        t, r, remap, moves = R.pages_compact(table, held, refs)
        if moves:
            a, b = zip(*moves)
            want_pool[:, list(b)] = pool[:, list(a)]
        dt, dr = dev(table), dev(refs)
        ws = jsx.kernels.pages_workspace(S, slots, P, "cuda")
        got = jsx.kernels.pages_compact(dt, dev(held), dr, pool, ws, table_out=dt if in_place else None, refs_out=dr if in_place else None)
        for w, g in zip((t, r, remap), got):
            assert np.array_equal(w, host(g))
        assert torch.equal(pool, want_pool)
        live = int((refs > 0).sum())
        assert (host(got[1])[:live] > 0).all() and not host(got[1])[live:].any()


def test_compacting_changes_no_answer(jsx, cuda):
    """Attention over a table and its compacted form gives the same bits."""
    K = jsx.kernels
    rng = np.random.default_rng(1)
    B, nkv, hd, pt, P = 5, 2, 128, 32, 64
    lens = [130, 3, 64, 200, 31]
    order = rng.permutation(P)
    table, at = np.full((B, 7), -1, np.int32), 0
    for b, n in enumerate(lens):
        k = -(-n // pt)
        table[b, :k] = order[at:at + k]
        at += k
    held = (table >= 0).sum(1).astype(np.int32)
    refs = np.zeros(P, np.int32)
    refs[order[:at]] = 1
    nb = K.kv4_page_bytes(nkv, hd, pt)
    pool = torch.zeros(2, P, nkv, nb // nkv, dtype=torch.uint8, device="cuda")
    k = torch.randn(B * 200, nkv, hd, device="cuda").to(torch.bfloat16)
    for layer in range(2):
        K.kv4_append(k, k, pool[layer], dev(table), dev([0] * B), tokens_per_seq=200, n_tokens=dev(lens))
    q = torch.randn(B, 16 * hd, device="cuda").to(torch.bfloat16)
    ws = K.kv4_attn_workspace(B, 1, 16, nkv, hd, q.device)
    pos = dev([n - 1 for n in lens])
    a = [K.kv4_attn(q, pool[i], dev(table), pos, hd, ws) for i in range(2)]
    t2, _, _ = K.pages_compact(dev(table), dev(held), dev(refs), pool, K.pages_workspace(B, 7, P, "cuda"))
    assert int(t2.max()) == at - 1
    for i in range(2):
        assert torch.equal(a[i], K.kv4_attn(q, pool[i], t2, pos, hd, ws))


def test_refusals(jsx, cuda):
    K = jsx.kernels
    t, h, r = dev([[0, 1]]), dev([2]), dev([1, 1, 0])
    pool = torch.zeros(1, 3, 1, 32, dtype=torch.uint8, device="cuda")
    ws = K.pages_workspace(1, 2, 3, "cuda")
    with pytest.raises(jsx._lib.JsxError):
        K.pages_fork(t, h, r, dev([0]), table_out=t)
    with pytest.raises(jsx._lib.JsxError):
        K.pages_resize(t, h, r, dev([0]), dev([1]), pool, 16, ws[:16])
    with pytest.raises(jsx._lib.JsxError):
        K.pages_resize(t, h, r, dev([0]), dev([1]), pool, 0, ws)
    for bad in (lambda: K.pages_fork(t, h, r, dev([0, 0])), lambda: K.pages_fork(t.long(), h, r, dev([0])),
                lambda: K.pages_resize(t, h, r, dev([0]), dev([1]), pool[:, :2], 16, ws),
                lambda: K.pages_compact(t, dev([1, 1]), r, pool, ws)):
        with pytest.raises((ValueError, TypeError)):
            bad()
