"""jsx_pages_resize where keep[b] goes past the pages that row b holds: a row keeps at most what it
has, and gets pages for the rest like for any other token.  This happens in use: after a resize
that lacked pages, while positions moved on; after a fork that emptied a row whose length is still
the old one."""

import importlib

import numpy as np
import pytest
import torch

R = importlib.import_module("oracle.paged_ref")


def holders(table, held, P):
    rows = [table[b, :held[b]] for b in range(len(held))]
    return np.bincount(np.concatenate(rows), minlength=P).astype(np.int32)


def case(name):
    """(table, held, refs, keep, need, page tokens): every count in refs is a row's."""
    pt, P = 16, 24
    table, held = np.full((4, 6), -1, np.int32), np.zeros(4, np.int32)
    if name == "one page of four":
        table[0, 0], held[0] = 5, 1
        keep, need = [64, 0, 0, 0], [80, 0, 0, 0]
    elif name == "empty rows":
        keep, need = [1, 40, 96, 0], [1, 41, 96, 17]
    elif name == "emptied by a fork":
        table[0, :3], table[1, :2] = [7, 3, 9], [0, 1]
        held[:2] = [3, 2]
        table, held, _ = R.pages_fork(table, held, holders(table, held, P), np.array([0, -1, 0, -1]))
        keep, need = [40, 30, 40, 0], [41, 33, 40, 0]
    else:                                     # after a resize that lacked pages
        pt = 4
        table[0, :2], table[1, :1], held[:2] = [3, 8], [2], [2, 1]
        refs = holders(table, held, P)
        *_, missing = R.pages_resize(table, held, refs, np.array([8, 4, 0, 0]), np.array([24, 24, 24, 25]), pt)
        assert missing
        keep, need = [9, 12, 3, 0], [10, 13, 4, 0]
    return table, held, holders(table, held, P), np.array(keep, np.int32), np.array(need, np.int32), pt


NAMES = ["one page of four", "empty rows", "emptied by a fork", "after too few pages"]


@pytest.mark.parametrize("name", NAMES)
def test_the_oracle_gives_every_slot_a_page(name):
    table, held, refs, keep, need, pt = case(name)
    t, h, r, copies, missing = R.pages_resize(table, held, refs, keep, need, pt)
    assert missing == 0 and h.tolist() == [-(-n // pt) for n in need]
    for b in range(4):
        assert (t[b, :h[b]] >= 0).all() and (t[b, h[b]:] == -1).all()
        kept = min(keep[b] // pt, held[b], h[b])
        assert (t[b, :kept] == table[b, :kept]).all()
    assert np.array_equal(r, holders(t, h, len(refs)))
    for a, b in copies:                       # only what was there is copied
        assert refs[a] > 1 and refs[b] == 0


def resize(jsx, table, held, refs, keep, need, pt, pool):
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x, np.int32)).cuda()  # noqa: E731
    dt, dh, dr = dev(table), dev(held), dev(refs)
    ws = jsx.kernels.pages_workspace(len(held), table.shape[1], len(refs), "cuda").zero_()
    m = jsx.kernels.pages_resize(dt, dh, dr, dev(keep), dev(need), pool, pt, ws)
    return dt.cpu().numpy(), dh.cpu().numpy(), dr.cpu().numpy(), int(m)


def compare(jsx, table, held, refs, keep, need, pt, layers=2, nbytes=32, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    pool = torch.randint(0, 256, (layers, len(refs), 1, nbytes), dtype=torch.uint8, device="cuda", generator=g)
    want_pool = pool.clone()
    t, h, r, copies, missing = R.pages_resize(table, held, refs, keep, need, pt)
    for a, b in copies:
        want_pool[:, b] = pool[:, a]
    gt, gh, gr, gm = resize(jsx, table, held, refs, keep, need, pt, pool)
    assert gm == missing
    assert np.array_equal(gt, t) and np.array_equal(gh, h) and np.array_equal(gr, r)
    assert torch.equal(pool, want_pool)
    if not missing:
        assert np.array_equal(gr - holders(gt, gh, len(refs)), refs - holders(table, held, len(refs)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_keep_past_the_held_pages(jsx, cuda, name):
    compare(jsx, *case(name))


@pytest.mark.gpu
@pytest.mark.parametrize("S,slots,P,pt", [(1, 3, 4, 16), (33, 20, 900, 64), (300, 40, 12001, 16)])   # the last: a cluster of CTAs
def test_keep_past_the_held_pages_of_many_rows(jsx, cuda, S, slots, P, pt):
    rng = np.random.default_rng(S)
    for trial in range(3):
        free = list(rng.permutation(P))
        table, held = np.full((S, slots), -1, np.int32), np.zeros(S, np.int32)
        for b in range(S):
            if b and rng.random() < 0.3:
                src = int(rng.integers(0, b))
                held[b] = rng.integers(0, held[src] + 1)
                table[b, :held[b]] = table[src, :held[b]]
            while held[b] < slots and len(free) > P // 2 and rng.random() < 0.7:
                table[b, held[b]] = free.pop()
                held[b] += 1
        keep = rng.integers(0, slots * pt + 1, S).astype(np.int32)
        need = np.minimum(keep + rng.integers(-pt, 2 * pt, S), slots * pt).astype(np.int32)
        if trial == 2:                        # few rows grow, so that the pages suffice
            grow = rng.random(S) < 0.1
            keep, need = np.where(grow, keep, 2 ** 31 - 1), np.where(grow, need, held * pt)
        compare(jsx, table, held, holders(table, held, P), keep.astype(np.int32), need.astype(np.int32), pt, seed=trial)
