"""The paged cache's and the verification's oracle on the CPU (oracle/paged_ref.py), and the entry
points' refusals, which answer before any launch."""

import ctypes
import importlib

import numpy as np
import pytest

R = importlib.import_module("oracle.paged_ref")


def test_formats():
    v = R.e4m3_values()
    assert v[0] == 0 and v[1] == 2.0 ** -9 and v[8] == 2.0 ** -6 and v[126] == 448 and np.isnan(v[127])
    assert (np.diff(v[:127]) > 0).all()
    # every code x scale is exact in bf16: 8 significant bits
    x = np.unique(np.outer(R.E2M1, v[:127]))
    assert np.array_equal(x, ((x.astype(np.float32).view(np.uint32) & 0xffff0000).view(np.float32)).astype(np.float64))


def test_ties_go_to_even():
    x = np.zeros((1, 16))
    x[0, :8] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    assert R.stored(x)[0, :8].tolist() == [6, 0, 1, 1, 2, 2, 4, 4]
    assert R.stored(-x)[0, :8].tolist() == [-6, 0, -1, -1, -2, -2, -4, -4]


def test_stored_rows_are_near_and_stable():
    x = np.random.default_rng(0).standard_normal((200, 64))
    y = R.stored(x)
    assert np.array_equal(R.stored(y), y)   # a stored row is stored as itself
    step = np.abs(x.reshape(200, 4, 16)).max(-1).repeat(16, -1) / 6
    assert (np.abs(x - y) <= 1.07 * step).all()


def test_a_planted_mistake_shows():
    """Halves away from zero instead of to even: the exact comparison of the GPU tests sees it."""
    def wrong(x, grid):
        hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
        return np.where(x - grid[hi - 1] >= grid[hi] - x, hi, hi - 1)
    x = np.zeros((1, 16))
    x[0, :3] = [6, 0.25, 1.25]
    right = R.stored(x)
    keep, R._nearest_even = R._nearest_even, wrong
    try:
        assert not np.array_equal(R.stored(x), right)
    finally:
        R._nearest_even = keep


def test_attention_is_softmax_over_what_is_seen():
    rng = np.random.default_rng(1)
    k, v = rng.standard_normal((4, 1, 16, 64)), rng.standard_normal((4, 1, 16, 64))
    q = rng.standard_normal((3, 2, 64))
    t = np.array([[2, 0, 3]])
    out, big = R.attention(q, k, v, t, [20], 3, window=10, sinks=2)
    rows_k, rows_v = np.concatenate([k[p, 0] for p in t[0]]), np.concatenate([v[p, 0] for p in t[0]])
    for i in range(3):
        see = [j for j in range(21 + i) if j > 20 + i - 10 or j < 2]
        s = rows_k[see] @ q[i, 1] / 8
        w = np.exp(s) / np.exp(s).sum()
        assert np.allclose(out[i, 1], w @ rows_v[see])
    none, _ = R.attention(q, k, v, np.array([[-1, -1, -1]]), [20], 3)
    assert not none.any()


def test_pages_keep_their_counts():
    rng = np.random.default_rng(2)
    S, slots, P, pt = 6, 8, 60, 16
    t, h, r = np.full((S, slots), -1, np.int32), np.zeros(S, np.int32), np.zeros(P, np.int32)
    holders = lambda t, h: np.bincount(np.concatenate([t[b, :h[b]] for b in range(S)]), minlength=P)  # noqa: E731
    length = np.zeros(S, int)
    for _ in range(60):
        keep = np.array([rng.integers(0, n + 1) for n in length])
        need = np.minimum(keep + rng.integers(0, 40, S), slots * pt)
        t, h, r, copies, missing = R.pages_resize(t, h, r, keep, need, pt)
        if not missing:
            length = need
        assert np.array_equal(r, holders(t, h))
        for b in range(S):   # written pages have one holder
            if not missing:
                assert all(r[p] == 1 for p in t[b, keep[b] // pt:h[b]])
        parent = np.where(rng.random(S) < 0.3, rng.integers(-1, S, S), np.arange(S))
        t, h, r = R.pages_fork(t, h, r, parent)
        length = np.where(parent >= 0, length[parent], 0)
        assert np.array_equal(r, holders(t, h))
        t, r, remap, moves = R.pages_compact(t, h, r)
        assert np.array_equal(r, holders(t, h)) and not r[(r > 0).sum():].any()


def test_verification_keeps_the_targets_distribution():
    """Exact: over a grid of uniforms, first tokens have the target's probabilities."""
    rng = np.random.default_rng(3)
    V, n = 4, 200
    x = rng.standard_normal((1, 2, V)).astype(np.float32)
    q = rng.random(V)
    q = (q / q.sum()).astype(np.float32)
    p = np.exp(x[0, 0].astype(float)) / np.exp(x[0, 0].astype(float)).sum()
    got = np.zeros(V)
    grid = (np.arange(n) + 0.5) / n
    for d in range(V):
        u = np.stack(np.meshgrid(grid, grid), -1).reshape(-1, 2).astype(np.float32)
        acc, tok, _, _ = R.verify(np.broadcast_to(x, (n * n, 2, V)), np.full((n * n, 1), d), u,
                                  np.broadcast_to(q, (n * n, 1, V)))
        got += q[d] * np.bincount(tok[:, 0], minlength=V) / (n * n)
    assert np.abs(got - p).max() < 2 / n


REFUSED = [
    ("jsx_kv4_append", (256, 256, 0, 256, 128, 0, 256, 4, 256, 2, 256, None, 1, 1, 2, 128, 48, None)),   # 48 tokens a page
    ("jsx_kv4_append", (256, 256, 0, 12, 128, 0, 256, 4, 256, 2, 256, None, 1, 1, 2, 128, 64, None)),    # stride of 12 elements
    ("jsx_kv4_append", (264, 256, 0, 256, 128, 0, 256, 4, 256, 2, 256, None, 1, 1, 2, 128, 64, None)),   # k not 16-byte aligned
    ("jsx_kv4_append", (None, 256, 0, 256, 128, 0, 256, 4, 256, 2, 256, None, 1, 1, 2, 128, 64, None)),
    ("jsx_kv4_read", (256, 4, 256, 2, 256, None, 256, 256, 0, 256, 128, -1, 1, 1, 2, 128, 64, None)),
    ("jsx_kv4_attn", (256, 1024, 256, 4, 256, 2, 256, None, 256, 1024, 1, 1, 8, 3, 128, 64, 0, 0, 0.1, 256, 1 << 30, None)),   # 8 heads over 3
    ("jsx_kv4_attn", (256, 512, 256, 4, 256, 2, 256, None, 256, 1024, 1, 1, 8, 2, 128, 64, 0, 0, 0.1, 256, 1 << 30, None)),    # stride below a row
    ("jsx_kv4_attn", (256, 1024, 256, 4, 256, 2, 256, None, 256, 1024, 1, 1, 8, 2, 128, 64, -1, 0, 0.1, 256, 1 << 30, None)),
    ("jsx_kv4_attn", (256, 1024, 256, 4, 256, 2, 256, None, 256, 1024, 1, 1, 8, 2, 128, 64, 0, 0, 0.1, 256, 0, None)),         # no workspace
    ("jsx_pages_fork", (256, 256, 256, 256, 256, 512, 512, 4, 4, 16, None)),                             # table_out is table
    ("jsx_pages_fork", (256, 256, 256, None, 512, 512, 512, 4, 4, 16, None)),
    ("jsx_pages_resize", (256, 256, 256, 256, 256, 256, 1, 24, 4, 4, 16, 16, 256, 256, 1 << 20, None)),  # 24 bytes a page
    ("jsx_pages_resize", (256, 256, 256, 256, 256, 256, 1, 32, 4, 4, 16, 16, 256, 256, 8, None)),        # small workspace
    ("jsx_pages_resize", (256, 256, 256, 256, 256, 256, 1, 32, 1 << 16, 4, 16, 16, 256, 256, 1 << 30, None)),   # too many sequences
    ("jsx_pages_compact", (256, 256, 256, 256, 0, 32, 256, 256, 256, 4, 4, 16, 256, 1 << 20, None)),     # no layer
    ("jsx_verify_drafts", (256, 0, 100, 256, None, None, 256, 1.0, 256, 256, 256, 2, 32, 100, 256, 1 << 20, None)),    # 32 drafts
    ("jsx_verify_drafts", (256, 0, 99, 256, None, None, 256, 1.0, 256, 256, 256, 2, 3, 100, 256, 1 << 20, None)),      # rows overlap
    ("jsx_verify_drafts", (256, 0, 100, 256, None, None, None, 1.0, 256, 256, 256, 2, 3, 100, 256, 1 << 20, None)),    # no uniforms
    ("jsx_verify_drafts", (256, 0, 100, 256, None, None, 256, float("inf"), 256, 256, 256, 2, 3, 100, 256, 1 << 20, None)),
    ("jsx_verify_drafts", (256, 0, 100, 256, None, None, 256, 1.0, 256, 256, 256, 2, 3, 100, 256, 8, None)),
]


@pytest.mark.parametrize("call,args", REFUSED)
def test_invalid_arguments_are_rejected_on_the_host(jsx, call, args):
    lib = jsx._lib
    with pytest.raises(lib.JsxError) as e:
        lib.call(call, *args)
    assert e.value.status == lib.JSX_EINVAL and lib.last_error()


def test_head_dims_outside_the_cache_are_not_supported(jsx):
    lib = jsx._lib
    n = ctypes.c_size_t(0)
    for call, args in (("jsx_kv4_page_bytes", (2, 96, 64, ctypes.byref(n))),
                       ("jsx_kv4_append", (256, 256, 0, 256, 256, 0, 256, 4, 256, 2, 256, None, 1, 1, 2, 256, 64, None))):
        with pytest.raises(lib.JsxError) as e:
            lib.call(call, *args)
        assert e.value.status == lib.JSX_ENOTSUP


def test_sizes(jsx):
    lib = jsx._lib
    n = ctypes.c_size_t(0)
    lib.call("jsx_kv4_page_bytes", 2, 128, 64, ctypes.byref(n))
    assert n.value == 2 * 64 * (128 + 16)      # 4.5 bits for each of 2 x 128 values
    for call, args in (("jsx_pages_workspace_size", (0, 4, 16)), ("jsx_verify_workspace_size", (1, 32, 100)),
                       ("jsx_verify_workspace_size", (1, 3, (1 << 20) + 1)), ("jsx_kv4_attn_workspace_size", (1, 1, 8, 3, 128))):
        with pytest.raises(lib.JsxError):
            lib.call(call, *args, ctypes.byref(n))
