"""The 4-bit cache's rows (jsx_kv4_append, jsx_kv4_read) and the attention over its pages
(jsx_kv4_attn) against the 64-bit oracle (oracle/paged_ref.py).

Rows read back are exact: the codes and scales are those of the definition, and their product
is a bf16 value.  Attention's bound per output, with V the largest visible |v|:
2^-8 |o| + 2^-9 V.  The output's rounding to bf16 is 2^-9 |o|; weights rounded to f16 (2^-11
each, numerator only) move o by at most 2^-11 V + 2^-11 |o|; an fp32 dot product over 128
dimensions of a tensor core that truncates is within 128 x 2^-22 of the sum of its terms'
magnitudes, below 2^-12 of a weight for scores up to 2^3, the rest is fp32 rounding."""

import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

R = importlib.import_module("oracle.paged_ref")
BF = torch.bfloat16


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x)).to(device="cuda", dtype=dtype)


def rows(rng, *shape):
    x = rng.standard_normal(shape, dtype=np.float32) * np.exp(rng.standard_normal(shape[:-1] + (1,), dtype=np.float32))
    return dev(x, BF)


def f64(t):
    return t.detach().double().cpu().numpy()


def make_table(rng, need, pt, slots=None, spare=2):
    """Scattered pages for `need` tokens per sequence."""
    n = [-(-max(x, 0) // pt) for x in need]
    order = rng.permutation(sum(n) + spare)
    t = np.full((len(need), slots or max(max(n), 1)), -1, np.int32)
    at = 0
    for b, k in enumerate(n):
        t[b, :k] = order[at:at + k]
        at += k
    return t, sum(n) + spare


def make_pool(jsx, pages, nkv, hd, pt, fill=0xff):
    """A pool of bytes that are NaN scales: rows nobody wrote must not be looked at."""
    n = jsx.kernels.kv4_page_bytes(nkv, hd, pt)
    return torch.full((pages, nkv, n // nkv), fill, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("B,T,nkv,hd,pt,start,static", [
    (1, 1, 1, 128, 16, 0, False),
    (3, 5, 2, 128, 64, 61, False),      # across a page's end
    (2, 33, 8, 64, 32, 7, True),
    (5, 130, 2, 64, 128, 1000, True),
    (2, 257, 3, 128, 16, 3, False),
])
def test_rows_read_back_exactly(jsx, cuda, B, T, nkv, hd, pt, start, static):
    rng = np.random.default_rng(hd + T)
    table, pages = make_table(rng, [start + b + T for b in range(B)], pt)
    pos = dev([start + b for b in range(B)])
    pool = make_pool(jsx, pages, nkv, hd, pt)
    L = start + B + T + 3
    k, v = (rows(rng, *((B, L) if static else (B * T,)), nkv, hd) for _ in "kv")
    jsx.kernels.kv4_append(k, v, pool, dev(table), pos, tokens_per_seq=T)
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    jsx.kernels.kv4_read(pool, dev(table), pos, ko, vo, tokens_per_seq=T)
    for x, y in ((k, ko), (v, vo)):
        want, got = f64(x), f64(y)
        if static:
            untouched = np.ones((B, L), bool)
            for b in range(B):
                untouched[b, start + b:start + b + T] = False
            assert (got[untouched] == 7.0).all()
            want, got = want[~untouched], got[~untouched]
        assert np.array_equal(R.stored(want), got)
    # the bytes in the pool decode to the same values
    kp, vp = R.unpack_pool(pool.cpu().numpy(), hd)
    for b in range(B):
        p = start + b + T - 1
        last = f64(k[b, p] if static else k[(b + 1) * T - 1])
        assert np.array_equal(kp[table[b, p // pt], :, p % pt], R.stored(last))


def test_ties_extremes_and_special_values(jsx, cuda):
    """Quotients on every rounding boundary, subnormal and saturated scales, zeros, infinities, NaN."""
    x = np.zeros((12, 1, 64), np.float32)
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    for r, s in enumerate([1.0, 0.8125, 2.0 ** -9, 448.0]):
        x[r, 0, :14] = np.array([m * s * sg for m in mids for sg in (1, -1)])
        x[r, 0, 15] = 6 * s
        x[r, 0, 16:23], x[r, 0, 31] = np.array(mids) * s * 1.0078125, -6 * s
    x[4, 0, :16] = 1e-6                     # scale rounds to 0
    x[5, 0, 0] = 6 * 2.0 ** -10             # half of the smallest scale: ties to 0
    x[6, 0, 0] = 6.2 * 2.0 ** -10
    x[7, 0, :3] = [1e30, -1e30, 5.0]        # saturates
    x[8, 0, :2] = [np.inf, 1.0]
    x[9, 0, :2] = [-np.inf, -3000.0]
    x[10, 0, 5] = np.nan                    # its group only
    x[10, 0, 20] = 1.0
    k = dev(x, BF)
    pool = make_pool(jsx, 1, 1, 64, 16)
    pos, table = dev([0]), dev([[0]])
    jsx.kernels.kv4_append(k, k, pool, table, pos, tokens_per_seq=12)
    out, out2 = torch.empty_like(k), torch.empty_like(k)
    jsx.kernels.kv4_read(pool, table, pos, out, out2, tokens_per_seq=12)
    assert np.array_equal(R.stored(f64(k)), f64(out), equal_nan=True)
    assert np.array_equal(f64(out), f64(out2), equal_nan=True)


def test_every_bf16_magnitude_against_every_tie(jsx, cuda):
    """All positive bf16 values within a group whose scale every one of them sets in turn."""
    bits = np.arange(0x0001, 0x7f80, dtype=np.uint16)
    top = (bits.astype(np.uint32) << 16).view(np.float32)
    rng = np.random.default_rng(0)
    x = np.zeros((len(top), 1, 64), np.float32)
    x[:, 0, 0] = top
    x[:, 0, 1:16] = top[:, None] * (rng.integers(0, 129, (len(top), 15)) / 128).astype(np.float32)
    k = dev(x, BF)
    n = len(top)
    pool = make_pool(jsx, -(-n // 128), 1, 64, 128)
    table, pos = dev(np.arange(-(-n // 128))[None]), dev([0])
    jsx.kernels.kv4_append(k, k, pool, table, pos, tokens_per_seq=n)
    out, o2 = torch.empty_like(k), torch.empty_like(k)
    jsx.kernels.kv4_read(pool, table, pos, out, o2, tokens_per_seq=n)
    assert np.array_equal(R.stored(f64(k)), f64(out))


def test_unused_tokens_missing_pages_and_strided_rows(jsx, cuda):
    rng = np.random.default_rng(5)
    B, T, nkv, hd, pt = 3, 4, 2, 128, 16
    fused = rows(rng, B * T, 6, hd)           # q | k | v of a fused projection
    k, v = fused[:, 2:4], fused[:, 4:6]
    table = dev([[0, 1], [2, -1], [3, 4]])
    pos = dev([14, 14, -2])                   # crosses a page; second page missing; two negative positions
    nt = dev([3, 4, 4])
    pool = make_pool(jsx, 5, nkv, hd, pt)
    before = pool.clone()
    jsx.kernels.kv4_append(k, v, pool, table, pos, tokens_per_seq=T, n_tokens=nt)
    out_k, out_v = torch.full((B * T, nkv, hd), 7.0, dtype=BF, device="cuda"), torch.full((B * T, nkv, hd), 7.0, dtype=BF, device="cuda")
    jsx.kernels.kv4_read(pool, table, pos, out_k, out_v, tokens_per_seq=T, n_tokens=nt)
    want = R.stored(f64(k))
    got = f64(out_k)
    used = {0: (0, 1, 2), 1: (0, 1), 2: (2, 3)}
    for b in range(B):
        for i in range(T):
            r = b * T + i
            if i in used[b]:
                assert np.array_equal(got[r], want[r])
            elif b == 1:
                assert (got[r] == 0).all()     # no page: zeros
            else:
                assert (got[r] == 7).all()     # not a token of the call
    assert np.array_equal(f64(out_v)[0], R.stored(f64(v))[0])
    blk = pool[0].cpu().numpy() != before[0].cpu().numpy()
    assert not blk[:, :14 * hd // 2].any()     # rows before the first position are as they were


def attn_case(jsx, rng, B, T, nq, nkv, hd, pt, positions, window=0, sinks=0, n_tokens=None, table=None, scale=None,
              slots=None):
    need = [p + T for p in positions]
    t, pages = make_table(rng, need, pt, slots)
    if table is not None:
        t = table(t)
    pool = make_pool(jsx, pages, nkv, hd, pt)
    n = max(max(need), 1)
    k, v = rows(rng, B, n, nkv, hd), rows(rng, B, n, nkv, hd)
    jsx.kernels.kv4_append(k, v, pool, dev(t), dev([0] * B), tokens_per_seq=n, n_tokens=dev([max(x, 0) for x in need]))
    q = rows(rng, B * T, nq * hd)
    nt = None if n_tokens is None else dev(n_tokens)
    ws = jsx.kernels.kv4_attn_workspace(B, T, nq, nkv, hd, q.device)
    pos = dev(positions)
    got = jsx.kernels.kv4_attn(q, pool, dev(t), pos, hd, ws, scale=scale, tokens_per_seq=T, n_tokens=nt, window=window,
                               sinks=sinks)
    kp, vp = R.unpack_pool(pool.cpu().numpy(), hd)
    want, big = R.attention(f64(q).reshape(B * T, nq, hd), kp, vp, t, positions, T, window, sinks, scale, n_tokens)
    err = np.abs(f64(got).reshape(want.shape) - want)
    bound = 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * big
    assert np.isfinite(f64(got)).all()
    assert (err <= bound).all(), (err / np.maximum(bound, 1e-30)).max()
    # the same call again: same bits, and a workspace fit for the next call
    again = jsx.kernels.kv4_attn(q, pool, dev(t), pos, hd, ws, scale=scale, tokens_per_seq=T, n_tokens=nt,
                                 window=window, sinks=sinks)
    assert torch.equal(got, again)
    return got


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,nkv,pt", [(32, 2, 64), (1, 1, 16), (8, 1, 32), (14, 2, 128), (12, 4, 16), (20, 1, 64)])
def test_attention_lengths(jsx, cuda, hd, nq, nkv, pt):
    """One token per sequence, lengths around the pages' and blocks' ends, and none at all."""
    rng = np.random.default_rng(hd * nq + pt)
    positions = [0, 1, 15, 16, 62, 63, 64, 127, 128, 200, 1023, -1]
    attn_case(jsx, rng, len(positions), 1, nq, nkv, hd, pt, positions)


@pytest.mark.parametrize("T,nq,nkv,hd,pt", [(2, 32, 2, 128, 64), (5, 32, 2, 128, 64), (8, 16, 1, 128, 16), (3, 14, 2, 64, 32),
                                            (8, 12, 12, 64, 16), (9, 32, 2, 128, 128), (70, 16, 1, 128, 64)])
def test_attention_several_tokens(jsx, cuda, T, nq, nkv, hd, pt):
    rng = np.random.default_rng(T)
    positions = [0, 60, 331, -T + 1]
    attn_case(jsx, rng, 4, T, nq, nkv, hd, pt, positions, n_tokens=[T, T - 1, T, T])


@pytest.mark.parametrize("T,window,sinks", [(1, 1, 0), (1, 7, 2), (1, 64, 4), (1, 100, 70), (4, 1, 0), (4, 16, 1),
                                            (4, 130, 200), (40, 33, 5), (1, 100000, 3)])
def test_attention_window_and_sinks(jsx, cuda, T, window, sinks):
    rng = np.random.default_rng(window + T)
    attn_case(jsx, rng, 4, T, 16, 2, 128, 32, [0, 63, 300, 777], window=window, sinks=sinks)


def test_attention_does_not_see_masked_rows(jsx, cuda):
    """NaN and infinite rows outside the window, after the position and in unwritten pages change nothing."""
    rng = np.random.default_rng(3)
    B, hd, pt, L = 2, 128, 16, 400
    t, pages = make_table(rng, [L] * B, pt)
    k, v = rows(rng, B, L, 1, hd), rows(rng, B, L, 1, hd)
    q = rows(rng, B * 2, 8 * hd)
    outs = []
    for bad in (False, True):
        kk, vv = k.clone(), v.clone()
        if bad:  # positions 300, 301 with window 100 and 3 sinks: rows 3..200 and from 302 on are hidden
            kk[:, 3:201], vv[:, 3:201] = float("nan"), float("nan")
            kk[:, 302:], vv[:, 302:] = float("inf"), float("nan")
        pool = make_pool(jsx, pages, 1, hd, pt)
        jsx.kernels.kv4_append(kk, vv, pool, dev(t), dev([0] * B), tokens_per_seq=L)
        ws = jsx.kernels.kv4_attn_workspace(B, 2, 8, 1, hd, q.device)
        outs.append(jsx.kernels.kv4_attn(q, pool, dev(t), dev([300] * B), hd, ws, tokens_per_seq=2, window=100, sinks=3))
    assert torch.isfinite(outs[0].float()).all()
    assert torch.equal(outs[0], outs[1])


def test_attention_nan_reaches_only_its_rows(jsx, cuda):
    """A NaN that is visible makes its own rows NaN and no others."""
    rng = np.random.default_rng(4)
    t, pages = make_table(rng, [100, 100], 32)
    k, v = rows(rng, 2, 100, 2, 64), rows(rng, 2, 100, 2, 64)
    v[0, 40, 1, 0] = float("nan")
    q = rows(rng, 2, 8 * 64)
    pool = make_pool(jsx, pages, 2, 64, 32)
    jsx.kernels.kv4_append(k, v, pool, dev(t), dev([0, 0]), tokens_per_seq=100)
    ws = jsx.kernels.kv4_attn_workspace(2, 1, 8, 2, 64, q.device)
    o = jsx.kernels.kv4_attn(q, pool, dev(t), dev([99, 99]), 64, ws).float().view(2, 2, 4, 64)
    bad = torch.isnan(o)
    assert bad[0, 1, :, :16].all() and not bad[0, 0].any() and not bad[1].any() and not bad[0, 1, :, 16:].any()


@pytest.mark.parametrize("T,nq,hd", [(2, 8, 128), (5, 16, 128), (4, 4, 64)])
def test_attention_nan_that_only_some_tokens_see(jsx, cuda, T, nq, hd):
    """V rows with a NaN inside one token's window and outside another's, K rows too: the tokens that
    do not see them are as without it, the others NaN in that row's 16 dimensions (V) or all (K)."""
    rng = np.random.default_rng(T)
    L, window, first = 300, 64, 250
    t, pages = make_table(rng, [L], 32)
    k, v = rows(rng, 1, L, 1, hd), rows(rng, 1, L, 1, hd)
    q = rows(rng, T, nq * hd)
    ws = jsx.kernels.kv4_attn_workspace(1, T, nq, 1, hd, q.device)

    def run(kk, vv):
        pool = make_pool(jsx, pages, 1, hd, 32)
        jsx.kernels.kv4_append(kk, vv, pool, dev(t), dev([0]), tokens_per_seq=L)
        o = jsx.kernels.kv4_attn(q, pool, dev(t), dev([first]), hd, ws, tokens_per_seq=T, window=window)
        return o.view(T, nq, hd)

    clean = run(k, v)
    oldest = first - window + 1          # token 0's oldest row: no other token sees it
    newest = first + T - 1               # the last token's own row
    vv = v.clone()
    vv[0, oldest, 0, 17] = float("nan")
    vv[0, newest, 0, 40] = float("nan")
    o = run(k, vv)
    want = torch.zeros(T, nq, hd, dtype=torch.bool, device="cuda")
    want[0, :, 16:32] = True
    want[T - 1, :, 32:48] = True
    assert torch.equal(torch.isnan(o), want) and torch.equal(o[~want], clean[~want])
    kk = k.clone()
    kk[0, newest, 0, 3] = float("nan")
    o = run(kk, v)
    assert torch.isnan(o[T - 1]).all() and torch.equal(o[:T - 1], clean[:T - 1])


def test_attention_missing_pages_and_short_tables(jsx, cuda):
    def holes(t):
        t = t.copy()
        t[0, 1] = -1
        t[1, :] = -1          # nothing left: zeros
        t[2, 0] = 10 ** 6     # not a page
        return t
    rng = np.random.default_rng(8)
    out = attn_case(jsx, rng, 4, 2, 32, 2, 128, 64, [200, 70, 130, 500], table=holes)
    assert (out.view(4, 2, -1)[1] == 0).all()
    attn_case(jsx, rng, 4, 2, 32, 2, 128, 64, [200, 70, 130, 500], table=holes, window=96, sinks=8)


def test_attention_large_scores_and_queries(jsx, cuda):
    """Scores far apart (one weight only), queries near bf16's largest powers, and zero queries."""
    rng = np.random.default_rng(9)
    t, pages = make_table(rng, [300], 64)
    k, v = rows(rng, 1, 300, 1, 128), rows(rng, 1, 300, 1, 128)
    pool = make_pool(jsx, pages, 1, 128, 64)
    jsx.kernels.kv4_append(k, v, pool, dev(t), dev([0]), tokens_per_seq=300)
    kp, vp = R.unpack_pool(pool.cpu().numpy(), 128)
    base = rng.standard_normal((1, 4, 128)).astype(np.float32)
    for gain in (0.0, 2.0 ** -100, 2.0 ** 100):
        q = dev(base * np.float32(gain), BF).reshape(1, -1)
        scale = 1.0 if gain == 0 else 0.05 / gain
        ws = jsx.kernels.kv4_attn_workspace(1, 1, 4, 1, 128, q.device)
        got = f64(jsx.kernels.kv4_attn(q, pool, dev(t), dev([299]), 128, ws, scale=scale)).reshape(1, 4, 128)
        want, big = R.attention(f64(q).reshape(1, 4, 128), kp, vp, t, [299], 1, scale=scale)
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * big).all(), gain
    q = dev(base * 64, BF).reshape(1, -1)      # scores hundreds apart
    got = f64(jsx.kernels.kv4_attn(q, pool, dev(t), dev([299]), 128, ws, scale=1.0)).reshape(1, 4, 128)
    want, big = R.attention(f64(q).reshape(1, 4, 128), kp, vp, t, [299], 1, scale=1.0)
    # a score of ~5000 has an fp32 error of about 128 x 2^-22 x its terms: up to 2^-3 in the exponent
    top = np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -2 * big
    assert np.isfinite(got).all() and top.all()


@pytest.mark.parametrize("B,T,nq,nkv,L", [(1, 1, 32, 2, 20000), (2, 1, 4, 1, 9000), (3, 6, 32, 2, 5000), (40, 1, 8, 1, 1500)])
def test_attention_long_and_unequal(jsx, cuda, B, T, nq, nkv, L):
    """One long sequence among short ones: work split over many CTAs and joined."""
    rng = np.random.default_rng(L)
    positions = [L - 1 if b == 0 else int(rng.integers(0, max(2, L // 20))) for b in range(B)]
    attn_case(jsx, rng, B, T, nq, nkv, 128, 64, positions)


# ---- many query rows: a table with room for long sequences takes the kernel of 128-row items ----


@pytest.mark.parametrize("T,nq,nkv,pt,counts", [(4, 32, 2, 64, False), (5, 32, 2, 128, False), (7, 14, 2, 32, False),
                                                (8, 16, 1, 16, False), (16, 32, 2, 64, True), (33, 12, 4, 32, True),
                                                (70, 16, 1, 64, True), (300, 1, 1, 16, False)])
def test_attention_many_rows(jsx, cuda, T, nq, nkv, pt, counts):
    rng = np.random.default_rng(T + nq)
    positions = [0, 60, 331, -T + 1, -T]
    attn_case(jsx, rng, 5, T, nq, nkv, 128, pt, positions, n_tokens=[T, T - 1, T, 0, T] if counts else None,
              slots=2 ** 18 // pt)


@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 5), (130, 200), (1000, 3)])
def test_attention_many_rows_window_and_sinks(jsx, cuda, window, sinks):
    rng = np.random.default_rng(window)
    attn_case(jsx, rng, 4, 240, 16, 2, 128, 32, [0, 63, 300, 777], window=window, sinks=sinks, slots=512)


@pytest.mark.parametrize("B,T,nq,nkv,L", [(3, 8, 32, 2, 5000), (2, 16, 16, 1, 9000), (1, 64, 32, 2, 2000)])
def test_attention_many_rows_long_and_unequal(jsx, cuda, B, T, nq, nkv, L):
    """The same item's records of many CTAs, long sequences in few of them."""
    rng = np.random.default_rng(L)
    positions = [L - 1 if b == 0 else int(rng.integers(0, max(2, L // 20))) for b in range(B)]
    attn_case(jsx, rng, B, T, nq, nkv, 128, 64, positions, slots=4096)


def test_attention_many_rows_missing_pages(jsx, cuda):
    def holes(t):
        t = t.copy()
        t[0, 1] = -1
        t[1, :] = -1          # nothing left: zeros
        t[2, 0] = 10 ** 6     # not a page
        return t
    rng = np.random.default_rng(8)
    out = attn_case(jsx, rng, 4, 8, 32, 2, 128, 16, [200, 70, 130, 500], table=holes, slots=2048)
    assert (out.view(4, 8, -1)[1] == 0).all()


def test_attention_many_rows_nan_that_only_some_tokens_see(jsx, cuda):
    """V rows with a NaN that the later tokens see, a K row with one that the last token sees."""
    rng = np.random.default_rng(16)
    T, nq, first, pt = 16, 16, 250, 32
    t, pages = make_table(rng, [300], pt, 2 ** 18 // pt)
    k, v = rows(rng, 1, 300, 1, 128), rows(rng, 1, 300, 1, 128)
    q = rows(rng, T, nq * 128)
    ws = jsx.kernels.kv4_attn_workspace(1, T, nq, 1, 128, q.device)

    def run(kk, vv):
        pool = make_pool(jsx, pages, 1, 128, pt)
        jsx.kernels.kv4_append(kk, vv, pool, dev(t), dev([0]), tokens_per_seq=300)
        return jsx.kernels.kv4_attn(q, pool, dev(t), dev([first]), 128, ws, tokens_per_seq=T).view(T, nq, 128)

    clean = run(k, v)
    assert torch.isfinite(clean.float()).all()
    vv = v.clone()
    vv[0, first + 3, 0, 17] = float("nan")
    vv[0, first + 10, 0, 127] = float("nan")
    vv[0, first + T, 0, 64] = float("nan")      # after the last token: no one's
    o = run(k, vv)
    want = torch.zeros(T, nq, 128, dtype=torch.bool, device="cuda")
    want[3:, :, 16:32] = True
    want[10:, :, 112:] = True
    assert torch.equal(torch.isnan(o), want) and torch.equal(o[~want], clean[~want])
    assert torch.equal(run(k, v), clean)        # and nothing of it stays
    kk = k.clone()
    kk[0, first + T - 1, 0, 3] = float("nan")
    o = run(kk, v)
    assert torch.isnan(o[T - 1]).all() and torch.equal(o[:T - 1], clean[:T - 1])


@pytest.mark.parametrize("T,nq", [(1, 4), (4, 16)])
def test_attention_many_sequences(jsx, cuda, T, nq):
    """More sequences than the list of chunks is kept for: whole items per CTA."""
    rng = np.random.default_rng(T)
    positions = [int(x) for x in rng.integers(-T, 300, 600)]
    attn_case(jsx, rng, 600, T, nq, 1, 128, 32, positions, slots=16)


def test_attention_workspace_of_the_largest_call(jsx, cuda):
    """One workspace, calls of several shapes in turn: each as with a workspace of its own."""
    rng = np.random.default_rng(21)
    B, hd, pt = 3, 128, 64
    t, pages = make_table(rng, [3000] * B, pt, 2048)
    pool = make_pool(jsx, pages, 2, hd, pt)
    k, v = rows(rng, B, 3000, 2, hd), rows(rng, B, 3000, 2, hd)
    jsx.kernels.kv4_append(k, v, pool, dev(t), dev([0] * B), tokens_per_seq=3000)
    tab, pos = dev(t), dev([2900, 17, 1500])
    shared = jsx.kernels.kv4_attn_workspace(B, 16, 32, 2, hd, pool.device)
    for T in (16, 1, 8, 2, 16, 1):
        q = rows(rng, B * T, 32 * hd)
        own = jsx.kernels.kv4_attn_workspace(B, T, 32, 2, hd, pool.device)
        assert own.numel() <= shared.numel()
        a = jsx.kernels.kv4_attn(q, pool, tab, pos, hd, own, tokens_per_seq=T)
        assert torch.equal(a, jsx.kernels.kv4_attn(q, pool, tab, pos, hd, shared, tokens_per_seq=T))


def test_attention_strided_queries_another_stream_and_graph(jsx, cuda):
    rng = np.random.default_rng(11)
    B, T, nq, nkv, hd, pt = 4, 2, 8, 2, 128, 32
    t, pages = make_table(rng, [500] * B, pt)
    pool = make_pool(jsx, pages, nkv, hd, pt)
    k, v = rows(rng, B, 500, nkv, hd), rows(rng, B, 500, nkv, hd)
    jsx.kernels.kv4_append(k, v, pool, dev(t), dev([0] * B), tokens_per_seq=500)
    wide = rows(rng, B * T, (nq + 2 * nkv) * hd)
    q = wide[:, :nq * hd]
    ws = jsx.kernels.kv4_attn_workspace(B, T, nq, nkv, hd, q.device)
    tab, pos = dev(t), dev([400, 17, 250, 498])
    a = jsx.kernels.kv4_attn(q.contiguous(), pool, tab, pos, hd, ws, tokens_per_seq=T)
    out = torch.zeros(B * T, 2 * nq * hd, dtype=BF, device="cuda")
    jsx.kernels.kv4_attn(q, pool, tab, pos, hd, ws, tokens_per_seq=T, out=out[:, nq * hd:])
    assert torch.equal(a, out[:, nq * hd:]) and (out[:, :nq * hd] == 0).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = jsx.kernels.kv4_attn(q, pool, tab, pos, hd, ws, tokens_per_seq=T)
    s.synchronize()
    assert torch.equal(a, c)
    g = torch.cuda.CUDAGraph()
    y = torch.empty_like(a)
    with torch.cuda.graph(g):
        jsx.kernels.kv4_attn(q, pool, tab, pos, hd, ws, tokens_per_seq=T, out=y)
    pos.copy_(dev([300, 60, 1, 77]))           # lengths are read on the device at replay
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, jsx.kernels.kv4_attn(q, pool, tab, pos, hd, ws, tokens_per_seq=T))


def test_offsets_past_32_bits(jsx, cuda):
    """Pages more than 4 GiB into the pool."""
    nkv, hd, pt = 8, 128, 128
    n = (1 << 32) // jsx.kernels.kv4_page_bytes(nkv, hd, pt) + 4
    pool = make_pool(jsx, n, nkv, hd, pt)
    rng = np.random.default_rng(2)
    t = np.array([[n - 1, n - 3, 0]], np.int32)
    k, v = rows(rng, 1, 300, nkv, hd), rows(rng, 1, 300, nkv, hd)
    jsx.kernels.kv4_append(k, v, pool, dev(t), dev([0]), tokens_per_seq=300)
    q = rows(rng, 1, 16 * hd)
    ws = jsx.kernels.kv4_attn_workspace(1, 1, 16, nkv, hd, q.device)
    got = f64(jsx.kernels.kv4_attn(q, pool, dev(t), dev([299]), hd, ws)).reshape(1, 16, hd)
    few = pool[dev(t[0], torch.int64)].cpu().numpy()
    kp, vp = R.unpack_pool(few, hd)
    want, big = R.attention(f64(q).reshape(1, 16, hd), kp, vp, np.array([[0, 1, 2]]), [299], 1)
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * big).all()


def test_python_refusals(jsx, cuda):
    K = jsx.kernels
    pool = make_pool(jsx, 4, 2, 128, 16)
    t, pos = dev([[0, 1]]), dev([0])
    k = torch.zeros(2, 2, 128, dtype=BF, device="cuda")
    q = torch.zeros(1, 4 * 128, dtype=BF, device="cuda")
    ws = K.kv4_attn_workspace(1, 1, 4, 2, 128, q.device)
    for bad in (lambda: K.kv4_append(k, k, pool, t, pos),                                  # two rows for one token
                lambda: K.kv4_append(k.float(), k.float(), pool, t, pos, tokens_per_seq=2),
                lambda: K.kv4_append(k[:, :1], k[:, :1], pool, t, pos, tokens_per_seq=2),  # one head of two
                lambda: K.kv4_append(k, k, pool, t.long(), pos, tokens_per_seq=2),
                lambda: K.kv4_append(k, k, pool, t, dev([0, 0]), tokens_per_seq=2),
                lambda: K.kv4_append(k.cpu(), k.cpu(), pool, t, pos, tokens_per_seq=2),
                lambda: K.kv4_attn(q[:, :100], pool, t, pos, 128, ws),
                lambda: K.kv4_attn(q, pool, t, pos, 96, ws),
                lambda: K.kv4_attn(q.float(), pool, t, pos, 128, ws)):
        with pytest.raises((ValueError, TypeError)):
            bad()
    for bad in (lambda: K.kv4_attn(q[:, :3 * 128].contiguous(), pool, t, pos, 128, ws),    # 3 heads over 2
                lambda: K.kv4_attn(q, pool, t, pos, 128, ws[:16]),
                lambda: K.kv4_attn(q, pool, t, pos, 128, ws, window=-1)):
        with pytest.raises(jsx._lib.JsxError) as e:
            bad()
        assert e.value.status == jsx._lib.JSX_EINVAL
