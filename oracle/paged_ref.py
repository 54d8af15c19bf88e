"""Oracle of the paged 4-bit cache and of draft verification, in numpy and 64 bits.

Written from the definitions in include/jsx.h: rows quantised to e2m1 codes with one e4m3
scale per 16 values, attention over pages with a window and sinks, page bookkeeping done
one sequence after the other, and verification by exact integer weights.
"""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values() -> np.ndarray:
    """Values of the 128 non-negative e4m3 codes (the last is NaN)."""
    c = np.arange(128)
    e, m = c >> 3, c & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[127] = np.nan
    return v


def _nearest_even(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest to x >= 0 (ties: even index), saturating."""
    hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
    lo = hi - 1
    a, b = x - grid[lo], grid[hi] - x
    pick_hi = (b < a) | ((b == a) & (hi % 2 == 0))
    return np.where(x >= grid[-1], len(grid) - 1, np.where(pick_hi, hi, lo))


def quantise(rows: np.ndarray):
    """rows [..., D] -> (codes [..., D] 0..15, scale codes [..., D / 16])."""
    x = np.asarray(rows, np.float64).reshape(*rows.shape[:-1], -1, 16)
    top = np.max(np.abs(x), axis=-1)  # NaN propagates
    grid = e4m3_values()[:127]
    with np.errstate(invalid="ignore"):
        sc = _nearest_even(np.minimum(np.where(np.isnan(top), 0, top) / 6, 448.0), grid)
        sc = np.where(np.isnan(top), 127, sc)
        s = e4m3_values()[sc][..., None]
        q = np.where((s > 0) & np.isfinite(x), np.abs(x) / np.where(s > 0, s, 1), np.where(np.isinf(x), 6.0, 0.0))
    code = _nearest_even(np.where(np.isnan(q), 0, q), E2M1)
    code = np.where((x < 0) & (code > 0), code + 8, code)
    return code.reshape(rows.shape), sc


def dequantise(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    v = np.where(codes > 7, -E2M1[codes & 7], E2M1[codes & 7]).reshape(*scales.shape, 16)
    return (v * e4m3_values()[scales][..., None]).reshape(codes.shape)


def stored(rows: np.ndarray) -> np.ndarray:
    """What a row reads back as."""
    return dequantise(*quantise(rows))


def unpack_pool(pool: np.ndarray, D: int):
    """uint8 pool [P, nkv, block] -> (K, V) values [P, nkv, pt, D]."""
    P, nkv, block = pool.shape
    pt = block * 8 // (9 * D)
    a, b = pt * D // 2, pt * D // 16
    out = []
    for w in (0, 1):
        c = pool[..., w * a:(w + 1) * a].reshape(P, nkv, pt, D // 2)
        codes = np.stack([c & 15, c >> 4], -1).reshape(P, nkv, pt, D).astype(np.int64)
        s = pool[..., 2 * a + w * b:2 * a + (w + 1) * b].reshape(P, nkv, pt, D // 16).astype(np.int64)
        out.append(np.where(s[..., None] > 127, -1, 1).repeat(16, -1).reshape(codes.shape) * dequantise(codes, s & 127))
    return out[0], out[1]


def attention(q, k_pages, v_pages, table, positions, T, window=0, sinks=0, scale=None, n_tokens=None):
    """q [B * T, nq, D]; k_pages, v_pages [P, nkv, pt, D] values -> (out [B * T, nq, D],
    largest |v| that each row sees)."""
    BT, nq, D = q.shape
    P, nkv, pt, _ = k_pages.shape
    G = nq // nkv
    scale = D ** -0.5 if scale is None else scale
    out, big = np.zeros((BT, nq, D)), np.zeros((BT, nq, 1))
    for r in range(BT):
        b, i = divmod(r, T)
        p = int(positions[b]) + i
        if (n_tokens is not None and i >= n_tokens[b]) or p < 0:
            continue
        j = np.arange(min(p + 1, table.shape[1] * pt))
        page = table[b][j // pt]
        see = (page >= 0) & (page < P)
        if window:
            see &= (j > p - window) | (j < sinks)
        j, page = j[see], page[see]
        if not len(j):
            continue
        for h in range(nq):
            k, v = k_pages[page, h // G, j % pt], v_pages[page, h // G, j % pt]
            s = scale * (k @ np.asarray(q[r, h], np.float64))
            w = np.exp(s - s.max())
            out[r, h] = (w / w.sum()) @ v
            big[r, h] = np.abs(v).max()
    return out, big


# ---- pages ----
def pages_fork(table, held, refs, parent):
    S = len(held)
    t, h, r = np.full_like(table, -1), np.zeros_like(held), refs.copy()
    for b in range(S):
        for p in table[b, :held[b]]:
            r[p] -= 1
    for b in range(S):
        if 0 <= parent[b] < S:
            h[b] = held[parent[b]]
            t[b, :h[b]] = table[parent[b], :h[b]]
            for p in t[b, :h[b]]:
                r[p] += 1
    return t, h, r


def pages_resize(table, held, refs, keep, need, page_tokens):
    """(table, held, refs, copies [(from, to)], missing)."""
    t, h, r = table.copy(), held.copy(), refs.copy()
    S, slots = table.shape
    free = [p for p in range(len(refs)) if refs[p] == 0]
    copies, used, over = [], 0, 0
    give_back = []
    for b in range(S):
        nd = max(int(need[b]), 0)
        kp = min(max(int(keep[b]), 0), nd, int(h[b]) * page_tokens)
        n = -(-nd // page_tokens)
        over += max(n - slots, 0)
        n = min(n, slots)
        for i in range(kp // page_tokens, n):
            old = int(t[b, i]) if i < h[b] else -1
            if i < h[b] and old >= 0 and refs[old] <= 1:
                continue
            new = free[used] if used < len(free) else None
            used += 1
            if new is None:
                continue
            t[b, i] = new
            r[new] = 1
            if old >= 0:
                give_back.append(old)
                if i * page_tokens < kp:
                    copies.append((old, new))
        for i in range(n, int(h[b])):
            give_back.append(int(t[b, i]))
            t[b, i] = -1
        h[b] = n
    missing = max(used - len(free), 0) + over
    if missing:
        return table.copy(), held.copy(), refs.copy(), [], missing
    for p in give_back:
        r[p] -= 1
    return t, h, r, copies, 0


def pages_compact(table, held, refs):
    """(table, refs, remap, moves [(from, to)])."""
    live = [p for p in range(len(refs)) if refs[p] > 0]
    n = len(live)
    moves = list(zip([p for p in live if p >= n], [p for p in range(n) if refs[p] <= 0]))
    remap = np.where(refs > 0, np.arange(len(refs)), -1).astype(refs.dtype)
    r = np.where(refs > 0, refs, 0).astype(refs.dtype)
    for a, b in moves:
        remap[a] = b
        r[b], r[a] = refs[a], 0
    t = np.full_like(table, -1)
    for b in range(len(held)):
        for i in range(held[b]):
            p = table[b, i]
            t[b, i] = remap[p] if 0 <= p < len(refs) else -1
    return t, r, remap, moves


# ---- drafted tokens ----
def _weights(row, inv_temp):
    """Integer weights of one row of logits (float32 products, 64-bit exponentials; products in
    64 bits where the largest logit's is finite only there)."""
    with np.errstate(invalid="ignore", over="ignore"):
        row = np.where(np.isnan(row), -np.inf, row).astype(np.float32)
        if not np.isfinite(row.max()):
            return None
        x = (row * np.float32(inv_temp)).astype(np.float64)
        if not np.isfinite(x.max()):
            x = row.astype(np.float64) * np.float64(inv_temp)
        m = x.max()
        return np.floor(np.exp(x - m) * 2.0 ** 40).astype(np.int64)


def verify(logits, ids, uniforms, probs=None, n_draft=None, temperature=1.0):
    """(accepted, tokens, accept_prob, margin): margin[b] is how near the sequence's decisions
    come to a boundary (relative, of an acceptance or of the draw's running sum)."""
    B, T1, V = logits.shape
    T = T1 - 1
    acc, tok, pr = np.zeros(B, np.int32), np.full((B, T1), -1, np.int32), np.zeros((B, T))
    margin = np.full(B, np.inf)
    inv = np.float32(1) / np.float32(temperature) if temperature else 0
    for b in range(B):
        nd = T if n_draft is None else min(max(int(n_draft[b]), 0), T)
        if temperature == 0:
            x = np.where(np.isnan(logits[b].astype(np.float64)), -np.inf, logits[b].astype(np.float64))
            best = [int(np.argmax(r)) if r.max() > -np.inf else -1 for r in x]
            for i in range(nd):
                pr[b, i] = float(ids[b, i] == best[i])
            n = 0
            while n < nd and ids[b, n] == best[n]:
                n += 1
            tok[b, :n], tok[b, n], acc[b] = ids[b, :n], best[n], n
            continue
        w = [_weights(logits[b, i], inv) for i in range(T1)]
        ok = []
        for i in range(nd):
            x = int(ids[b, i])
            if not 0 <= x < V:
                ok.append(False)
                continue
            p = 0.0 if w[i] is None else w[i][x] / w[i].sum()
            q = 1.0 if probs is None else float(probs[b, i, x])
            pr[b, i] = min(1.0, p / q) if q > 0 else float(p > 0)
            ok.append(float(uniforms[b, i]) * q < p)
            if all(ok[:-1]) and p > 0:
                margin[b] = min(margin[b], abs(float(uniforms[b, i]) * q / p - 1))
        n = ok.index(False) if False in ok else nd
        acc[b], tok[b, :n] = n, ids[b, :n]
        if w[n] is None:
            continue
        left = w[n]
        if n < nd:
            if probs is None:
                left = left.copy()
                if 0 <= ids[b, n] < V:
                    left[ids[b, n]] = 0
            else:
                q = probs[b, n].astype(np.float64)
                d = w[n] / w[n].sum() - q
                left = np.floor(np.where(d > 0, d, 0) * 2.0 ** 40).astype(np.int64)
            if left.sum() == 0:
                left = w[n]
        total = int(left.sum())
        u = float(uniforms[b, T])
        k = total * int(min(max(u * 2 ** 24, 0), 2 ** 24 - 1)) >> 24
        run = np.cumsum(left)
        tok[b, n] = int(np.searchsorted(run, k, side="right"))
        margin[b] = min(margin[b], np.abs(run - k).min() / total)
    return acc, tok, pr, margin
