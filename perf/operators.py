"""Drafted decoding over a paged 4-bit key/value cache: the cases it is measured on.

Four operators: rows written to and read back from the cache's pages ("store"), attention over the
pages with a sliding window and first tokens that stay visible ("attn"), sharing, copying and moving
pages ("fork", "compact"), and the check of drafted tokens against the target's distribution ("verify").

A page holds `pt` tokens of every kv head; for one head it is
    K codes [pt][hd / 2] | V codes [pt][hd / 2] | K scales [pt][hd / 16] | V scales [pt][hd / 16]
with two e2m1 codes per byte (the even dimension in the low half) and one e4m3 scale per 16 values.
"""

import importlib
import math

import numpy as np
import torch

own = False

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FIX = float(2 ** 40)  # fixed-point unit of the verification's weights


def listed():
    return [
        # one user's decode step at a short context: 1025 cache rows, the model's 32 query and 2 kv heads
        dict(name="attn 1x1025", op="attn", B=1, T=1, nq=32, nkv=2, hd=128, pt=64, L=1025, ragged=False, window=0, sinks=0, part=False),
        # a decode step of a full batch at long, unequal contexts: the cache is what is read
        dict(name="attn 32x32768", op="attn", B=32, T=1, nq=32, nkv=2, hd=128, pt=64, L=32768, ragged=True, window=0, sinks=0, part=False),
        # a drafted step: the last token and up to four drafted ones per sequence, some sequences with fewer
        dict(name="attn 16x8191 drafted", op="attn", B=16, T=5, nq=32, nkv=2, hd=128, pt=64, L=8191, ragged=True, window=0, sinks=0, part=True),
        # one rank of four (8 query heads, 1 kv head), long streams that see 4 first and the last 4096 tokens
        dict(name="attn 64x60001 window", op="attn", B=64, T=1, nq=8, nkv=1, hd=128, pt=32, L=60001, ragged=True, window=4096, sinks=4, part=False),
        # the new rows of one decode step of 32 sequences, one layer
        dict(name="store 32x1", op="store", B=32, T=1, nkv=2, hd=128, pt=64, start=1000, static=False),
        # a block of prompts, one layer, from the static cache into pages, and back as the next block's prefix
        dict(name="store 32x1024", op="store", B=32, T=1024, nkv=2, hd=128, pt=64, start=0, static=True),
        # one prompt continued four ways, ten layers
        dict(name="fork 1 into 4", op="fork", S=4, src=1, layers=10, nkv=2, hd=128, pt=64, L=1000, T=5),
        # eight prompts continued eight ways each, all forty layers: every child copies its last page
        dict(name="fork 8 into 64", op="fork", S=64, src=8, layers=40, nkv=2, hd=128, pt=64, L=2100, T=5),
        # a pool of 4096 pages, a quarter of whose live pages sit above the others' holes
        dict(name="compact 4096 pages", op="compact", S=64, P=4096, live=2000, moves=500, layers=40, nkv=2, hd=128, pt=64),
        # one user's step, four tokens proposed by looking the prompt up (no draft distribution)
        dict(name="verify 1x4", op="verify", B=1, T=4, V=151552, probs=False, temp=1.0, wide=False, part=False),
        # a full batch with a drafting model's distributions
        dict(name="verify 32x4 probs", op="verify", B=32, T=4, V=151552, probs=True, temp=0.8, wide=False, part=True),
        # greedy decoding with long drafts over an odd vocabulary, logits in 32 bits
        dict(name="verify 16x7 greedy", op="verify", B=16, T=7, V=32003, probs=False, temp=0.0, wide=True, part=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attn", "attn", "store", "fork", "compact", "verify"])
    if op == "attn":
        nq, nkv = rng.choice([(32, 2), (16, 1), (8, 1), (4, 1), (32, 8), (14, 2), (12, 12)])
        T = rng.choice([1, 1, 2, 3, 5, 8])
        L = log(1, 32768)
        B = min(log(1, 64), max(1, (1 << 21) // (L * nkv)))
        window = rng.choice([0, 0, log(16, 8192)])
        return dict(op="attn", B=B, T=T, nq=nq, nkv=nkv, hd=rng.choice([64, 128, 128]), pt=rng.choice([16, 32, 64, 128]), L=L,
                    ragged=rng.random() < 0.7, window=window, sinks=rng.choice([0, 1, 4, 70]) if window else 0, part=T > 1 and rng.random() < 0.5)
    if op == "store":
        T = log(1, 2048)
        return dict(op="store", B=min(log(1, 64), max(1, 32768 // T)), T=T, nkv=rng.choice([1, 2, 2, 8]) if T < 1024 else rng.choice([1, 2]), hd=rng.choice([64, 128, 128]),
                    pt=rng.choice([16, 32, 64, 128]), start=log(1, 5000), static=rng.random() < 0.5)
    if op == "fork":
        S = log(2, 64)
        return dict(op="fork", S=S, src=max(1, S // rng.choice([2, 4, 8])), layers=log(2, 40), nkv=rng.choice([1, 2]), hd=128, pt=rng.choice([16, 32, 64]), L=log(10, 2100), T=rng.randint(1, 9))
    if op == "compact":
        P = log(64, 4096)
        live = max(8, int(P * rng.uniform(0.2, 0.6)))
        return dict(op="compact", S=log(2, 64), P=P, live=live, moves=min(500, max(1, int(live * rng.uniform(0.05, 0.4)))), layers=log(2, 40), nkv=rng.choice([1, 2]), hd=128, pt=rng.choice([16, 32, 64]))
    T = rng.randint(1, 8)
    V = log(1000, 151552)
    return dict(op="verify", B=min(log(1, 64), max(1, 24_000_000 // (V * (T + 1)))), T=T, V=V, probs=rng.random() < 0.5, temp=rng.choice([0.0, 0.7, 1.0, 1.3]), wide=rng.random() < 0.3, part=rng.random() < 0.5)


# ---- sizes that follow from a case alone ------------------------------------------------------------
def _lengths(n, L, ragged):
    """Tokens of each of n sequences: L, or spread from about a quarter of it up to it."""
    return [max(1, int(L * (0.25 + 0.75 * ((0.618034 * (b + 1)) % 1.0)))) if ragged and b else L for b in range(n)]


def _counts(n, most, part):
    """How many of its `most` tokens each sequence uses."""
    return [most - (5 * b + b // 3) % most if part else most for b in range(n)]


def _page_bytes(c):
    return c["nkv"] * c["pt"] * c["hd"] * 9 // 8


def _fork_sizes(c):
    lens = _lengths(c["src"], c["L"], True)
    parent = [b if b < c["src"] else (b - c["src"]) % c["src"] for b in range(c["S"])]
    keep = [lens[p] for p in parent]
    need = [n + c["T"] for n in keep]
    slots = -(-(c["L"] + c["T"]) // c["pt"])
    pages = sum(-(-n // c["pt"]) for n in lens)
    shared = {p for p in parent if parent.count(p) > 1}
    fresh = copied = 0
    for b, p in enumerate(parent):
        held = -(-keep[b] // c["pt"])
        fresh += -(-need[b] // c["pt"]) - held
        copied += int(p in shared and keep[b] % c["pt"] != 0)
    return lens, parent, keep, need, slots, pages, pages + fresh + copied + 7, copied


def work(c):
    if c["op"] == "attn":
        pos, used = [n - c["T"] for n in _lengths(c["B"], c["L"] + c["T"] - 1, c["ragged"])], _counts(c["B"], c["T"], c["part"])
        rows = seen = 0
        for p, n in zip(pos, used):
            union = set()
            for i in range(n):
                hi = p + i + 1
                if hi <= 0:
                    continue
                lo = max(0, hi - c["window"]) if c["window"] else 0
                seen += hi - lo + min(lo, c["sinks"])
                union |= {("k", lo, hi)}
            if union:
                lo, hi = min(u[1] for u in union), max(u[2] for u in union)
                rows += hi - lo + min(lo, c["sinks"])
        bytes_ = rows * c["nkv"] * c["hd"] * 9 / 8 + sum(used) * c["nq"] * c["hd"] * 4
        return {"bytes": bytes_, "flops": 4.0 * seen * c["nq"] * c["hd"]}
    if c["op"] == "store":
        n = c["B"] * c["T"] * c["nkv"] * c["hd"] * 2
        return {"bytes": n * 2 * 2 + n * 2 * 9 / 16, "flops": 0.0}
    if c["op"] == "fork":
        _, _, _, _, slots, _, P, copied = _fork_sizes(c)
        return {"bytes": 2.0 * copied * c["layers"] * _page_bytes(c) + 8.0 * c["S"] * slots + 8.0 * P, "flops": 0.0}
    if c["op"] == "compact":
        return {"bytes": 2.0 * c["moves"] * c["layers"] * _page_bytes(c) + 8.0 * c["live"] + 12.0 * c["P"], "flops": 0.0}
    row = c["V"] * (4 if c["wide"] else 2)
    return {"bytes": float(c["B"] * ((c["T"] + 1) * row + (c["V"] * 4 if c["probs"] else 0))), "flops": 0.0}


# ---- inputs ------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, *shape):
    """Rows of keys or values: near normal, with some dimensions of a head several times larger than the others."""
    x = torch.randn(*shape, generator=g, device="cuda")
    gain = 1.0 + 5.0 * (torch.rand(shape[-2:], generator=g, device="cuda") > 0.95).float()
    return (x * gain).to(torch.bfloat16)


def _table(g, lens, pt, spare):
    """Pages of each sequence in a scattered order."""
    n = [-(-x // pt) for x in lens]
    order = torch.randperm(sum(n) + spare, generator=g, device="cuda").to(torch.int32)
    slots = torch.arange(max(n), device="cuda")
    n_dev = torch.tensor(n, device="cuda")
    first = torch.cumsum(n_dev, 0) - n_dev
    at = first[:, None] + slots[None]
    return torch.where(slots[None] < n_dev[:, None], order[at.clamp(max=sum(n) - 1)], -1).to(torch.int32).contiguous(), sum(n) + spare


def prepare(c, seed):
    g = _gen(seed)
    s = dict(c)
    if c["op"] == "attn":
        lens = _lengths(c["B"], c["L"] + c["T"] - 1, c["ragged"])
        s["table"], pages = _table(g, lens, c["pt"], 3)
        s["positions"] = torch.tensor([n - c["T"] for n in lens], dtype=torch.int32, device="cuda")
        s["n_tokens"] = torch.tensor(_counts(c["B"], c["T"], True), dtype=torch.int32, device="cuda") if c["part"] else None
        s["q"] = torch.randn(c["B"] * c["T"], c["nq"] * c["hd"], generator=g, device="cuda").to(torch.bfloat16)
        s["scale"] = c["hd"] ** -0.5
        pool = torch.empty(pages, c["nkv"], _page_bytes(c) // c["nkv"], dtype=torch.uint8, device="cuda")
        at = 0
        step = max(1, 1 << 26 >> int(math.log2(c["nkv"] * c["pt"] * c["hd"])))
        while at < pages:
            n = min(step, pages - at)
            _pack(pool[at:at + n], *(_rows(g, n, c["pt"], c["nkv"], c["hd"]).transpose(1, 2) for _ in "kv"))
            at += n
        s["pool"] = pool
    elif c["op"] == "store":
        lens = [c["start"] + c["T"]] * c["B"]
        s["table"], pages = _table(g, lens, c["pt"], 3)
        s["positions"] = torch.full((c["B"],), c["start"], dtype=torch.int32, device="cuda")
        s["pool"] = torch.zeros(pages, c["nkv"], _page_bytes(c) // c["nkv"], dtype=torch.uint8, device="cuda")
        shape = (c["B"], lens[0], c["nkv"], c["hd"]) if c["static"] else (c["B"] * c["T"], c["nkv"], c["hd"])
        s["k"], s["v"] = _rows(g, *shape), _rows(g, *shape)
        s["k_out"], s["v_out"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
    elif c["op"] == "fork":
        lens, parent, keep, need, slots, pages, P, _ = _fork_sizes(c)
        table, _ = _table(g, lens, c["pt"], P - pages)
        s["table"] = torch.full((c["S"], slots), -1, dtype=torch.int32, device="cuda")
        s["table"][: c["src"], : table.shape[1]] = table
        s["held"] = torch.tensor([-(-n // c["pt"]) for n in lens] + [0] * (c["S"] - c["src"]), dtype=torch.int32, device="cuda")
        s["refs"] = torch.zeros(P, dtype=torch.int32, device="cuda")
        s["refs"][table[table >= 0].long()] = 1
        for name, v in (("parent", parent), ("keep", keep), ("need", need)):
            s[name] = torch.tensor(v, dtype=torch.int32, device="cuda")
        s["pool"] = torch.randint(0, 256, (c["layers"], P, c["nkv"], _page_bytes(c) // c["nkv"]), dtype=torch.uint8, generator=g, device="cuda")
    elif c["op"] == "compact":
        low = torch.randperm(c["live"], generator=g, device="cuda")[: c["live"] - c["moves"]]
        high = c["live"] + torch.randperm(c["P"] - c["live"], generator=g, device="cuda")[: c["moves"]]
        live = torch.cat([low, high])
        live = live[torch.randperm(c["live"], generator=g, device="cuda")].to(torch.int32)
        s["refs"] = torch.zeros(c["P"], dtype=torch.int32, device="cuda")
        s["refs"][live.long()] = 1
        per = -(-c["live"] // c["S"])
        pad = torch.full((per * c["S"],), -1, dtype=torch.int32, device="cuda")
        pad[: c["live"]] = live
        s["table"] = pad.view(c["S"], per).contiguous()
        s["held"] = (s["table"] >= 0).sum(1).to(torch.int32)
        s["pool"] = torch.randint(0, 256, (c["layers"], c["P"], c["nkv"], _page_bytes(c) // c["nkv"]), dtype=torch.uint8, generator=g, device="cuda")
    else:
        B, T, V = c["B"], c["T"], c["V"]
        logits = torch.randn(B, T + 1, V, generator=g, device="cuda") * 2.5
        logits = logits.to(torch.float32 if c["wide"] else torch.bfloat16)
        near = logits[:, :T].float() + 0.3 * torch.randn(B, T, V, generator=g, device="cuda")
        probs = torch.softmax(near / (c["temp"] or 1.0), -1)
        ids = torch.multinomial(probs.view(B * T, V), 1, generator=g).view(B, T)
        best = logits[:, :T].float().argmax(-1)
        lucky = torch.rand(B, T, generator=g, device="cuda") < 0.7
        s["logits"] = logits
        s["draft_ids"] = (ids if c["probs"] else torch.where(lucky, best, ids)).to(torch.int32)
        s["draft_probs"] = probs.contiguous() if c["probs"] else None
        s["n_draft"] = torch.tensor(_counts(B, T, True), dtype=torch.int32, device="cuda") if c["part"] else None
        s["uniforms"] = torch.rand(B, T + 1, generator=g, device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------------
def _parts(block, hd):
    """K codes, V codes, K scales, V scales of blocks [..., pt * hd * 9 / 8]."""
    pt = block.shape[-1] * 8 // (9 * hd)
    a, b = pt * hd // 2, pt * hd // 16
    lead = block.shape[:-1]
    cut = block[..., :a], block[..., a:2 * a], block[..., 2 * a:2 * a + b], block[..., 2 * a + b:]
    return tuple(x.unflatten(-1, (pt, w)) for x, w in zip(cut, (hd // 2, hd // 2, hd // 16, hd // 16)))


def _quantise(x):
    """(codes, scales) of rows [..., hd]."""
    x = x.float().unflatten(-1, (-1, 16))
    top = x.abs().amax(-1, keepdim=True)
    # divided by a tensor: a division by a number is a product with its rounded inverse, which loses the ties
    scale = (top / torch.full_like(top, 6.0)).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float()
    m = torch.where(s == 0, torch.zeros_like(x), x.abs() / s)
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = (code | ((x < 0).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """Rows in 32 bits."""
    codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    x = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)[codes.int()]
    return (x.unflatten(-1, (-1, 16)) * scales.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _pack(pool, k, v):
    """Quantises whole blocks: k and v [pages, nkv, pt, hd]."""
    kc, vc, ks, vs = _parts(pool, k.shape[-1])
    for dst_c, dst_s, x in ((kc, ks, k), (vc, vs, v)):
        codes, scales = _quantise(x)
        dst_c.copy_(codes)
        dst_s.copy_(scales)


def _plain_attn(s):
    B, T, nkv, hd, pt = s["B"], s["T"], s["nkv"], s["hd"], s["pt"]
    G = s["nq"] // nkv
    kc, vc, ks, vs = (x.transpose(1, 2).flatten(2, 3) for x in _parts(s["pool"][s["table"].clamp(min=0)], hd))  # [B, nkv, n * pt, .]
    q = s["q"].float().view(B, T, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, hd)
    score = (q * s["scale"]) @ _values(kc, ks).transpose(-1, -2)
    j = torch.arange(kc.shape[2], device="cuda")
    i = torch.arange(T, device="cuda")
    p = s["positions"][:, None] + i
    used = torch.full((B,), T, device="cuda") if s["n_tokens"] is None else s["n_tokens"]
    seen = (j <= p[..., None]) & (i < used[:, None])[..., None] & (s["table"] >= 0).repeat_interleave(pt, 1)[:, None]
    if s["window"]:
        seen &= (j > p[..., None] - s["window"]) | (j < s["sinks"])
    score = score.masked_fill(~seen.repeat_interleave(G, 1)[:, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    o = (w @ _values(vc, vs)) / torch.where(total == 0, torch.ones_like(total), total)
    return o.view(B, nkv, T, G, hd).permute(0, 2, 1, 3, 4).reshape(B * T, -1).to(torch.bfloat16)


def _plain_store(s):
    B, T, pt, hd = s["B"], s["T"], s["pt"], s["hd"]
    p = s["positions"][:, None].long() + torch.arange(T, device="cuda")
    page, slot = s["table"].long().gather(1, p // pt).flatten(), (p % pt).flatten()
    b = torch.arange(B, device="cuda")[:, None].expand(B, T).flatten()
    at = (b, p.flatten()) if s["static"] else (torch.arange(B * T, device="cuda"),)
    kc, vc, ks, vs = _parts(s["pool"], hd)
    for codes, scales, x, out in ((kc, ks, s["k"], s["k_out"]), (vc, vs, s["v"], s["v_out"])):
        c, sc = _quantise(x[at])
        codes[page, :, slot], scales[page, :, slot] = c, sc
        out[at] = _values(codes[page, :, slot], scales[page, :, slot]).to(torch.bfloat16)
    return s["k_out"], s["v_out"]


def _holders(table, held, P):
    keep = torch.arange(table.shape[1], device="cuda") < held[:, None]
    return torch.zeros(P, dtype=torch.int32, device="cuda").index_add_(0, table[keep].long(), torch.ones_like(table[keep]))


def _plain_fork(s):
    table, held, P, pt, pool = s["table"], s["held"], s["refs"].shape[0], s["pt"], s["pool"]
    at = s["parent"].clamp(min=0).long()
    gone = s["parent"] < 0
    t1, h1 = table[at].masked_fill(gone[:, None], -1), held[at].masked_fill(gone, 0)
    r1 = s["refs"] + _holders(t1, h1, P) - _holders(table, held, P)
    # room for the tokens to come: pages of one's own from the first one that is written
    slot = torch.arange(t1.shape[1], device="cuda")
    n = (s["need"] + pt - 1) // pt
    old = slot < h1[:, None]
    shared = old & (slot >= (s["keep"] // pt)[:, None]) & (slot < n[:, None]) & (r1[t1.clamp(min=0).long()] > 1)
    taken = shared | (~old & (slot < n[:, None]))
    back = shared | (old & (slot >= n[:, None]))
    free = torch.nonzero(r1 == 0)[:, 0].to(torch.int32)[: int(taken.sum())]
    t2 = t1.masked_fill(slot >= n[:, None], -1)
    t2[taken] = free
    copied = shared & (slot * pt < s["keep"][:, None])
    pool[:, t2[copied].long()] = pool[:, t1[copied].long()]
    r2 = r1.index_add(0, t1[back].long(), -torch.ones_like(t1[back]))
    r2[free.long()] = 1
    return {"table": t2, "held": n.to(torch.int32), "refs": r2, "missing": torch.zeros(1, dtype=torch.int32, device="cuda"), "pool": pool.view(torch.int32)}


def _plain_compact(s):
    table, refs, pool = s["table"], s["refs"], s["pool"]
    live = refs > 0
    n = int(live.sum())
    dst, src = torch.nonzero(~live[:n])[:, 0], n + torch.nonzero(live[n:])[:, 0]
    remap = torch.where(live, torch.arange(refs.shape[0], device="cuda"), -1).to(torch.int32)
    remap[src] = dst.to(torch.int32)
    out = refs.clone()
    out[dst], out[src] = refs[src], 0
    pool[:, dst] = pool[:, src]
    t = torch.where(table >= 0, remap[table.clamp(min=0).long()], -1)
    return {"table": t.to(torch.int32), "refs": out, "remap": remap, "pool": pool.view(torch.int32)}


def _plain_verify(s):
    x, ids, u, B, T, V = s["logits"].float(), s["draft_ids"].long(), s["uniforms"], s["B"], s["T"], s["V"]
    i = torch.arange(T, device="cuda")
    used = torch.full((B, 1), T, device="cuda") if s["n_draft"] is None else s["n_draft"][:, None]
    if s["temp"] == 0:
        best = x.argmax(-1)
        prob = (best[:, :T] == ids).float()
        ok = (prob > 0) & (i < used)
    else:
        x = x * float(np.float32(1) / np.float32(s["temp"]))
        w = (torch.exp(x - x.amax(-1, keepdim=True)) * FIX).to(torch.int64)
        total = w.sum(-1, keepdim=True)
        p = w.float() / total.float()
        px = p[:, :T].gather(2, ids[..., None])[..., 0]
        qx = torch.ones_like(px) if s["draft_probs"] is None else s["draft_probs"].gather(2, ids[..., None])[..., 0]
        ok = (u[:, :T] * qx < px) & (i < used)
        prob = torch.where(qx > 0, (px / qx).clamp(max=1.0), (px > 0).float())
    n = ok.to(torch.int64).cumprod(1).sum(1)
    row = n[:, None]
    if s["temp"] == 0:
        extra = best.gather(1, row)[:, 0]
    else:
        pick = row[..., None].expand(B, 1, V)
        w, p = w.gather(1, pick)[:, 0], p.gather(1, pick)[:, 0]
        refused = row < used
        last = row.clamp(max=T - 1)
        if s["draft_probs"] is None:
            left = w.scatter(1, ids.gather(1, last), 0)
        else:
            d = p - s["draft_probs"].gather(1, last[..., None].expand(B, 1, V))[:, 0]
            left = (torch.where(d > 0, d, torch.zeros_like(d)) * FIX).to(torch.int64)
        left = torch.where(refused & (left.sum(1, keepdim=True) > 0), left, w)
        total = left.sum(1, keepdim=True)
        part = (u[:, T:] * 16777216.0).to(torch.int64).clamp(0, 16777215)
        k = (total >> 32) * part * 256 + ((total & 0xFFFFFFFF) * part >> 24)
        extra = (left.cumsum(1) <= k).sum(1)
    at = torch.arange(T + 1, device="cuda")
    tokens = torch.where(at < row, torch.nn.functional.pad(ids, (0, 1)), torch.where(at == row, extra[:, None], -1))
    return {"accepted": n.to(torch.int32), "tokens": tokens.to(torch.int32), "prob": torch.where(i < used, prob, torch.zeros_like(prob))}


PLAIN = {"attn": _plain_attn, "store": _plain_store, "fork": _plain_fork, "compact": _plain_compact, "verify": _plain_verify}


# ---- the framework's calls ---------------------------------------------------------------------------
def _own_attn(s, K):
    if "workspace" not in s:
        s["workspace"] = K.kv4_attn_workspace(s["B"], s["T"], s["nq"], s["nkv"], s["hd"], s["q"].device)
    return K.kv4_attn(s["q"], s["pool"], s["table"], s["positions"], s["hd"], s["workspace"], scale=s["scale"], tokens_per_seq=s["T"],
                      n_tokens=s["n_tokens"], window=s["window"], sinks=s["sinks"])


def _own_store(s, K):
    K.kv4_append(s["k"], s["v"], s["pool"], s["table"], s["positions"], tokens_per_seq=s["T"])
    K.kv4_read(s["pool"], s["table"], s["positions"], s["k_out"], s["v_out"], tokens_per_seq=s["T"])
    return s["k_out"], s["v_out"]


def _own_fork(s, K):
    if "workspace" not in s:
        s["workspace"] = K.pages_workspace(s["S"], s["table"].shape[1], s["refs"].shape[0], s["table"].device)
    table, held, refs = K.pages_fork(s["table"], s["held"], s["refs"], s["parent"])
    missing = K.pages_resize(table, held, refs, s["keep"], s["need"], s["pool"], s["pt"], s["workspace"])
    return {"table": table, "held": held, "refs": refs, "missing": missing, "pool": s["pool"].view(torch.int32)}


def _own_compact(s, K):
    if "workspace" not in s:
        s["workspace"] = K.pages_workspace(s["S"], s["table"].shape[1], s["refs"].shape[0], s["table"].device)
    table, refs, remap = K.pages_compact(s["table"], s["held"], s["refs"], s["pool"], s["workspace"])
    return {"table": table, "refs": refs, "remap": remap, "pool": s["pool"].view(torch.int32)}


def _own_verify(s, K):
    if "workspace" not in s:
        s["workspace"] = K.verify_workspace(s["B"], s["T"], s["V"], s["logits"].device)
    n, tokens, prob = K.verify_drafts(s["logits"], s["draft_ids"], s["uniforms"], s["workspace"], draft_probs=s["draft_probs"],
                                      n_draft=s["n_draft"], temperature=s["temp"])
    return {"accepted": n, "tokens": tokens, "prob": prob}


OWN = {"attn": _own_attn, "store": _own_store, "fork": _own_fork, "compact": _own_compact, "verify": _own_verify}


def run(s):
    if own:
        return OWN[s["op"]](s, importlib.import_module("e2e-jaxscale_b200").kernels)
    return PLAIN[s["op"]](s)


# ---- the same from the definitions, in 64 bits -------------------------------------------------------
def _two(e):
    """Powers of two, exact (a GPU's pow() is not)."""
    return torch.tensor([2.0 ** k for k in range(-32, 33)], dtype=torch.float64, device=e.device)[e.long() + 32]


def _decode64(block, hd):
    """K and V [pt, hd] of one page's block of one head, by the formats' bit fields."""
    raw = block.cpu().numpy()
    pt = raw.shape[0] * 8 // (9 * hd)
    out, at = [], 0
    codes = []
    for _ in "kv":
        c = raw[at:at + pt * hd // 2].reshape(pt, hd // 2)
        at += pt * hd // 2
        codes.append(np.stack([c % 16, c // 16], -1).reshape(pt, hd).astype(np.int64))
    for c in codes:
        b = raw[at:at + pt * hd // 16].reshape(pt, hd // 16).astype(np.int64)
        at += pt * hd // 16
        e, m = (b >> 3) & 15, b & 7
        scale = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
        mag, e, m = c & 7, (c >> 1) & 3, c & 1
        val = np.where(e == 0, m / 2, (1 + m / 2) * 2.0 ** (e - 1.0)) * np.where(c > 7, -1.0, 1.0)
        out.append((val.reshape(pt, -1, 16) * scale[..., None]).reshape(pt, hd))
    return out


def _exact_attn(c, s):
    if c["B"] * c["L"] * c["nkv"] * c["T"] > 700_000:
        return _exact_attn_some(c, s)
    return _attn64(c, s, range(c["B"]))


def _attn64(c, s, which):
    hd, pt, G, T = c["hd"], c["pt"], c["nq"] // c["nkv"], c["T"]
    q = s["q"].double().cpu().numpy().reshape(c["B"], T, c["nq"], hd)
    table, pos = s["table"].cpu().numpy(), s["positions"].cpu().numpy()
    used = [T] * c["B"] if s["n_tokens"] is None else s["n_tokens"].tolist()
    o = np.zeros((c["B"], T, c["nq"], hd))
    for b in which:
        last = int(pos[b]) + T
        if last <= 0:
            continue
        for h in range(c["nkv"]):
            blocks = [_decode64(s["pool"][int(table[b, n]), h], hd) for n in range(-(-last // pt))]
            k, v = (np.concatenate([x[w] for x in blocks])[:last] for w in (0, 1))
            for t in range(used[b]):
                p = int(pos[b]) + t
                j = np.arange(last)
                seen = (j <= p) & ((c["window"] == 0) | (j > p - c["window"]) | (j < c["sinks"]))
                if not seen.any():
                    continue
                a = q[b, t, h * G:(h + 1) * G] @ k[seen].T * s["scale"]
                a = np.exp(a - a.max(1, keepdims=True))
                o[b, t, h * G:(h + 1) * G] = (a / a.sum(1, keepdims=True)) @ v[seen]
    return torch.from_numpy(o.reshape(c["B"] * T, -1))


def _exact_attn_some(c, s):
    """Large caches: the same on the GPU, one sequence and head at a time."""
    hd, pt, G, T = c["hd"], c["pt"], c["nq"] // c["nkv"], c["T"]
    q = s["q"].double().view(c["B"], T, c["nkv"], G, hd)
    pos = s["positions"].tolist()
    used = [T] * c["B"] if s["n_tokens"] is None else s["n_tokens"].tolist()
    o = torch.zeros(c["B"], T, c["nkv"], G, hd, dtype=torch.float64, device="cuda")
    a = pt * hd // 2
    for b in range(c["B"]):
        last = pos[b] + T
        pages = s["table"][b, : -(-last // pt)].long()
        for h in range(c["nkv"]):
            raw = s["pool"][pages, h].to(torch.int64)
            kv = []
            for w in (0, 1):
                code = raw[:, w * a:(w + 1) * a].reshape(-1, hd // 2)
                code = torch.stack([code % 16, code // 16], -1).reshape(-1, hd)
                e, m = (code >> 1) & 3, (code & 1).double()
                val = torch.where(e == 0, m / 2, (1 + m / 2) * _two(e - 1))
                val = torch.where(code > 7, -val, val)
                sb = raw[:, 2 * a + w * (a // 8):2 * a + (w + 1) * (a // 8)].reshape(-1, hd // 16)
                e, m = (sb >> 3) & 15, (sb & 7).double()
                sc = torch.where(e == 0, m / 8 / 64, (1 + m / 8) * _two(e - 7))
                kv.append((val.view(-1, hd // 16, 16) * sc[..., None]).reshape(-1, hd)[:last])
            for t in range(used[b]):
                p = pos[b] + t
                j = torch.arange(last, device="cuda")
                seen = (j <= p) & ((c["window"] == 0) | (j > p - c["window"]) | (j < c["sinks"]))
                x = torch.where(seen, q[b, t, h] @ kv[0].T * s["scale"], torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
                o[b, t, h] = torch.nan_to_num(torch.softmax(x, -1)) @ kv[1]  # a row that sees nothing is 0
    return o.reshape(c["B"] * T, -1)


def _exact_store(c, s):
    def back(x):
        x = x.double().unflatten(-1, (-1, 16))
        top = x.abs().amax(-1, keepdim=True)
        want = torch.clamp(top / torch.full_like(top, 6.0), max=448.0)
        step = _two(torch.frexp(want.clamp(min=2.0 ** -6)).exponent - 4)
        scale = torch.round(want / step) * step  # torch.round: halves to even
        unit = torch.where(scale > 0, scale, torch.ones_like(scale))
        m = torch.where(scale > 0, x.abs() / unit, torch.zeros_like(x))
        grid = torch.where(m < 2, torch.round(m * 2) / 2, torch.where(m < 4, torch.round(m), torch.round(m / 2) * 2)).clamp(max=6)
        return (grid * torch.sign(x) * scale).flatten(-2)

    out = []
    for x in (s["k"], s["v"]):
        y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        if c["static"]:
            y[:, c["start"]:] = back(x[:, c["start"]:])
        else:
            y = back(x)
        out.append(y)
    return tuple(out)


def _exact_verify(c, s):
    prob = torch.zeros(c["B"], c["T"], dtype=torch.float64, device="cuda")
    used = [c["T"]] * c["B"] if s["n_draft"] is None else s["n_draft"].tolist()
    for b in range(c["B"]):
        for i in range(used[b]):
            x, at = s["logits"][b, i].double(), int(s["draft_ids"][b, i])
            if c["temp"] == 0:
                prob[b, i] = float(bool((x[at] == x.max()) and not (x[:at] == x.max()).any()))
                continue
            p = torch.softmax(x / float(np.float32(c["temp"])), 0)[at]
            q = 1.0 if s["draft_probs"] is None else s["draft_probs"][b, i, at].double()
            prob[b, i] = min(1.0, float(p / q))
    return {"accepted": None, "tokens": None, "prob": prob}


def exact(c, seed):
    if c["op"] in ("fork", "compact"):
        return None  # whole numbers only
    s = prepare(c, seed)
    return {"attn": _exact_attn, "store": _exact_store, "verify": _exact_verify}[c["op"]](c, s)
