"""PagedKV4Cache.attend keeps one growing workspace per stream, not one per shape of a call."""

import pytest
import torch

pytestmark = pytest.mark.gpu

B, NQ, NKV, HD, L = 2, 32, 2, 128, 600


def filled(jsx):
    cache = jsx.PagedKV4Cache(1, B, L, NKV, HD)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    assert int(cache.reserve(zero, torch.full_like(zero, L))) == 0
    k = torch.randn(B, L, NKV, HD, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    cache.append(0, k, k, zero, tokens_per_seq=L)
    return cache


def queries(T):
    return torch.randn(B * T, NQ * HD, generator=torch.Generator("cuda").manual_seed(T), device="cuda").to(torch.bfloat16)


def test_memory_does_not_grow_with_every_length(jsx, cuda):
    """What is kept over 24 lengths is at most twice the largest length's workspace."""
    cache = filled(jsx)
    pos = torch.full((B,), 100, dtype=torch.int32, device="cuda")
    lengths = list(range(1, 25))
    largest = max(jsx.kernels.kv4_attn_workspace(B, T, NQ, NKV, HD, "cuda").numel() for T in lengths)
    q = {T: queries(T) for T in lengths}
    out = {T: torch.empty_like(q[T]) for T in lengths}
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for T in lengths:
        cache.attend(0, q[T], pos, HD ** -0.5, tokens_per_seq=T, out=out[T])
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 2 * largest + (1 << 20)
    for T in lengths:                              # each as with a workspace of its own
        ws = jsx.kernels.kv4_attn_workspace(B, T, NQ, NKV, HD, "cuda")
        assert torch.equal(out[T], jsx.kernels.kv4_attn(q[T], cache.pool[0], cache.table, pos, HD, ws, tokens_per_seq=T))


def test_streams_do_not_share_one(jsx, cuda, monkeypatch):
    cache = filled(jsx)
    pos = torch.full((B,), 500, dtype=torch.int32, device="cuda")
    q = queries(1)
    used, real = [], jsx.kernels.kv4_attn
    monkeypatch.setattr(jsx.kernels, "kv4_attn", lambda q, pool, table, pos, hd, ws, **kw: used.append(ws) or real(q, pool, table, pos, hd, ws, **kw))
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (one, two, one):
        with torch.cuda.stream(s):
            outs.append(cache.attend(0, q, pos, HD ** -0.5))
    torch.cuda.synchronize()
    assert used[0].data_ptr() != used[1].data_ptr() and used[0].data_ptr() == used[2].data_ptr()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_a_captured_call_outlives_growth(jsx, cuda):
    """The workspace a graph was captured with stays while later calls take a larger one."""
    cache = filled(jsx)
    pos = torch.full((B,), 500, dtype=torch.int32, device="cuda")
    q, out = queries(1), torch.zeros(B, NQ * HD, dtype=torch.bfloat16, device="cuda")
    want = cache.attend(0, q, pos, HD ** -0.5)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(cache.attend(0, q, pos, HD ** -0.5), want)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        cache.attend(0, q, pos, HD ** -0.5, out=out)
    with torch.cuda.stream(s):
        for T in (16, 24):                         # grows on the stream of the capture
            cache.attend(0, queries(T), pos, HD ** -0.5, tokens_per_seq=T)
        other = torch.full((1 << 24,), 0xff, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and bool((other == 0xff).all())


def test_a_workspace_made_in_a_capture_is_that_graphs_own(jsx, cuda, monkeypatch):
    """Its zero-fill is a node of the graph: a second graph that is replayed first cannot rely on it."""
    cache = filled(jsx)
    pos = torch.full((B,), 500, dtype=torch.int32, device="cuda")
    q = queries(1)
    want = cache.attend(0, q, pos, HD ** -0.5)
    used, real = [], jsx.kernels.kv4_attn
    monkeypatch.setattr(jsx.kernels, "kv4_attn", lambda q, pool, table, pos, hd, ws, **kw: used.append(ws) or real(q, pool, table, pos, hd, ws, **kw))
    s = torch.cuda.Stream()
    graphs, outs = [], []
    for _ in range(2):
        g, o = torch.cuda.CUDAGraph(), [torch.zeros_like(want) for _ in range(3)]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            for y in o:                            # several calls of a graph share one
                cache.attend(0, q, pos, HD ** -0.5, out=y)
        graphs.append(g)
        outs.append(o)
    assert len({w.data_ptr() for w in used[:3]}) == 1 and len({w.data_ptr() for w in used[3:]}) == 1
    used[0].fill_(1)                               # as memory that nobody filled
    torch.cuda.synchronize()
    for g, o in zip(reversed(graphs), reversed(outs)):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for y in o)
    with torch.cuda.stream(s):                     # and neither can a call outside of graphs
        got = cache.attend(0, q, pos, HD ** -0.5)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and not used[-1][:4096].any()   # (counters)


def test_capture_id(jsx, cuda):
    K = jsx.kernels
    assert K.capture_id() == 0
    x, seen = torch.zeros(4, device="cuda"), []
    for _ in range(2):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            seen += [K.capture_id(), K.capture_id()]
            x.add_(1)
    assert K.capture_id() == 0 and seen[0] == seen[1] != 0 and seen[2] == seen[3] not in (0, seen[0])
    with pytest.raises(jsx._lib.JsxError):
        jsx._lib.call("jsx_stream_capture_id", None, None)
