"""PagedKV4Cache.fork leaves `table`, `held` and `refs` where they are: a step captured in a graph reads the
forked table when it is replayed."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_fork_keeps_the_tensors(jsx, cuda):
    cache = jsx.PagedKV4Cache(1, 3, 64, 1, 64, page_tokens=16)
    assert int(cache.reserve(i32(0, 0, 0), i32(40, 10, 0))) == 0
    table, held, refs = cache.table, cache.held, cache.refs
    row = table[0].tolist()
    for parent, counts in (((0, 0, 1), [3, 3, 1]), ((2, -1, 0), [1, 0, 3]), ((0, 1, 2), [1, 0, 3])):
        cache.fork(i32(*parent))
        assert cache.table is table and cache.held is held and cache.refs is refs
        assert held.tolist() == counts
    assert table[2].tolist() == row and (table[1] == -1).all()
    assert int((refs > 0).sum()) == 4


def test_a_captured_step_follows_a_fork(jsx, cuda):
    B, nq, nkv, hd, L = 3, 8, 2, 128, 200
    cache = jsx.PagedKV4Cache(1, B, L, nkv, hd, page_tokens=32)
    zero = i32(0, 0, 0)
    assert int(cache.reserve(zero, i32(L, L, L))) == 0
    rows = torch.randn(B, L, nkv, hd, device="cuda").to(torch.bfloat16)
    cache.append(0, rows, rows, zero, tokens_per_seq=L)
    q = torch.randn(1, nq * hd, device="cuda").to(torch.bfloat16).expand(B, -1).contiguous()
    pos, out = i32(150, 150, 150), torch.zeros(B, nq * hd, dtype=torch.bfloat16, device="cuda")
    first = cache.attend(0, q, pos, hd ** -0.5)    # (workspaces exist before the capture)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(0, q, pos, hd ** -0.5, out=out)
    for parent in ((1, 1, 0), (2, 0, 1)):
        cache.fork(i32(*parent))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, cache.attend(0, q, pos, hd ** -0.5))
        first = first[list(parent)]
        assert torch.equal(out, first)
