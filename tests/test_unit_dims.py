"""Strides of dimensions of length one say nothing about where elements are: calls that differ in
them alone give the same answers."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(jsx, pages, nkv, hd, pt):
    return torch.zeros(pages, nkv, jsx.kernels.kv4_page_bytes(nkv, hd, pt) // nkv, dtype=torch.uint8, device="cuda")


def odd(t, dim):
    """The same elements, with a stride of 1 in a dimension of length one."""
    assert t.shape[dim] == 1
    s = list(t.stride())
    s[dim] = 1
    return t.as_strided(t.shape, s, t.storage_offset())


def test_one_query_row(jsx, cuda):
    K = jsx.kernels
    p, t = pool(jsx, 4, 2, 128, 16), i32(3, 1).view(1, 2)
    k = torch.randn(20, 2, 128, device="cuda").to(BF)
    K.kv4_append(k, k, p, t, i32(0), tokens_per_seq=20)
    q = torch.randn(1, 8 * 128, device="cuda").to(BF)
    ws = K.kv4_attn_workspace(1, 1, 8, 2, 128, "cuda")
    want = K.kv4_attn(q, p, t, i32(19), 128, ws)
    out = torch.zeros_like(want)
    assert torch.equal(K.kv4_attn(odd(q, 0), p, t, i32(19), 128, ws, out=odd(out, 0)), want) and torch.equal(out, want)
    assert torch.equal(K.kv4_attn(q.flatten()[:, None].t(), p, t, i32(19), 128, ws), want)


def test_one_token_one_head_one_sequence(jsx, cuda):
    K = jsx.kernels
    for nkv, shape, dims in ((2, (1, 2, 64), [0]), (1, (1, 1, 64), [0, 1]), (1, (6, 1, 64), [1]), (2, (1, 32, 2, 64), [0]), (1, (1, 32, 1, 64), [0, 2])):
        B, T = 1, shape[0] if len(shape) == 3 else 30
        t = i32(1, 0, 2).view(1, 3)
        k, v = (torch.randn(*shape, device="cuda").to(BF) for _ in "kv")
        a, b = pool(jsx, 4, nkv, 64, 16), pool(jsx, 4, nkv, 64, 16)
        K.kv4_append(k, v, a, t, i32(0), tokens_per_seq=T)
        ko = k
        for d in dims:
            ko = odd(ko, d)
        K.kv4_append(ko, v, b, t, i32(0), tokens_per_seq=T)    # v as it is: the layouts are the same
        assert torch.equal(a, b) and a.any()
        outs = [torch.zeros_like(k) for _ in range(4)]
        K.kv4_read(a, t, i32(0), outs[0], outs[1], tokens_per_seq=T)
        x = outs[3]
        for d in dims:
            x = odd(x, d)
        K.kv4_read(a, t, i32(0), outs[2], x, tokens_per_seq=T)
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_one_row_of_logits_per_sequence(jsx, cuda, temperature):
    """No drafts: logits [B, V] of a padded vocabulary, with a dimension put in."""
    K = jsx.kernels
    B, V, wide = 5, 1000, 1024
    padded = (torch.randn(B, wide, device="cuda") * 3).to(BF)
    none, u = torch.zeros(B, 0, dtype=torch.int32, device="cuda"), torch.from_numpy(np.random.default_rng(0).random((B, 1), dtype=np.float32)).cuda()
    ws = K.verify_workspace(B, 0, V, "cuda")
    want = K.verify_drafts(padded[:, :V].contiguous()[:, None], none, u, ws, temperature=temperature)
    got = K.verify_drafts(padded[:, :V][:, None], none, u, ws, temperature=temperature)
    assert torch.equal(got[1], want[1]) and (got[1] >= 0).all()
    one = K.verify_drafts(odd(odd(padded[:1, :V][:, None], 0), 1), none[:1], u[:1], ws, temperature=temperature)
    assert torch.equal(one[1], want[1][:1])
    drafted = padded[:4, :V].contiguous().view(1, 4, V)        # one sequence with three drafts
    ids = drafted[:, :3].float().argmax(-1).int()
    a = K.verify_drafts(drafted, ids, u[:4].view(1, 4), K.verify_workspace(1, 3, V, "cuda"), temperature=temperature)
    b = K.verify_drafts(odd(padded[None, :4, :V], 0), ids, u[:4].view(1, 4), K.verify_workspace(1, 3, V, "cuda"), temperature=temperature)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_other_strides_are_still_refused(jsx, cuda):
    K = jsx.kernels
    p, t = pool(jsx, 4, 2, 64, 16), i32(1, 0).view(1, 2)
    k = torch.randn(2, 2, 64, device="cuda").to(BF)
    with pytest.raises(ValueError):
        K.kv4_append(k, torch.empty(2, 3, 64, device="cuda", dtype=BF)[:, :2], p, t, i32(0), tokens_per_seq=2)
    x = torch.zeros(3, 4, 50, device="cuda")[:, :3]
    with pytest.raises(ValueError):
        K.verify_drafts(x, torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.zeros(3, 3, device="cuda"), K.verify_workspace(3, 2, 50, "cuda"))
