"""After a wait of the attention over 4-bit pages gave up, counters of shares that never met stay in
its workspace: device_error, which reports it, makes every live workspace fit for the next call."""

import gc

import pytest
import torch


def fake(jsx, monkeypatch, status, size=4096):
    """The library's answers, without a device: a workspace's size, and a status of the device."""
    def call(name, *args):
        if name == "jsx_kv4_attn_workspace_size":
            args[-1]._obj.value = size
        elif name == "jsx_device_error":
            args[-1]._obj.value = status
        else:
            raise AssertionError(name)
    monkeypatch.setattr(jsx.kernels, "call", call)


@pytest.mark.parametrize("status", [0, 3])
def test_workspaces_are_zero_after_a_timeout(jsx, monkeypatch, status):
    fake(jsx, monkeypatch, status)
    ws = [jsx.kernels.kv4_attn_workspace(1, 1, 32, 2, 128, "cpu") for _ in range(3)]
    for w in ws:
        w[100:200] = 1
    dropped = jsx.kernels.kv4_attn_workspace(2, 1, 32, 2, 128, "cpu")
    del dropped
    gc.collect()
    assert jsx.kernels.device_error() == status
    for w in ws:
        assert bool(w.any()) == (status == 0)


@pytest.mark.gpu
def test_attention_after_a_timeout(jsx, cuda, monkeypatch):
    """Counters as a call that gave up leaves them, a device that reports it: the next call is right."""
    K = jsx.kernels
    B, nq, nkv, hd, L = 2, 32, 2, 128, 3000
    cache = jsx.PagedKV4Cache(1, B, L, nkv, hd)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    assert int(cache.reserve(zero, torch.full_like(zero, L))) == 0
    k = torch.randn(B, L, nkv, hd, device="cuda").to(torch.bfloat16)
    cache.append(0, k, k, zero, tokens_per_seq=L)
    q = torch.randn(B, nq * hd, device="cuda").to(torch.bfloat16)
    ws = K.kv4_attn_workspace(B, 1, nq, nkv, hd, q.device)
    pos = torch.tensor([L - 1, 1700], dtype=torch.int32, device="cuda")
    want = K.kv4_attn(q, cache.pool[0], cache.table, pos, hd, ws)
    assert not ws[:4096].any()                     # counters are zero between calls
    ws[:4096].view(torch.int32)[::3] = 1
    real = K.call

    def call(name, *args):
        if name == "jsx_device_error":
            args[-1]._obj.value = 3
        else:
            real(name, *args)
    with monkeypatch.context() as m:
        m.setattr(K, "call", call)
        assert K.device_error() == 3
    assert not ws[:4096].any()
    assert torch.equal(K.kv4_attn(q, cache.pool[0], cache.table, pos, hd, ws), want)
