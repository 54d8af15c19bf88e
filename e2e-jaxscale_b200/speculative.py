"""Generation with drafted tokens over the paged 4-bit cache.

Where the reference decodes one token per step over a static bf16 cache (runner.py:240-308,
:366-460), a step here takes every sequence's last token and up to `draft_tokens` proposed
ones through the model at once, on the tensor-core projections (jsx_tc_*, 32 tokens per call).
Up to 32 tokens of all sequences together share one pass over the weights; more go in spans of
whole sequences, a pass each, so drafting pays for small batches (9B shape, 40 layers, context
1024, in a graph: 1 x 5 tokens 5.1 ms, 6 x 5 5.7 ms, 16 x 5 14.2 ms, 32 x 5 26.8 ms; one token of
32 sequences in the plain decode step: 5.4 ms, of one: 3.6 ms).  The target's logits then accept
or replace the proposals (jsx_verify_drafts), so at a temperature (without top-k, top-p or
penalties) the output is distributed as without drafts.  At temperature 0 it is the greedy
continuation; different numbers of tokens per step round differently, so two near-equal logits
may change places between a run with drafts and one without.

Per layer: q/k/v + bias + RoPE into a one-layer bf16 staging cache, its new rows into the
4-bit pages (jsx_kv4_append), attention over the pages (jsx_kv4_attn, with an optional window
and first tokens that stay visible), o_proj, gate/up, down.  Pages are reserved before a step
and what refused drafts had written is simply overwritten by the next one.

Proposals come from the text itself (prompt lookup): the longest recent n-gram that occurred
before is continued as it was then.  `draft` replaces this by another proposer.
"""

from __future__ import annotations

import numpy as np
import torch

from . import kernels as K
from .glm4 import TC_CHUNK, GLM4ForCausalLM
from .layers.kv_cache import KVCache
from .layers.paged_cache import PagedKV4Cache
from .runner import _full_logits


def prompt_lookup(history: list[int], count: int, longest: int = 3) -> list[int]:
    """Up to `count` tokens that followed the last earlier occurrence of the history's final
    n-gram, n = longest .. 1."""
    h = np.asarray(history)
    for n in range(min(longest, len(h) - 1), 0, -1):
        windows = np.lib.stride_tricks.sliding_window_view(h[:-1], n)
        at = np.nonzero((windows == h[-n:]).all(1))[0]
        if len(at):
            return h[at[-1] + n:at[-1] + n + count].tolist()
    return []


class DraftedState:
    """Device buffers of B sequences with T tokens each per step."""

    def __init__(self, model: GLM4ForCausalLM, batch: int, tokens: int, max_tokens: int, page_tokens: int = 64,
                 num_pages: int | None = None):
        c, dev = model.config, model.device
        if tokens > TC_CHUNK:
            raise ValueError(f"at most {TC_CHUNK} tokens per sequence and step (got {tokens})")
        self.batch, self.tokens, self.max_tokens = batch, tokens, max_tokens
        M, H = batch * tokens, c.hidden_size
        bf = dict(dtype=torch.bfloat16, device=dev)
        i32 = dict(dtype=torch.int32, device=dev)
        self.cache = PagedKV4Cache(c.num_hidden_layers, batch, max_tokens, model.nkv_l, c.head_dim, page_tokens,
                                   num_pages, device=dev)
        # rows of the layer at work, before they are quantised (every layer uses it in turn)
        shape = (batch, max_tokens, model.nkv_l, c.head_dim)
        self.staging = KVCache(torch.zeros(shape, **bf), torch.zeros(shape, **bf))
        self.ids = torch.zeros(M, **i32)
        self.pos = torch.zeros(M, **i32)
        self.first = torch.zeros(batch, **i32)     # position of every sequence's first token of the step
        self.count = torch.zeros(batch, **i32)     # tokens it uses
        self.argmax = torch.zeros(M, **i32)
        self.h = torch.zeros(M, H, **bf)
        self.q = torch.zeros(M, model.nq_l * c.head_dim, **bf)
        self.attn = torch.zeros_like(self.q)
        self.act = torch.zeros(M, model.I_l, **bf)
        self.logits = torch.zeros(M, model.V_l, **bf)
        lp = model.layers[0]
        shapes = [tuple(reversed(w.shape)) for w in (lp.w_qkv, lp.w_o, lp.w_gu, lp.w_d)] + [(H, model.V_l)]
        self.tc_ws = K.tc_workspace(min(M, TC_CHUNK), shapes, dev)
        self.verify_ws = K.verify_workspace(batch, tokens - 1, c.vocab_size, dev)
        self._steps = torch.arange(tokens, **i32)


def prefill(model: GLM4ForCausalLM, st: DraftedState, input_ids: torch.Tensor, window: int = 0,
            sinks: int = 0) -> torch.Tensor:
    """Takes [B, S] prompts through the model in one pass, leaves their rows in the pages and
    returns the logits [B, V] after the last token.  Without a window the prompt attends to its
    own bf16 rows; with one, to the pages."""
    c, dev = model.config, model.device
    B, S = input_ids.shape
    M, H, eps, hd, rot = B * S, c.hidden_size, c.rms_norm_eps, c.head_dim, model.rotary.rotary_dim
    lp0 = model.layers[0]
    shapes = [tuple(reversed(w.shape)) for w in (lp0.w_qkv, lp0.w_o, lp0.w_gu, lp0.w_d)]
    ws = K.wide_workspace(M, shapes, dev)
    comm = model.mesh.comm_tiles(M, H) if model.tp > 1 else None
    pos = torch.arange(S, dtype=torch.int32, device=dev).repeat(B)
    zero = torch.zeros(B, dtype=torch.int32, device=dev)
    _reserve(st, zero, torch.full_like(zero, S))
    h = K.embed(input_ids.reshape(-1).to(torch.int32).contiguous(), model.embed)
    q = torch.empty(M, model.nq_l * hd, dtype=torch.bfloat16, device=dev)
    attn, act = torch.empty_like(q), torch.empty(M, model.I_l, dtype=torch.bfloat16, device=dev)
    k, v = st.staging.k, st.staging.v
    for i, lp in enumerate(model.layers):
        K.wide_qkv_rope_cache(h, lp.ln1, eps, lp.w_qkv, lp.b_qkv, model.inv_freq, pos, q, k, v, model.nq_l,
                              model.nkv_l, hd, rot, ws, tokens_per_seq=S)
        st.cache.append(i, k, v, zero, tokens_per_seq=S)
        if window:
            st.cache.attend(i, q, zero, model.scale, tokens_per_seq=S, window=window, sinks=sinks, out=attn)
        else:
            K.attn_prefill(q, k, v, model.nq_l, model.nkv_l, hd, S, scale=model.scale, out=attn)
        K.wide_row_linear_allreduce(comm, attn, lp.w_o, h, ws)
        K.wide_gate_up_swiglu(h, lp.ln2, eps, lp.w_gu, act, ws)
        K.wide_row_linear_allreduce(comm, act, lp.w_d, h, ws)
    last = h.view(B, S, H)[:, -1].contiguous()
    logits = torch.empty(B, model.V_l, dtype=torch.bfloat16, device=dev)
    _head(model, last, K.tc_workspace(min(B, TC_CHUNK), [(H, model.V_l)], dev), torch.empty_like(zero), logits)
    return _full_logits(model, logits)


def step(model: GLM4ForCausalLM, st: DraftedState, window: int = 0, sinks: int = 0) -> torch.Tensor:
    """One pass over st.ids (T per sequence, at st.first .. + T - 1, of which st.count are
    used): the rows go into the pages (room is reserved by the caller), the logits [B, T, V]
    come back."""
    c, eps, hd, rot = model.config, model.config.rms_norm_eps, model.config.head_dim, model.rotary.rotary_dim
    B, T, ws = st.batch, st.tokens, st.tc_ws
    # unused tokens of a sequence at its end stay inside the staging cache
    st.pos.view(B, T).copy_((st.first[:, None] + st._steps).clamp_(max=st.max_tokens - 1))
    K.embed(st.ids, model.embed, out=st.h)
    spans = [(b, min(B, b + TC_CHUNK // T)) for b in range(0, B, TC_CHUNK // T)]
    k, v = st.staging.k, st.staging.v
    for i, lp in enumerate(model.layers):
        for b0, b1 in spans:
            m = slice(b0 * T, b1 * T)
            K.tc_qkv_rope_cache(st.h[m], lp.ln1, eps, lp.w_qkv, lp.b_qkv, model.inv_freq, st.pos[m], st.q[m],
                                k[b0:b1], v[b0:b1], model.nq_l, model.nkv_l, hd, rot, ws, tokens_per_seq=T)
        st.cache.append(i, k, v, st.first, tokens_per_seq=T, n_tokens=st.count)
        st.cache.attend(i, st.q, st.first, model.scale, tokens_per_seq=T, n_tokens=st.count, window=window,
                        sinks=sinks, out=st.attn)
        for b0, b1 in spans:
            m = slice(b0 * T, b1 * T)
            K.tc_row_linear_allreduce(model.comm, st.attn[m], lp.w_o, st.h[m], ws)
            K.tc_gate_up_swiglu(st.h[m], lp.ln2, eps, lp.w_gu, st.act[m], ws)
            K.tc_row_linear_allreduce(model.comm, st.act[m], lp.w_d, st.h[m], ws)
    _head(model, st.h, ws, st.argmax, st.logits)
    return _full_logits(model, st.logits).view(B, T, -1)


def _head(model, h, ws, ids, logits) -> None:
    for m0 in range(0, h.shape[0], TC_CHUNK):
        m = slice(m0, min(h.shape[0], m0 + TC_CHUNK))
        K.tc_lmhead_argmax(model.comm, h[m], model.norm, model.config.rms_norm_eps, model.lm_head, model.vocab_offset,
                           ids[m], ws, logits[m])


class PoolExhausted(RuntimeError):
    """The page pool cannot hold the next step.  `tokens`: what speculative_generate had until then,
    in the shape that it returns."""

    tokens: torch.Tensor | None = None


def _reserve(st: DraftedState, keep, need) -> None:
    missing = int(st.cache.reserve(keep, need))
    if missing:
        raise PoolExhausted(f"the page pool is too small: {missing} pages missing")


def speculative_generate(model: GLM4ForCausalLM, input_ids, max_new_tokens: int = 128, draft_tokens: int = 4,
                         temperature: float = 0.0, window: int = 0, sinks: int = 0, page_tokens: int = 64,
                         num_pages: int | None = None, eos_token_id=None, seed: int = 42, draft=prompt_lookup,
                         stats: dict | None = None) -> torch.Tensor:
    """Generates over the paged 4-bit cache with up to draft_tokens proposals per step.
    draft(history, count) -> at most count token ids; temperature 0 is greedy.  Sequences go on
    until max_new_tokens or an EOS id, each at its own pace.  Returns [B, prompt + max_new_tokens]
    int32 on the host, filled up with the EOS id (or -1) after a sequence's end.  `stats`
    receives the steps taken and the drafts proposed and accepted.  Where num_pages do not
    suffice, PoolExhausted has the text so far."""
    ids = torch.as_tensor(input_ids, dtype=torch.int32).cpu()
    B, S = ids.shape
    T, V, dev = draft_tokens + 1, model.config.vocab_size, model.device
    eos = [] if eos_token_id is None else [eos_token_id] if isinstance(eos_token_id, int) else list(eos_token_id)
    st = DraftedState(model, B, T, S + max_new_tokens + T, page_tokens, num_pages)
    gen = torch.Generator(device=dev).manual_seed(seed)
    history = [row.tolist() for row in ids]
    out = [[] for _ in range(B)]
    tally = {"steps": 0, "drafted": 0, "accepted": 0}

    def take(b, tokens):
        for t in tokens:
            if len(out[b]) < max_new_tokens and not (out[b] and out[b][-1] in eos):
                out[b].append(t)
                history[b].append(t)

    def over(b):
        return len(out[b]) >= max_new_tokens or (len(out[b]) > 0 and out[b][-1] in eos)

    def text():
        fill = eos[0] if eos else -1
        rows = [out[b] + [fill] * (max_new_tokens - len(out[b])) for b in range(B)]
        return torch.cat([ids, torch.tensor(rows, dtype=torch.int32).reshape(B, max_new_tokens)], dim=1)

    try:
        # the first token: a draw without drafts
        logits = prefill(model, st, ids.to(dev), window, sinks)
        none = torch.zeros(B, 0, dtype=torch.int32, device=dev)
        _, tokens, _ = K.verify_drafts(logits[:, None], none, torch.rand(B, 1, generator=gen, device=dev),
                                       K.verify_workspace(B, 0, V, dev), temperature=temperature)
        for b, row in enumerate(tokens.tolist()):
            take(b, row)

        while not all(over(b) for b in range(B)):
            drafts = [[] if over(b) else list(draft(history[b], min(draft_tokens, max_new_tokens - len(out[b]) - 1)))
                      for b in range(B)]
            # (a sequence that is over keeps nothing: its pages are free for the others)
            first = torch.tensor([0 if over(b) else len(history[b]) - 1 for b in range(B)], dtype=torch.int32)
            count = torch.tensor([0 if over(b) else 1 + len(drafts[b]) for b in range(B)], dtype=torch.int32)
            fed = torch.tensor([[history[b][-1]] + drafts[b] + [0] * (draft_tokens - len(drafts[b])) for b in range(B)],
                               dtype=torch.int32)
            st.first.copy_(first)
            st.count.copy_(count)
            st.ids.copy_(fed.reshape(-1))
            _reserve(st, st.first, st.first + st.count)
            logits = step(model, st, window, sinks)
            accepted, tokens, _ = K.verify_drafts(
                logits, st.ids.view(B, T)[:, 1:].contiguous(), torch.rand(B, T, generator=gen, device=dev),
                st.verify_ws, n_draft=(st.count - 1).clamp_(min=0), temperature=temperature)
            accepted, tokens = accepted.tolist(), tokens.tolist()
            tally["steps"] += 1
            for b in range(B):
                if not over(b):
                    tally["drafted"] += len(drafts[b])
                    tally["accepted"] += accepted[b]
                    take(b, tokens[b][:accepted[b] + 1])
    except PoolExhausted as e:
        e.tokens = text()
        raise
    if stats is not None:
        stats.update(tally)
    return text()
