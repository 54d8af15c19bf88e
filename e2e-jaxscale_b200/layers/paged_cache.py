"""Paged key/value cache in 4 bits (e2m1 codes, one e4m3 scale per 16 values), the long-context
counterpart of the static bf16 cache (layers/kv_cache.py:16-61 of the reference): 4.5 bits per
value, pages handed out on demand, shared between sequences and moved, all on the device.

One pool holds every layer: [layers, num_pages, kv_heads_on_this_rank, block]; a page number is
the same page in each of them.  `table` names the pages of every sequence, `held` how many slots
of a row are in use, `refs` how many holders a page has.
"""

from __future__ import annotations

import torch

from .. import kernels as K


class PagedKV4Cache:
    def __init__(self, num_layers: int, batch_size: int, max_tokens: int, num_kv_heads: int, head_dim: int,
                 page_tokens: int = 64, num_pages: int | None = None, device="cuda"):
        """num_pages None: room for every sequence's max_tokens."""
        self.page_tokens, self.head_dim, self.num_kv_heads = page_tokens, head_dim, num_kv_heads
        page_bytes = K.kv4_page_bytes(num_kv_heads, head_dim, page_tokens)
        self.slots = -(-max_tokens // page_tokens)
        self.num_pages = batch_size * self.slots if num_pages is None else num_pages
        i32 = dict(dtype=torch.int32, device=device)
        self.pool = torch.zeros(num_layers, self.num_pages, num_kv_heads, page_bytes // num_kv_heads,
                                dtype=torch.uint8, device=device)
        # table and held are parts of one buffer, so that fork sets aside both in one copy
        n = batch_size * self.slots
        self._rows, self._old_rows = (torch.full((n + batch_size,), -1, **i32) for _ in range(2))
        self.table, self.held, self._old_table, self._old_held = (
            part for rows in (self._rows, self._old_rows) for part in (rows[:n].view(batch_size, self.slots), rows[n:]))
        self.held.zero_()
        self.refs = torch.zeros(self.num_pages, **i32)
        self.missing = torch.zeros(1, **i32)
        self._remap = torch.empty_like(self.refs)
        self._ws = K.pages_workspace(batch_size, self.slots, self.num_pages, device)
        self._attn_ws = {}       # by stream: its workspace, of the largest call so far
        self._attn_bytes = {}    # by shape
        self._captured = {}      # those that graphs write to
        self._capture_ws = {}    # by capture and stream: made in the present capture

    # ---- pages ----
    def reserve(self, keep: torch.Tensor, need: torch.Tensor) -> torch.Tensor:
        """Every sequence keeps its first keep[b] tokens (no more than its pages hold) and gets pages
        of its own from there to token need[b] - 1; the rest goes back.  Returns `missing` (int32 [1]
        on the device): 0, or how many pages there were too few; nothing is changed then."""
        return K.pages_resize(self.table, self.held, self.refs, keep, need, self.pool, self.page_tokens, self._ws,
                              missing=self.missing)

    def fork(self, parent: torch.Tensor) -> None:
        """Sequence b goes on from sequence parent[b] (-1: empty).  Pages are shared until they are
        written.  `table`, `held` and `refs` are changed in place, for the graphs that read them."""
        self._old_rows.copy_(self._rows)
        K.pages_fork(self._old_table, self._old_held, self.refs, parent, table_out=self.table, held_out=self.held,
                     refs_out=self.refs)

    def compact(self) -> torch.Tensor:
        """Live pages move to the lowest numbers; returns the new number of every old one (-1: free)."""
        K.pages_compact(self.table, self.held, self.refs, self.pool, self._ws, table_out=self.table,
                        refs_out=self.refs, remap=self._remap)
        return self._remap

    def free_pages(self) -> int:
        """Free pages (reads the device)."""
        return int((self.refs == 0).sum())

    # ---- rows ----
    def append(self, layer: int, k, v, positions, tokens_per_seq: int = 1, n_tokens=None) -> None:
        K.kv4_append(k, v, self.pool[layer], self.table, positions, tokens_per_seq=tokens_per_seq, n_tokens=n_tokens)

    def read(self, layer: int, positions, k, v, tokens_per_seq: int = 1, n_tokens=None) -> None:
        K.kv4_read(self.pool[layer], self.table, positions, k, v, tokens_per_seq=tokens_per_seq, n_tokens=n_tokens)

    def attend(self, layer: int, q, positions, scale: float, tokens_per_seq: int = 1, n_tokens=None, window: int = 0,
               sinks: int = 0, out=None):
        """q [B * T, heads * head_dim] -> out, over the sequences' pages (kernels.kv4_attn).  Calls on
        different streams have different workspaces.  A captured call has the one of the stream that
        it was captured on, if an earlier call made it large enough, else one of its graph's own:
        graphs of the first kind may not be replayed at the same time."""
        ws = self._workspace(positions.numel(), tokens_per_seq, q.shape[1] // self.head_dim, q.device)
        return K.kv4_attn(q, self.pool[layer], self.table, positions, self.head_dim, ws, scale=scale,
                          tokens_per_seq=tokens_per_seq, n_tokens=n_tokens, window=window, sinks=sinks, out=out)

    def _workspace(self, B: int, T: int, nq: int, device) -> torch.Tensor:
        """The current stream's workspace, large enough for this call: calls on one stream follow one
        another and may share it."""
        shape = (B, T, nq)
        need = self._attn_bytes.get(shape)
        if need is None:
            need = self._attn_bytes[shape] = K.kv4_attn_workspace_bytes(*shape, self.num_kv_heads, self.head_dim)
        stream, capture = K._stream(), K.capture_id()
        ws = self._attn_ws.get(stream)
        if ws is not None and ws.numel() >= need:
            if capture:
                self._captured[ws.data_ptr()] = ws   # (it outlives its replacement)
            return ws
        kept, key = self._attn_ws, stream
        if capture:
            # its zero-fill is a node of this graph, so nothing outside of the graph may rely on it
            kept, key = self._capture_ws, (capture, stream)
            ws = kept.get(key)
            if ws is not None and ws.numel() >= need:
                return ws
            for old in [k for k in kept if k[0] != capture]:
                del kept[old]
        # (whole megabytes: lengths near one another need a few bytes more or less)
        ws = kept[key] = K.kv4_attn_workspace(*shape, self.num_kv_heads, self.head_dim, device,
                                              at_least=(need + 0xfffff) >> 20 << 20)
        return ws
