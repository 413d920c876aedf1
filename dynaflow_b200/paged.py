"""A key/value cache in pages of 4-bit codes: the buffers that the paged operators of ``ops`` share.

A request holds as many pages as its tokens need instead of a row of ``max_len`` positions, and a token takes 136 bytes a
key/value head instead of 512 (bf16). One page table, free list and set of row buffers serves all layers: ``plan`` once a step,
then ``append`` and ``attend`` a layer. The reference leaves the cache to the host engine and swaps the per-nano-batch
attention metadata before each operator (``examples/ae/scheduler/vllm/nanoflow.py:231``); here that metadata is this object's.
"""
from __future__ import annotations

import torch

from . import ops


class PagedKVCache4:
    def __init__(self, layers: int, kv_heads: int, *, num_pages: int, page_size: int, max_requests: int, max_len: int,
                 max_rows: int, rope_theta: float = 10000.0, device: torch.device | str = "cuda") -> None:
        """``num_pages`` pages of ``page_size`` tokens in every layer, for at most ``max_requests`` requests of at most
        ``max_len`` tokens (in whole pages: what the last one holds past ``max_len`` can be used, a longer request is reported) and
        steps of at most ``max_rows`` rows."""
        if layers <= 0 or max_requests <= 0 or max_len <= 0 or max_rows <= 0:
            raise ValueError("layers, max_requests, max_len and max_rows must be positive")
        self.page_size, self.kv_heads = page_size, kv_heads
        self.layers = [ops.paged4_cache(num_pages, kv_heads, page_size, device) for _ in range(layers)]
        i32 = dict(dtype=torch.int32, device=device)
        self.page_table = torch.full((max_requests, -(-max_len // page_size)), -1, **i32)
        self.page_counts = torch.zeros(max_requests, **i32)
        self.free_pages = torch.arange(num_pages, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)
        self.row_starts = torch.zeros(max_requests + 1, **i32)
        self.slots = torch.full((max_rows,), -1, **i32)
        self.positions = torch.zeros(max_rows, **i32)
        self.angles = ops.rope_angles(self.page_table.shape[1] * page_size, rope_theta, device)   # whatever position a page gives a slot

    def plan(self, seq_lens: torch.Tensor, new_lens: torch.Tensor, rows_per_request: int = 0) -> None:
        """Pages, slots and positions of a step (``ops.page_plan``): ``seq_lens`` the requests' lengths after it, ``new_lens`` how
        many of the tokens are new; a length of 0 gives a request's pages back. The new tokens' rows lie back to back, or request
        ``b``'s from row ``b * rows_per_request`` on."""
        ops.page_plan(seq_lens, new_lens, self.page_table, self.page_counts, self.free_pages, self.free_count, self.row_starts,
                      self.slots, self.positions, page_size=self.page_size, rows_per_request=rows_per_request)

    def append(self, layer: int, qkv: torch.Tensor, q_heads: int, first_row: int = 0) -> None:
        """Rotary embedding and quantising append of ``qkv`` (the step's rows from ``first_row``) in place, one launch."""
        rows = slice(first_row, first_row + qkv.shape[0])
        ops.rope_append_paged4(qkv, self.positions[rows], self.slots[rows], self.angles, q_heads, self.kv_heads, self.layers[layer],
                               page_size=self.page_size)

    def attend(self, layer: int, q: torch.Tensor, out: torch.Tensor, workspace: torch.Tensor, seq_lens: torch.Tensor,
               first_request: int = 0, max_ctas: int = 0, *, new_lens: torch.Tensor | None = None, max_new: int = 1) -> torch.Tensor:
        """Attention of the new tokens of requests ``first_request ...`` (as many as ``seq_lens``, their lengths, has). Without
        ``new_lens`` row ``i`` of ``q`` is the last token of request ``first_request + i``, as a plan with ``rows_per_request=1`` lays a
        step out. With ``new_lens``, the plan's of these requests, ``q`` and ``out`` are all of the step's rows, and a request's, at most
        ``max_new``, are where the plan put them: any other layout needs it, since a request without a new token has no row there."""
        requests = slice(first_request, first_request + seq_lens.shape[0])
        starts = None if new_lens is None else self.row_starts[requests.start:requests.stop + 1]
        return ops.attention_paged4(q, self.layers[layer], self.page_table[requests], seq_lens, out, workspace, page_size=self.page_size,
                                    max_ctas=max_ctas, row_starts=starts, new_lens=new_lens, max_new=max_new)
