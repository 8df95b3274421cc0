"""A batch of requests whose bookkeeping lives on the GPU.

``PagedKVCache`` keeps block tables and lengths in Python lists and uploads
index tensors step by step. ``PackedBatch`` keeps them in device tensors:
one ``advance_batch`` launch per step takes pages from a ring of free ones,
extends the block tables and writes the step's slots, positions, sequence
starts and lengths, so nothing is built on the host, nothing is read back,
and steps can be captured into a graph. Attention is packed (requests bring
any number of new tokens each) and grouped (fewer key heads than query
heads): ``prompt_attention`` where all requests are new, ``packed_attention``
over the cache else.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

import memopt_C

from .kv_cache import pages_needed


class PackedBatch:
    """``num_requests`` requests of one attention layer over the ``memopt_C`` pool.

    Args:
        num_blocks, num_kv_heads, head_dim, block_size, kv_format: the pool
            (``init_pool``); 64 or 128 dims, 16-token pages (fp16 pools: a
            multiple of 16). Any pool before is dropped.
        num_requests: requests, live or free, at most 4096; a request is an
            index ``0 .. num_requests - 1``.
        max_tokens: the longest context that a request may reach.
        num_rows: new tokens that one step may bring, of all requests together.
        window_size, num_sink_tokens: the layer's mask (``dynamic_sparse_attention``).

    A step is ``advance(new_tokens)`` (which tokens of which requests come,
    decided by the caller), then ``attend(query, keys, values)`` with their
    rows. The pool is the process-wide one: one ``PackedBatch`` or
    ``PagedKVCache`` at a time.
    """

    def __init__(self, num_blocks: int, num_kv_heads: int, head_dim: int, num_requests: int, max_tokens: int,
                 num_rows: int, block_size: int = 16, kv_format: str = "int4", window_size: int = -1,
                 num_sink_tokens: int = 0) -> None:
        if num_blocks <= 0 or block_size <= 0 or num_blocks * block_size > 2 ** 31:
            raise RuntimeError("PackedBatch: the pool must hold 1 to 2^31 tokens (slots are int32)")
        if not 0 < num_requests <= 4096:
            raise RuntimeError("PackedBatch: num_requests must be 1 to 4096")
        if max_tokens <= 0 or num_rows <= 0:
            raise RuntimeError("PackedBatch: max_tokens and num_rows must be positive")
        if head_dim not in (64, 128) or block_size % 16 or (kv_format == "int4" and block_size != 16):
            raise RuntimeError("PackedBatch: head_dim must be 64 or 128, pages 16 tokens (fp16: a multiple of 16)")
        memopt_C.reset_pool()
        memopt_C.init_pool(num_blocks, block_size, num_kv_heads, head_dim, kv_format=kv_format)
        self.block_size = block_size
        self.max_tokens = max_tokens
        self.window_size = window_size
        self.num_sink_tokens = num_sink_tokens
        dev = memopt_C.get_key_pool().device
        # The pages leave the host's free list for a ring on the device.
        self.free_pages = torch.tensor(memopt_C.allocate_blocks(num_blocks), dtype=torch.int32, device=dev)
        self.tables = torch.full((num_requests, pages_needed(max_tokens, block_size)), -1, dtype=torch.int32, device=dev)
        # context_lens and free_span are advanced in place.
        self.state = memopt_C.advance_batch_buffers(num_requests, num_rows, dev)
        for t in (self.state.context_lens, self.state.cu_seqlens, self.state.status):
            t.zero_()
        for t in (self.state.slots, self.state.positions):
            t.fill_(-1)
        self.state.free_span.copy_(torch.tensor([0, num_blocks], dtype=torch.int32))

    @property
    def num_rows(self) -> int:
        return self.state.slots.shape[0]

    def advance(self, new_tokens: torch.Tensor) -> "memopt_C.BatchStep":
        """Make room for ``new_tokens`` (int32 ``[num_requests]`` on the device).

        Returns the step's index tensors, which the next step overwrites:
        ``status`` (0: served; a request that is refused brings no rows and
        stays as it was), ``cu_seqlens`` (request r's rows), ``positions`` of
        the rows, ``context_lens`` with the new tokens.
        """
        return memopt_C.advance_batch(new_tokens, self.state.context_lens, self.tables, self.free_pages,
                                      self.state.free_span, self.block_size, out=self.state)

    def attend(self, query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, max_new: Optional[int] = None,
               prompts: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Write the step's keys and values and attend; returns ``[num_rows, Hq, D]``.

        ``query`` ``[num_rows, Hq, D]``, ``keys`` / ``values`` ``[num_rows,
        num_kv_heads, D]``: fp16, the rows of the last ``advance``; those past
        the last request's are not looked at, and ``out`` keeps them.
        ``max_new``: at least the most rows of a request (default: num_rows).
        ``prompts``: every request with rows is new, so attention reads the
        rows themselves, not their quantized copies.
        """
        if query.shape[0] != self.num_rows:
            raise RuntimeError(f"PackedBatch: query has {query.shape[0]} rows, not num_rows={self.num_rows}")
        memopt_C.write_cache(keys, values, None, self.state.slots, validate_slots=False)
        if prompts:
            return memopt_C.prompt_attention(query, keys, values, self.state.cu_seqlens, self.window_size,
                                             num_sink_tokens=self.num_sink_tokens, out=out)
        k, v = memopt_C.get_key_pool(), memopt_C.get_value_pool()
        return memopt_C.packed_attention(query, k, v, self.tables, self.state.context_lens, self.state.cu_seqlens,
                                         self.num_rows if max_new is None else max_new, self.max_tokens,
                                         self.window_size, num_sink_tokens=self.num_sink_tokens, out=out)

    def attend_plan(self, query: torch.Tensor, max_new: Optional[int] = None,
                    out: Optional[torch.Tensor] = None) -> "memopt_C.PreparedPackedAttention":
        """The attention of ``attend`` as a plan over this ``query`` tensor, for loops and graphs."""
        return memopt_C.PreparedPackedAttention(query, memopt_C.get_key_pool(), memopt_C.get_value_pool(), self.tables,
                                                self.state.context_lens, self.state.cu_seqlens,
                                                self.num_rows if max_new is None else max_new, self.max_tokens,
                                                self.window_size, num_sink_tokens=self.num_sink_tokens, out=out)

    def evict(self, requests: Sequence[int], scores: torch.Tensor, retain_ratio: float,
              num_sink_tokens: int = 4) -> List[int]:
        """Ada-KV eviction of the requests' tokens; pages that it unlinks go back to the ring.

        ``scores``: f32 ``[requests, num_kv_heads, L]`` over the first L
        positions, which every one of them holds (``evict_tokens``). Unlinked
        pages stay as holes (-1) in the block tables, which attention skips.
        Returns the freed pages, in ring order. (Waits for the device.
        ``free_evicted_blocks`` would give them to the pool's own free list,
        which this class does not use.)
        """
        requests = self._known(requests)
        if len(set(requests)) != len(requests):
            raise RuntimeError("PackedBatch: a request is named twice")
        if scores.dim() != 3 or scores.shape[0] != len(requests):
            raise RuntimeError(f"PackedBatch: scores must be [{len(requests)}, kv heads, positions]")
        if not requests:
            return []
        rows = torch.tensor(requests, dtype=torch.int64, device=self.tables.device)
        least = int(self.state.context_lens[rows].min())
        if scores.shape[2] > least:
            raise RuntimeError(f"PackedBatch: scores of {scores.shape[2]} positions, where a request holds {least}")
        tables = self.tables[rows]
        votes = torch.zeros_like(self.free_pages)
        memopt_C.evict_tokens(scores, tables, votes, retain_ratio, num_sink_tokens)
        self.tables[rows] = tables
        freed = torch.nonzero(votes == scores.shape[1]).flatten().tolist()
        self._give_back(freed)
        return freed

    def release(self, requests: Sequence[int]) -> None:
        """Return the requests' linked pages to the ring; their indices are free
        for new requests. (Waits for the device: the pages are read back.)"""
        requests = list(dict.fromkeys(self._known(requests)))
        if not requests:
            return
        rows = torch.tensor(requests, dtype=torch.int64, device=self.tables.device)
        tables, lens = self.tables[rows].cpu(), self.state.context_lens[rows].cpu()
        self._give_back([p for t, n in zip(tables.tolist(), lens.tolist())
                         for p in t[:pages_needed(n, self.block_size)] if p >= 0])
        self.tables[rows] = -1
        self.state.context_lens[rows] = 0

    def _known(self, requests: Sequence[int]) -> List[int]:
        requests = [int(r) for r in requests]
        if any(not 0 <= r < self.tables.shape[0] for r in requests):
            raise RuntimeError("PackedBatch: no such request")
        return requests

    def _give_back(self, pages: List[int]) -> None:
        """Append ``pages`` to the ring."""
        head, count = self.state.free_span.tolist()
        at = (head + count + torch.arange(len(pages))) % self.free_pages.shape[0]
        dev = self.free_pages.device
        self.free_pages[at.to(dev)] = torch.tensor(pages, dtype=torch.int32, device=dev)
        self.state.free_span[1] = count + len(pages)
