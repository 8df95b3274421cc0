"""A batch of requests whose bookkeeping lives on the GPU.

``PagedKVCache`` keeps block tables and lengths in Python lists and uploads
index tensors step by step. ``PackedBatch`` keeps them in device tensors:
one ``advance_batch`` launch per step takes pages from a ring of free ones,
extends the block tables and writes the step's slots, positions, sequence
starts and lengths, so nothing is built on the host, nothing is read back,
and steps can be captured into a graph. Attention is packed (requests bring
any number of new tokens each) and grouped (fewer key heads than query
heads): ``prompt_attention`` where all requests are new, ``packed_attention``
over the cache else. It can keep count of the attention weight that each
cached token gets and take those of least weight out (``compact``).
``LatentBatch`` is the same over a latent cache.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

import memopt_C

from .kv_cache import pages_needed


class _Requests:
    """Block tables, lengths and the ring of free pages of ``num_requests`` requests, on the device."""

    def _start(self, name: str, pages: Sequence[int], num_requests: int, max_tokens: int, num_rows: int, block_size: int,
               dev: torch.device) -> None:
        self._name = name
        self.block_size = block_size
        self.max_tokens = max_tokens
        self.free_pages = torch.tensor(pages, dtype=torch.int32, device=dev)
        self.tables = torch.full((num_requests, pages_needed(max_tokens, block_size)), -1, dtype=torch.int32, device=dev)
        # context_lens and free_span are advanced in place.
        self.state = memopt_C.advance_batch_buffers(num_requests, num_rows, dev)
        for t in (self.state.context_lens, self.state.cu_seqlens, self.state.status):
            t.zero_()
        for t in (self.state.slots, self.state.positions):
            t.fill_(-1)
        self.state.free_span.copy_(torch.tensor([0, len(pages)], dtype=torch.int32))

    @staticmethod
    def _check_sizes(name: str, num_blocks: int, block_size: int, num_requests: int, max_tokens: int, num_rows: int) -> None:
        if num_blocks <= 0 or block_size <= 0 or num_blocks * block_size > 2 ** 31:
            raise RuntimeError(f"{name}: the pool must hold 1 to 2^31 tokens (slots are int32)")
        if not 0 < num_requests <= 4096:
            raise RuntimeError(f"{name}: num_requests must be 1 to 4096")
        if max_tokens <= 0 or num_rows <= 0:
            raise RuntimeError(f"{name}: max_tokens and num_rows must be positive")

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

    def _rows_of(self, query: torch.Tensor) -> None:
        if query.shape[0] != self.num_rows:
            raise RuntimeError(f"{self._name}: query has {query.shape[0]} rows, not num_rows={self.num_rows}")

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
            raise RuntimeError(f"{self._name}: no such request")
        return requests

    def _give_back(self, pages: List[int]) -> None:
        """Append ``pages`` to the ring."""
        head, count = self.state.free_span.tolist()
        at = (head + count + torch.arange(len(pages))) % self.free_pages.shape[0]
        dev = self.free_pages.device
        self.free_pages[at.to(dev)] = torch.tensor(pages, dtype=torch.int32, device=dev)
        self.state.free_span[1] = count + len(pages)


class PackedBatch(_Requests):
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
        track_weights: keep ``weights`` f32 ``[num_requests, num_kv_heads,
            positions]``, what ``accumulate`` adds up and ``compact`` goes by.

    A step is ``advance(new_tokens)`` (which tokens of which requests come,
    decided by the caller), then ``attend(query, keys, values)`` with their
    rows. The pool is the process-wide one: one ``PackedBatch`` or
    ``PagedKVCache`` at a time.
    """

    def __init__(self, num_blocks: int, num_kv_heads: int, head_dim: int, num_requests: int, max_tokens: int,
                 num_rows: int, block_size: int = 16, kv_format: str = "int4", window_size: int = -1,
                 num_sink_tokens: int = 0, track_weights: bool = False) -> None:
        self._check_sizes("PackedBatch", num_blocks, block_size, num_requests, max_tokens, num_rows)
        if head_dim not in (64, 128) or block_size % 16 or (kv_format == "int4" and block_size != 16):
            raise RuntimeError("PackedBatch: head_dim must be 64 or 128, pages 16 tokens (fp16: a multiple of 16)")
        memopt_C.reset_pool()
        memopt_C.init_pool(num_blocks, block_size, num_kv_heads, head_dim, kv_format=kv_format)
        self.window_size = window_size
        self.num_sink_tokens = num_sink_tokens
        dev = memopt_C.get_key_pool().device
        # The pages leave the host's free list for a ring on the device.
        self._start("PackedBatch", memopt_C.allocate_blocks(num_blocks), num_requests, max_tokens, num_rows, block_size, dev)
        positions = self.tables.shape[1] * block_size
        self.weights = torch.zeros((num_requests, num_kv_heads, positions), device=dev) if track_weights else None
        # Tokens that compaction took out of each request: what its positions lack.
        self.removed = torch.zeros(num_requests, dtype=torch.int32, device=dev)

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
        self._rows_of(query)
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

    def accumulate(self, query: torch.Tensor, max_new: Optional[int] = None) -> torch.Tensor:
        """Add to ``weights`` what the step's queries (as in ``attend``, which
        comes first) give each cached token; returns it. Every step, or only
        where a prompt ends, as the policy has it. ``max_new``: at least the
        most rows of a request; steps of few tokens a request (16 rows per key
        head) are two to four times as fast where it says so."""
        if self.weights is None:
            raise RuntimeError("PackedBatch: made without track_weights")
        self._rows_of(query)
        return memopt_C.attention_scores(query, memopt_C.get_key_pool(), self.tables, self.state.context_lens,
                                         self.state.cu_seqlens, self.num_rows if max_new is None else max_new,
                                         self.max_tokens, self.window_size, num_sink_tokens=self.num_sink_tokens,
                                         scores=self.weights, out=self.weights)

    def compact(self, requests: Sequence[int], keep: int, num_sink_tokens: int = 4, num_recent_tokens: int = 0) -> List[int]:
        """Cut the requests to ``keep`` tokens per head, those of most weight (``compact_cache``); returns the
        requests that now have their tokens in fresh pages.

        Old pages go back to the ring. A request that has no more than
        ``keep`` stays as it is. The fresh pages come from the ring while the
        old ones are still taken: where they do not last for all, the others
        are compacted into what the first gave back, and where they do not
        last for one, all stay. Tokens that come later stand behind the ``keep``
        (``token_positions`` says where they stand in the text). It belongs
        behind a step's ``attend`` and ``accumulate``, before the next
        ``advance``: the step's slots lie in pages that it gives back. (Waits
        for the device.)
        """
        if self.weights is None:
            raise RuntimeError("PackedBatch: made without track_weights")
        requests = self._known(requests)
        if len(set(requests)) != len(requests):
            raise RuntimeError("PackedBatch: a request is named twice")
        if keep < 0:
            raise RuntimeError("PackedBatch: keep must not be negative")
        done: List[int] = []
        todo, limit = requests, min(keep, self.weights.shape[2])
        while todo:
            rows = torch.tensor(todo, dtype=torch.int64, device=self.tables.device)
            want = torch.full((len(todo),), limit, dtype=torch.int32, device=self.tables.device)
            lens = self.state.context_lens[rows]
            r = memopt_C.compact_cache(self.weights[rows], memopt_C.get_key_pool(), memopt_C.get_value_pool(), self.tables[rows],
                                       lens, want, self.free_pages, self.state.free_span, num_sink_tokens=num_sink_tokens,
                                       num_recent_tokens=num_recent_tokens, max_keep=limit)
            self.tables[rows] = r.block_tables
            self.state.context_lens[rows] = r.context_lens
            self.weights[rows] = r.scores
            self.removed[rows] += lens - r.context_lens
            self.state.free_span.copy_(r.free_span)
            status = r.status.tolist()
            served = [b for b, s in zip(todo, status) if s == 0]
            done += served
            # Those refused are tried again over what the others gave back. All ask for as many fresh pages, and the ring
            # takes any old ones: where the first finds no room, none does.
            todo = [b for b, s in zip(todo, status) if s == 3] if served else []
        return done

    def token_positions(self) -> torch.Tensor:
        """Where the rows of the last ``advance`` stand in their texts (int32 ``[num_rows]``): ``state.positions``, which
        count cached tokens, plus the tokens that compaction had taken out by then; -1 behind the last row, and for rows
        of requests released since."""
        rows = torch.arange(self.num_rows, dtype=torch.int32, device=self.tables.device)
        owner = (torch.searchsorted(self.state.cu_seqlens, rows, right=True) - 1).clamp(0, self.removed.shape[0] - 1)
        # A text ends with its request's last row. Its length, what is cached and what was removed, is the same before and
        # after a compaction; `positions` beside `removed` are not.
        text = (self.state.context_lens + self.removed)[owner]
        at = text - (self.state.cu_seqlens[1:][owner] - rows)
        return torch.where((self.state.positions >= 0) & (at >= 0), at, -1)

    def release(self, requests: Sequence[int]) -> None:
        requests = self._known(requests)  # (once: an iterator is spent then)
        super().release(requests)
        rows = torch.tensor(requests, dtype=torch.int64, device=self.tables.device)
        self.removed[rows] = 0
        if self.weights is not None:
            self.weights[rows] = 0.0


class LatentBatch(_Requests):
    """``num_requests`` requests of one layer of latent attention.

    The cache is this object's own (``cache`` ``[num_blocks, block_size, rank
    + rope_dim]``, one row per token for all heads), not the ``memopt_C`` pool.

    Args:
        num_blocks, rank, rope_dim, block_size, dtype, device: the cache; rank
            128, 256 or 512, rope_dim 32 or 64, pages of a multiple of 16
            tokens, fp16 or bf16 (device: the current one).
        num_requests, max_tokens, num_rows, window_size, num_sink_tokens: as in ``PackedBatch``.

    A step is ``advance(new_tokens)``, then ``attend`` (or, where every
    request with rows is new, ``attend_prompts``) with their rows.
    """

    def __init__(self, num_blocks: int, rank: int, rope_dim: int, num_requests: int, max_tokens: int, num_rows: int,
                 block_size: int = 16, dtype: torch.dtype = torch.bfloat16, window_size: int = -1,
                 num_sink_tokens: int = 0, device: Optional[torch.device] = None) -> None:
        self._check_sizes("LatentBatch", num_blocks, block_size, num_requests, max_tokens, num_rows)
        if rank not in (128, 256, 512) or rope_dim not in (32, 64) or block_size % 16:
            raise RuntimeError("LatentBatch: rank must be 128, 256 or 512, rope_dim 32 or 64, pages a multiple of 16 tokens")
        if dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError("LatentBatch: dtype must be fp16 or bf16")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.rank = rank
        self.window_size = window_size
        self.num_sink_tokens = num_sink_tokens
        self.cache = torch.zeros((num_blocks, block_size, rank + rope_dim), dtype=dtype, device=dev)
        self._start("LatentBatch", range(num_blocks), num_requests, max_tokens, num_rows, block_size, dev)

    def attend(self, query: torch.Tensor, latents: torch.Tensor, rope_keys: torch.Tensor, scale: float,
               max_new: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Write the step's latents ``[num_rows, rank]`` and rotary keys
        ``[num_rows, rope_dim]`` and attend over the cache (``latent_attention``);
        returns ``[num_rows, Hq, rank]``. ``max_new``: at least the most rows
        of a request (default: num_rows)."""
        self._rows_of(query)
        memopt_C.write_latent(latents, rope_keys, self.state.slots, self.cache)
        return memopt_C.latent_attention(query, self.cache, self.tables, self.state.context_lens, self.state.cu_seqlens,
                                         self.num_rows if max_new is None else max_new, self.max_tokens, scale, self.rank,
                                         self.window_size, num_sink_tokens=self.num_sink_tokens, out=out)

    def attend_prompts(self, query: torch.Tensor, keys: torch.Tensor, latents: torch.Tensor, rope_keys: torch.Tensor,
                       values: torch.Tensor, scale: Optional[float] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The same where every request with rows is new: attention from the
        heads' own ``keys`` and ``values`` (``latent_prompt_attention``);
        returns ``[num_rows, H, head_dim]``."""
        self._rows_of(query)
        memopt_C.write_latent(latents, rope_keys, self.state.slots, self.cache)
        return memopt_C.latent_prompt_attention(query, keys, rope_keys, values, self.state.cu_seqlens, self.window_size,
                                                num_sink_tokens=self.num_sink_tokens, scale=scale, out=out)
