"""memopt_C — drop-in for the reference's pybind11 extension, backed by gfx950 HIP.

Same module name, function names, argument order/keywords, return types and
error type (``RuntimeError``) as TheRadDani/memopt-transformer-runtime
``src/csrc/extension.cpp:10-124``, so ``memopt.DynamicAttention`` and the
reference tests run unchanged against it. Calls go through the C ABI of
``libmemopt_hip.so`` (declared in ``include/memopt_hip.h``); torch is used only
to allocate device tensors and to pass the current HIP stream.

Additions (new names or keyword-only arguments whose defaults keep the
reference behaviour):
  * ``get_key_pool()`` / ``get_value_pool()`` — called by the reference's
    ``DynamicAttention`` (src/memopt/attention.py:330-331) but missing from
    its extension;
  * ``init_pool(..., kv_format="int4")`` — INT4 page pool: one u8 buffer
    [nb, H, 17*D] of (page, head) blocks holding K codes, V codes, K scales
    and V scales (layout in csrc/page_format.hpp); ``write_cache`` then
    quantizes on the fly, ``get_int4_pages()`` returns the buffer and
    ``get_pool_scales()`` the fp16 scale regions;
  * ``dynamic_sparse_attention(..., *, num_sink_tokens=0, causal=False,
    key_scales=None, value_scales=None, kv_layout=None)`` — INT4 caches are
    dequantized just in time inside the kernel;
  * ``free_evicted_blocks(is_block_free)`` — the post-eviction sweep the
    reference documents but never implements (src/csrc/kv_cache.cu:1033-1036);
  * ``prompt_attention``, ``packed_attention`` / ``PreparedPackedAttention``
    and ``advance_batch`` — packed batches with grouped heads: whole prompts
    straight from q, k and v, the paged cache, and a step's index tensors;
  * ``attention_scores`` and ``compact_cache`` — attention weights added up
    per cached token, and the tokens of least weight taken out of the cache;
  * ``write_latent``, ``latent_attention`` and ``latent_prompt_attention`` —
    a cache of one latent row per token for all heads, attention over it, and
    over whole prompts from the expanded keys and values.

The library is loaded at import; a missing or unloadable library raises
``ImportError`` naming the path (there is no CPU fallback).
"""
from __future__ import annotations

import contextlib
import ctypes
import os
import struct
import threading
from typing import List, Optional, Sequence, Tuple

import torch  # must precede the HIP library so both share one HIP runtime

__all__ = [
    "get_hello", "init_pool", "allocate_block", "free_block", "get_pool_tensors",
    "get_key_pool", "get_value_pool", "get_pool_scales", "get_int4_pages", "int4_layout", "free_blocks_count",
    "write_cache", "evict_cache", "evict_tokens", "free_evicted_blocks",
    "dynamic_sparse_attention", "PreparedAttention", "quantize_kv_cache_int4", "dequantize_kv_cache_int4",
    "prompt_attention", "packed_attention", "packed_workspace_bytes", "PreparedPackedAttention", "advance_batch", "advance_batch_buffers",
    "BatchStep", "attention_scores", "compact_cache", "compact_cache_buffers", "CompactStep", "write_latent", "latent_attention",
    "latent_prompt_attention", "library_path",
]

_HERE = os.path.dirname(os.path.abspath(__file__))
library_path = os.environ.get("MEMOPT_HIP_LIB", os.path.join(_HERE, "libmemopt_hip.so"))

if not os.path.exists(library_path):
    raise ImportError(
        f"memopt_C: {library_path} is missing; build it with "
        "`python memopt-transformer-runtime_amd/build.py` (there is no CPU fallback)")
try:
    _lib = ctypes.CDLL(library_path)
except OSError as exc:  # pragma: no cover - environment specific
    raise ImportError(f"memopt_C: cannot load {library_path}: {exc}") from exc

_i32, _i64, _f32, _vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p


class AttnDesc(ctypes.Structure):
    """Mirror of ``memopt_attn_desc`` (include/memopt_hip.h)."""

    _fields_ = [
        ("query", _vp), ("out", _vp),
        ("batch", _i32), ("q_len", _i32), ("num_heads", _i32), ("head_dim", _i32),
        ("kv_format", _i32),
        ("key_cache", _vp), ("value_cache", _vp), ("key_scales", _vp), ("value_scales", _vp),
        ("scale_dtype", _i32), ("block_size", _i32), ("num_kv_blocks", _i64),
        ("kv_page_stride", _i64), ("kv_head_stride", _i64), ("kv_token_stride", _i64),
        ("sc_page_stride", _i64), ("sc_head_stride", _i64), ("sc_token_stride", _i64),
        ("block_tables", _vp), ("max_blocks_per_seq", _i32), ("context_lens", _vp),
        ("max_seq_len", _i32), ("window_size", _i32), ("num_sink_tokens", _i32), ("causal", _i32),
        ("workspace", _vp), ("workspace_bytes", _i64),
    ]


class PromptDesc(ctypes.Structure):
    """Mirror of ``memopt_prompt_desc`` (include/memopt_hip.h)."""

    _fields_ = [
        ("query", _vp), ("key", _vp), ("value", _vp), ("out", _vp),
        ("dtype", _i32), ("tokens", _i32), ("batch", _i32), ("num_heads", _i32), ("num_kv_heads", _i32),
        ("head_dim", _i32),
        ("q_token_stride", _i64), ("q_head_stride", _i64), ("k_token_stride", _i64), ("k_head_stride", _i64),
        ("v_token_stride", _i64), ("v_head_stride", _i64), ("o_token_stride", _i64), ("o_head_stride", _i64),
        ("query_starts", _vp), ("window_size", _i32), ("num_sink_tokens", _i32),
    ]


class PackedDesc(ctypes.Structure):
    """Mirror of ``memopt_packed_desc`` (include/memopt_hip.h)."""

    _fields_ = [
        ("query", _vp), ("out", _vp),
        ("tokens", _i32), ("batch", _i32), ("num_heads", _i32), ("num_kv_heads", _i32), ("head_dim", _i32),
        ("q_token_stride", _i64), ("q_head_stride", _i64), ("o_token_stride", _i64), ("o_head_stride", _i64),
        ("kv_format", _i32), ("key_cache", _vp), ("value_cache", _vp), ("block_size", _i32), ("num_kv_blocks", _i64),
        ("block_tables", _vp), ("max_blocks_per_seq", _i32), ("context_lens", _vp), ("query_starts", _vp),
        ("max_query_len", _i32), ("max_seq_len", _i32), ("window_size", _i32), ("num_sink_tokens", _i32),
        ("workspace", _vp), ("workspace_bytes", _i64),
    ]


def _sig(name, args, res=_i32):
    f = getattr(_lib, name)
    f.argtypes = args
    f.restype = res
    return f


_lib.memopt_last_error.restype = ctypes.c_char_p
_lib.memopt_get_hello.restype = ctypes.c_char_p
_c_init_pool = _sig("memopt_init_pool", [_i64, _i32, _i32, _i32, _i32, _vp, _vp, _vp, _vp])
_c_pool_info = _sig("memopt_pool_info", [ctypes.POINTER(_i64)] + [ctypes.POINTER(_i32)] * 4)
_c_reset_pool = _sig("memopt_reset_pool", [])
_c_set_storage = _sig("memopt_pool_set_storage", [_i32, _vp, _vp])
_c_pages_to_fp16 = _sig("memopt_int4_pages_to_fp16", [_vp, _i64, _i32, _i32, _vp, _vp, _vp])
_c_alloc = _sig("memopt_allocate_block", [ctypes.POINTER(_i64)])
_c_free = _sig("memopt_free_block", [_i64])
_c_alloc_n = _sig("memopt_allocate_blocks", [_i64, ctypes.POINTER(_i64)])
_c_free_n = _sig("memopt_free_blocks", [_i64, ctypes.POINTER(_i64)])
_c_free_count = _sig("memopt_free_blocks_count", [ctypes.POINTER(_i64)])
_c_write = _sig("memopt_write_cache", [_vp, _vp, _i64, _i32, _i32, _vp, _vp])
_c_evict_cache = _sig("memopt_evict_cache", [_vp, _i64, _f32, _i32, _vp])
_c_evict_tokens = _sig("memopt_evict_tokens",
                       [_vp, _i32, _i32, _i32, _vp, _i32, _vp, _i64, _f32, _i32, _vp, _i64, _vp])
_c_evict_ws = _sig("memopt_evict_workspace_size", [_i32, _i32, _i32, _i32, _i64, ctypes.POINTER(_i64)])
_c_quant = _sig("memopt_quantize_kv_cache_int4", [_vp, _i64, _i64, _i32, _vp, _vp, _vp])
_c_dequant = _sig("memopt_dequantize_kv_cache_int4", [_vp, _i64, _vp, _i64, _i32, _vp, _vp])
_c_dsa = _sig("memopt_dynamic_sparse_attention",
              [_vp, _i32, _i32, _i32, _i32, _vp, _vp, _i64, _i32, _vp, _i32, _vp, _i32, _i32, _vp, _vp])
_c_ws = _sig("memopt_attention_workspace_size", [ctypes.POINTER(AttnDesc), ctypes.POINTER(_i64)])
_c_attn = _sig("memopt_paged_attention", [ctypes.POINTER(AttnDesc), _vp])
_c_attn_noalloc = _sig("memopt_paged_attention_noalloc", [ctypes.POINTER(AttnDesc), _vp])
_c_prompt = _sig("memopt_prompt_attention", [ctypes.POINTER(PromptDesc), _vp])
_c_packed_ws = _sig("memopt_packed_workspace_size",
                    [ctypes.POINTER(PackedDesc), ctypes.POINTER(_i64), ctypes.POINTER(_i64)])
_c_packed = _sig("memopt_packed_attention", [ctypes.POINTER(PackedDesc), _vp])
_c_advance = _sig("memopt_advance_batch", [ctypes.c_char_p, _vp])
_c_scores_ws = _sig("memopt_scores_workspace_size", [ctypes.c_char_p, ctypes.POINTER(_i64)])
_c_scores = _sig("memopt_attention_scores", [ctypes.c_char_p, _vp])
_c_compact_ws = _sig("memopt_compact_workspace_size", [ctypes.c_char_p, ctypes.POINTER(_i64)])
_c_compact = _sig("memopt_compact_cache", [ctypes.c_char_p, _vp])
_c_latent_ws = _sig("memopt_latent_workspace_size", [ctypes.c_char_p, ctypes.POINTER(_i64)])
_c_latent = _sig("memopt_latent_attention", [ctypes.c_char_p, _vp])
_c_latent_prompt = _sig("memopt_latent_prompt_attention", [ctypes.c_char_p, _vp])
_c_write_latent = _sig("memopt_write_latent", [_vp, _i64, _vp, _i64, _i32, _i32, _i32, _vp, _vp, _i64, _vp])

KV_FP16, KV_INT4, KV_INT4_ROWS = 0, 1, 2
_FORMATS = {"fp16": KV_FP16, "int4": KV_INT4}


def _check(rc: int) -> None:
    if rc != 0:
        raise RuntimeError(_lib.memopt_last_error().decode())


def _stream(t: torch.Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.device.index)


_SAME_DEVICE = contextlib.nullcontext()


def _on(device: torch.device):
    """``torch.cuda.device(device)``, or nothing to enter where it is current already."""
    return _SAME_DEVICE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _cuda(t: torch.Tensor, name: str, fn: str) -> None:
    _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{fn}: {name} must be a CUDA tensor")


# ---------------------------------------------------------------------------
# Handshake
# ---------------------------------------------------------------------------

def get_hello() -> str:
    """src/csrc/extension.cpp:6-8 (string carries "MemOpt C++ Backend Initialized")."""
    return _lib.memopt_get_hello().decode()


# ---------------------------------------------------------------------------
# Pool — src/csrc/kv_cache.cu:83-201
# ---------------------------------------------------------------------------

_pool_lock = threading.Lock()
_pool: dict = {}


def init_pool(num_blocks: int, block_size: int, num_heads: int, head_dim: int,
              kv_format: str = "fp16") -> None:
    """Allocate zeroed pool storage on the current device and seed the FIFO free list.

    Idempotent for identical parameters (src/csrc/kv_cache.cu:115-122);
    different parameters reset the pool. Invalid parameters raise
    ``RuntimeError`` and leave no pool behind.
    """
    fmt = _FORMATS.get(kv_format)
    _require(fmt is not None, f"init_pool: kv_format must be one of {sorted(_FORMATS)}")
    with _pool_lock:
        nb, bs, h, d, f = _i64(), _i32(), _i32(), _i32(), _i32()
        if _c_pool_info(ctypes.byref(nb), ctypes.byref(bs), ctypes.byref(h), ctypes.byref(d), ctypes.byref(f)):
            if (nb.value, bs.value, h.value, d.value, f.value) == (num_blocks, block_size, num_heads, head_dim, fmt):
                return
        _pool.clear()
        _c_reset_pool()
        ok = num_blocks > 0 and block_size > 0 and num_heads > 0 and head_dim > 0 and head_dim % 2 == 0
        if not ok or (fmt == KV_INT4 and head_dim % 64):
            # Let the library produce the reference's message (and stay torn down).
            _check(_c_init_pool(num_blocks, block_size, num_heads, head_dim, fmt, 1, 1, 1, 1))
        if fmt == KV_INT4 and block_size != 16:
            _check(_c_init_pool(num_blocks, block_size, num_heads, head_dim, fmt, 1, None, None, None))
        dev = torch.device("cuda", torch.cuda.current_device())
        if fmt == KV_FP16:
            shape = (num_blocks, block_size, num_heads, head_dim)
            k = torch.zeros(shape, dtype=torch.float16, device=dev)
            v = torch.zeros(shape, dtype=torch.float16, device=dev)
            _check(_c_init_pool(num_blocks, block_size, num_heads, head_dim, fmt, k.data_ptr(), v.data_ptr(),
                                None, None))
            _pool.update(k=k, v=v, pages=None)
        else:
            lay = int4_layout(head_dim)
            pages = torch.empty((num_blocks, num_heads, lay["block"]), dtype=torch.uint8, device=dev)
            pages.copy_(_empty_int4_block(head_dim, dev).expand_as(pages))
            _check(_c_init_pool(num_blocks, block_size, num_heads, head_dim, fmt, pages.data_ptr(), None, None, None))
            _pool.update(pages=pages, k=pages[:, :, lay["kcodes"]:lay["vcodes"]],
                         v=pages[:, :, lay["vcodes"]:lay["kscales"]],
                         ks=pages[:, :, lay["kscales"]:lay["vscales"]].view(torch.float16),
                         vs=pages[:, :, lay["vscales"]:].view(torch.float16))
        _pool.update(fmt=fmt, nb=num_blocks, bs=block_size, h=num_heads, d=head_dim)


def reset_pool() -> None:
    """Drop the pool (storage and free list); the next ``init_pool`` starts fresh."""
    with _pool_lock:
        _pool.clear()
        _c_reset_pool()


def int4_layout(head_dim: int) -> dict:
    """Byte offsets of the regions of one (page, head) block of the INT4 page
    pool (include/memopt_hip.h MEMOPT_KV_INT4)."""
    D, G = head_dim, head_dim // 64
    return {"kcodes": 0, "vcodes": 8 * D, "kscales": 16 * D, "vscales": 16 * D + 32 * G, "block": 16 * D + 64 * G}


def _empty_int4_block(head_dim: int, dev) -> torch.Tensor:
    """One (page, head) block of an empty row set: codes 8 (0x88), scales 1.0."""
    lay = int4_layout(head_dim)
    blk = torch.full((lay["block"],), 0x88, dtype=torch.uint8)
    blk[lay["kscales"]:] = torch.ones((lay["block"] - lay["kscales"]) // 2, dtype=torch.float16).view(torch.uint8)
    return blk.to(dev)


def _pool_or_raise(fn: str) -> dict:
    _require(bool(_pool), f"{fn}: pool not initialized")
    return _pool


def allocate_block() -> int:
    """Pop one free block (FIFO); -1 when exhausted (src/csrc/kv_cache.cu:163-172)."""
    out = _i64()
    _check(_c_alloc(ctypes.byref(out)))
    return int(out.value)


def free_block(block_idx: int) -> None:
    """Return a block to the free list (src/csrc/kv_cache.cu:179-185)."""
    _check(_c_free(int(block_idx)))


def allocate_blocks(count: int) -> Optional[List[int]]:
    """``count`` blocks popped as ``allocate_block`` would; ``None``, and none taken, when fewer are free."""
    out = (_i64 * max(1, count))()
    _check(_c_alloc_n(count, out))
    return None if count and out[0] < 0 else out[:count]


def free_blocks(blocks: Sequence[int]) -> None:
    """Return blocks to the free list in order; every index is checked before the first is returned."""
    _check(_c_free_n(len(blocks), (_i64 * max(1, len(blocks)))(*blocks)))


def free_blocks_count() -> int:
    out = _i64()
    _check(_c_free_count(ctypes.byref(out)))
    return int(out.value)


def get_pool_tensors() -> Tuple[torch.Tensor, torch.Tensor]:
    """(key_pool, value_pool) aliases of the live storage (src/csrc/kv_cache.cu:190-193).

    fp16 pools: [nb, bs, H, D] fp16. INT4 pools: views of the K and V code
    regions of the page buffer, uint8 [nb, H, 8*D] (codes in the page
    layout); passing them to ``dynamic_sparse_attention`` attends over the pool.
    """
    p = _pool_or_raise("get_pool_tensors")
    return p["k"], p["v"]


def get_int4_pages() -> torch.Tensor:
    """The INT4 page buffer, uint8 [nb, H, 16*D + 64*(D/64)]."""
    p = _pool_or_raise("get_int4_pages")
    _require(p["fmt"] == KV_INT4, "get_int4_pages: pool is not an INT4 pool")
    return p["pages"]


def pool_kv_format() -> str:
    """Storage format of the live pool: ``"fp16"`` or ``"int4"``."""
    return "int4" if _pool_or_raise("pool_kv_format")["fmt"] == KV_INT4 else "fp16"


def get_key_pool() -> torch.Tensor:
    return _pool_or_raise("get_key_pool")["k"]


def get_value_pool() -> torch.Tensor:
    return _pool_or_raise("get_value_pool")["v"]


def get_pool_scales() -> Tuple[torch.Tensor, torch.Tensor]:
    """fp16 group-scale regions of an INT4 pool, views [nb, H, 16*D/64] (page layout order)."""
    p = _pool_or_raise("get_pool_scales")
    _require(p["fmt"] == KV_INT4, "get_pool_scales: pool is not an INT4 pool")
    return p["ks"], p["vs"]


def dequantize_int4_pages(pages: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Dequantize an INT4 page buffer ``[nb, H, block]`` (default: the live pool)
    into fresh fp16 ``(K, V)`` pools ``[nb, 16, H, D]``.

    Each value is ``fp16(float(code - 8) * page_scale)``, the arithmetic of
    the reference dequantize kernel (src/csrc/quantization.cu:232-270) on this
    build's page layout; the attention kernels read the same values.
    """
    p = _pool_or_raise("dequantize_int4_pages")
    if pages is None:
        _require(p["fmt"] == KV_INT4, "dequantize_int4_pages: pool is not an INT4 pool")
        pages, D = p["pages"], p["d"]
    else:
        _require(pages.dim() == 3 and pages.dtype == torch.uint8, "dequantize_int4_pages: pages must be u8 [nb, H, B]")
        D = next((d for d in (64, 128) if int4_layout(d)["block"] == pages.shape[2]), None)
        _require(D is not None, "dequantize_int4_pages: block size matches no supported head_dim (64, 128)")
        _cuda(pages, "pages", "dequantize_int4_pages")
    pages = pages.contiguous()
    nb, H = pages.shape[0], pages.shape[1]
    k = torch.empty((nb, 16, H, D), dtype=torch.float16, device=pages.device)
    v = torch.empty_like(k)
    with _on(pages.device):
        _check(_c_pages_to_fp16(pages.data_ptr(), nb, H, D, k.data_ptr(), v.data_ptr(), _stream(pages)))
    return k, v


def convert_pool(kv_format: str) -> None:
    """Switch the live pool between ``"fp16"`` and ``"int4"`` storage in place.

    The free list and every block table stay valid: fp16 pages are quantized
    into INT4 pages (what ``write_cache`` into an INT4 pool would store for
    the same rows), INT4 pages are dequantized into fp16 pools. This is the
    switch MemoryScheduler.use_int4 asks for (src/memopt/scheduler.py:15-18);
    the reference has no code that performs it.
    """
    fmt = _FORMATS.get(kv_format)
    _require(fmt is not None, f"convert_pool: kv_format must be one of {sorted(_FORMATS)}")
    with _pool_lock:
        p = _pool_or_raise("convert_pool")
        if p["fmt"] == fmt:
            return
        nb, bs, H, D = p["nb"], p["bs"], p["h"], p["d"]
        dev = p["k"].device
        if fmt == KV_INT4:
            _require(bs == 16 and D % 64 == 0, "convert_pool: INT4 pools need 16-token pages and head_dim % 64 == 0")
            lay = int4_layout(D)
            pages = torch.empty((nb, H, lay["block"]), dtype=torch.uint8, device=dev)
            old_k, old_v = p["k"], p["v"]
            _check(_c_set_storage(KV_INT4, pages.data_ptr(), None))
            slots = torch.arange(nb * bs, dtype=torch.int32, device=dev)
            with _on(dev):
                _check(_c_write(old_k.data_ptr(), old_v.data_ptr(), nb * bs, H, D, slots.data_ptr(),
                                _stream(old_k)))
            _pool.update(fmt=fmt, pages=pages, k=pages[:, :, lay["kcodes"]:lay["vcodes"]],
                         v=pages[:, :, lay["vcodes"]:lay["kscales"]],
                         ks=pages[:, :, lay["kscales"]:lay["vscales"]].view(torch.float16),
                         vs=pages[:, :, lay["vscales"]:].view(torch.float16))
        else:
            k, v = dequantize_int4_pages()
            _check(_c_set_storage(KV_FP16, k.data_ptr(), v.data_ptr()))
            _pool.update(fmt=fmt, pages=None, k=k, v=v, ks=None, vs=None)


# ---------------------------------------------------------------------------
# write_cache — src/csrc/kv_cache.cu:282-348
# ---------------------------------------------------------------------------

def write_cache(keys: torch.Tensor, values: torch.Tensor, block_tables: torch.Tensor,
                slot_mapping: torch.Tensor, *, validate_slots: bool = True) -> None:
    """Scatter [T, H, D] fp16 rows into pool slots (INT4 pools: quantize on the fly).

    ``block_tables`` is accepted and unused, as in the reference (:279-280).
    Slots outside the pool raise ``RuntimeError("... out of bounds")``; that
    check costs one device-to-host sync, so hot loops whose slots are known
    good may pass ``validate_slots=False`` (the kernel still skips, never
    writes, out-of-range slots).
    """
    p = _pool_or_raise("write_cache")
    _require(keys.dim() == 3, "write_cache: keys must be 3-D [num_tokens, num_heads, head_dim]")
    _require(values.dim() == 3, "write_cache: values must be 3-D [num_tokens, num_heads, head_dim]")
    _require(slot_mapping.dim() == 1, "write_cache: slot_mapping must be 1-D [num_tokens]")
    T, H, D = keys.shape
    _require(tuple(values.shape) == (T, H, D), "write_cache: keys/values shape mismatch")
    _require(slot_mapping.shape[0] == T, "write_cache: slot_mapping length != num_tokens")
    _require(H == p["h"], "write_cache: num_heads != pool.num_heads")
    _require(D == p["d"], "write_cache: head_dim != pool.head_dim")
    _require(keys.dtype == torch.float16 and values.dtype == torch.float16, "write_cache: keys/values must be fp16")
    _cuda(keys, "keys", "write_cache")
    _cuda(values, "values", "write_cache")
    _cuda(slot_mapping, "slot_mapping", "write_cache")
    _require(slot_mapping.dtype == torch.int32, "write_cache: slot_mapping must be int32")
    if T == 0:
        return
    keys, values, slot_mapping = keys.contiguous(), values.contiguous(), slot_mapping.contiguous()
    if validate_slots:
        lo, hi = (int(x) for x in torch.aminmax(slot_mapping))
        _require(lo >= 0 and hi < p["nb"] * p["bs"], "write_cache: slot_mapping out of bounds")
    with _on(keys.device):
        _check(_c_write(keys.data_ptr(), values.data_ptr(), T, H, D, slot_mapping.data_ptr(), _stream(keys)))


# ---------------------------------------------------------------------------
# Eviction — src/csrc/kv_cache.cu:503-559, :1053-1156
# ---------------------------------------------------------------------------

def evict_cache(block_tables: torch.Tensor, attention_scores: torch.Tensor, retain_ratio: float,
                num_sink_tokens: int = 4) -> None:
    """Pool-centric eviction over scores [num_blocks, block_size, H] (f32)."""
    p = _pool_or_raise("evict_cache")
    _require(0.0 < retain_ratio <= 1.0, "evict_cache: retain_ratio must be in (0, 1]")
    _require(attention_scores.dim() == 3,
             "evict_cache: attention_scores must be 3-D [num_blocks, block_size, num_heads]")
    _require(attention_scores.dtype == torch.float32, "evict_cache: attention_scores must be float32")
    nb, bs, h = attention_scores.shape
    _require(nb <= p["nb"], "evict_cache: attention_scores num_blocks > pool.num_blocks")
    _require(bs == p["bs"], "evict_cache: attention_scores block_size != pool.block_size")
    _require(h == p["h"], "evict_cache: attention_scores num_heads != pool.num_heads")
    _cuda(attention_scores, "attention_scores", "evict_cache")
    scores = attention_scores.contiguous()
    with _on(scores.device):
        _check(_c_evict_cache(scores.data_ptr(), nb, float(retain_ratio), int(num_sink_tokens), _stream(scores)))


def evict_workspace_bytes(num_seqs: int, num_heads: int, seq_len: int, max_blocks_per_seq: int,
                          total_pool_blocks: int) -> int:
    """Device workspace bytes an ``evict_tokens`` call of this shape needs
    (``memopt_evict_workspace_size``)."""
    need = _i64(0)
    _check(_c_evict_ws(num_seqs, num_heads, seq_len, max_blocks_per_seq, total_pool_blocks, ctypes.byref(need)))
    return need.value


def evict_tokens(attention_scores: torch.Tensor, block_tables: torch.Tensor, is_block_free: torch.Tensor,
                 retain_ratio: float, num_sink_tokens: int = 4, workspace: Optional[torch.Tensor] = None) -> None:
    """Sequence-centric Ada-KV eviction; mutates the pool, ``block_tables`` and ``is_block_free``.

    ``block_tables`` and ``is_block_free`` must be contiguous int32 CUDA
    tensors (the reference silently drops mutations of non-contiguous ones).
    ``workspace``: a contiguous uint8 tensor on the scores' device of at
    least ``evict_workspace_bytes`` bytes, any content (default: one from
    torch's caching allocator per call).
    """
    p = _pool_or_raise("evict_tokens")
    _require(0.0 < retain_ratio <= 1.0, "evict_tokens: retain_ratio must be in (0, 1]")
    _require(attention_scores.dim() == 3,
             "evict_tokens: attention_scores must be 3-D [num_seqs, num_heads, seq_len]")
    _require(attention_scores.dtype == torch.float32, "evict_tokens: attention_scores must be float32")
    _require(block_tables.dim() == 2, "evict_tokens: block_tables must be 2-D [num_seqs, max_blocks_per_seq]")
    _require(block_tables.dtype == torch.int32, "evict_tokens: block_tables must be int32")
    _require(is_block_free.dim() == 1, "evict_tokens: is_block_free must be 1-D [total_pool_blocks]")
    _require(is_block_free.dtype == torch.int32, "evict_tokens: is_block_free must be int32")
    N, H, L = attention_scores.shape
    _require(H == p["h"], "evict_tokens: attention_scores num_heads != pool.num_heads")
    _require(block_tables.shape[0] == N, "evict_tokens: block_tables batch size != num_seqs")
    _require(is_block_free.shape[0] <= p["nb"], "evict_tokens: is_block_free size > pool.num_blocks")
    for t, n in ((attention_scores, "attention_scores"), (block_tables, "block_tables"),
                 (is_block_free, "is_block_free")):
        _cuda(t, n, "evict_tokens")
        _require(t.device == attention_scores.device, f"evict_tokens: {n} on a different device")
    _require(block_tables.is_contiguous() and is_block_free.is_contiguous(),
             "evict_tokens: block_tables and is_block_free must be contiguous (they are mutated in place)")
    if N == 0 or L == 0:
        return
    scores = attention_scores.contiguous()
    M, nb = block_tables.shape[1], is_block_free.shape[0]
    need = evict_workspace_bytes(N, H, L, M, nb)
    with _on(scores.device):
        if workspace is None:
            # scratch from torch's caching allocator on the current stream (page
            # marks and long-row selection state; nothing is kept between calls)
            ws = torch.empty(need, dtype=torch.uint8, device=scores.device)
        else:
            _require(workspace.dtype == torch.uint8 and workspace.is_contiguous() and
                     workspace.device == scores.device and workspace.numel() >= need,
                     f"evict_tokens: workspace must be a contiguous uint8 tensor of >= {need} bytes on the "
                     "scores' device")
            ws = workspace
        _check(_c_evict_tokens(scores.data_ptr(), N, H, L, block_tables.data_ptr(), M,
                               is_block_free.data_ptr(), nb, float(retain_ratio),
                               int(num_sink_tokens), ws.data_ptr(), ws.numel(), _stream(scores)))


def free_evicted_blocks(is_block_free: torch.Tensor) -> List[int]:
    """Return every block with ``is_block_free == num_heads`` to the free list and reset its counter.

    The caller-side step documented at src/csrc/kv_cache.cu:1033-1036.
    Returns the freed block indices.
    """
    p = _pool_or_raise("free_evicted_blocks")
    idx = torch.nonzero(is_block_free == p["h"]).flatten()
    freed = [int(i) for i in idx.tolist()]
    for b in freed:
        free_block(b)
    if freed:
        is_block_free[idx] = 0
    return freed


# ---------------------------------------------------------------------------
# Quantization — src/csrc/quantization.cu:294-428
# ---------------------------------------------------------------------------

def quantize_kv_cache_int4(cache: torch.Tensor, group_size: int) -> List[torch.Tensor]:
    """[packed uint8 (last dim / 2), scales float32 [numel / 64]]."""
    _cuda(cache, "cache", "quantize_kv_cache_int4")
    _require(cache.is_contiguous(), "quantize_kv_cache_int4: cache must be contiguous")
    _require(cache.dtype == torch.float16, "quantize_kv_cache_int4: cache must be float16")
    _require(group_size == 64, f"quantize_kv_cache_int4: group_size must equal 64 (got {group_size})")
    _require(cache.dim() >= 1, "quantize_kv_cache_int4: cache must have at least one dimension")
    n = cache.numel()
    _require(n % group_size == 0,
             f"quantize_kv_cache_int4: total_elements ({n}) must be divisible by group_size ({group_size})")
    last = cache.shape[-1]
    _require(last % 2 == 0, f"quantize_kv_cache_int4: last dimension ({last}) must be even for INT4 packing")
    packed = torch.empty(cache.shape[:-1] + (last // 2,), dtype=torch.uint8, device=cache.device)
    scales = torch.empty((n // group_size,), dtype=torch.float32, device=cache.device)
    if n:
        with _on(cache.device):
            _check(_c_quant(cache.data_ptr(), n, last, group_size, packed.data_ptr(), scales.data_ptr(),
                            _stream(cache)))
    return [packed, scales]


def dequantize_kv_cache_int4(q_cache: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    """fp16 tensor with the last dim doubled."""
    _cuda(q_cache, "q_cache", "dequantize_kv_cache_int4")
    _cuda(scales, "scales", "dequantize_kv_cache_int4")
    _require(q_cache.is_contiguous(), "dequantize_kv_cache_int4: q_cache must be contiguous")
    _require(scales.is_contiguous(), "dequantize_kv_cache_int4: scales must be contiguous")
    _require(q_cache.dtype == torch.uint8, "dequantize_kv_cache_int4: q_cache must be uint8")
    _require(scales.dtype == torch.float32, "dequantize_kv_cache_int4: scales must be float32")
    _require(group_size == 64, "dequantize_kv_cache_int4: group_size must equal 64")
    total = q_cache.numel() * 2
    _require(total % 64 == 0 and scales.numel() == total // 64,
             f"dequantize_kv_cache_int4: scales length ({scales.numel()}) != expected num_groups ({total // 64})")
    out = torch.empty(q_cache.shape[:-1] + (q_cache.shape[-1] * 2,), dtype=torch.float16, device=q_cache.device)
    if total:
        with _on(q_cache.device):
            _check(_c_dequant(q_cache.data_ptr(), q_cache.numel(), scales.data_ptr(), scales.numel(), group_size,
                              out.data_ptr(), _stream(q_cache)))
    return out


# ---------------------------------------------------------------------------
# Attention — src/csrc/attention.cu:371-521
# ---------------------------------------------------------------------------

def _int4_rows_layout(key_cache, key_scales, num_heads, head_dim):
    """Token-major INT4 codes [nb, bs, H, D/2] (quantize_kv_cache_int4 of an fp16
    pool) + f32/f16 scales [nb*bs*H*D/64]: (bs, nb, code strides, scale strides, scale dtype)."""
    G = head_dim // 64
    nb, bs, h, dh = key_cache.shape
    _require(h == num_heads and dh * 2 == head_dim, "dynamic_sparse_attention: INT4 cache shape mismatch")
    _require(key_cache.is_contiguous(), "key_cache must be contiguous")
    _require(key_scales.dtype in (torch.float16, torch.float32), "dynamic_sparse_attention: scales must be f16/f32")
    _require(key_scales.numel() == nb * bs * num_heads * G, "dynamic_sparse_attention: scales size mismatch")
    kv = (bs * h * dh, dh, h * dh)
    sc = (bs * h * G, G, h * G)
    return bs, nb, kv, sc, 1 if key_scales.dtype == torch.float16 else 0


def _int4_pages_base(key_cache, value_cache, num_heads, head_dim, fn="dynamic_sparse_attention"):
    """Base pointer and page count when the caches are the INT4 page buffer (or
    its K/V code views from get_pool_tensors), else None. fn: who refuses."""
    lay = int4_layout(head_dim)
    if _pool and _pool["fmt"] == KV_INT4 and _pool["d"] == head_dim and _pool["h"] == num_heads:
        base = _pool["pages"].data_ptr()
        if key_cache.data_ptr() in (base, base + lay["kcodes"]) and \
                value_cache.data_ptr() in (base, base + lay["vcodes"]):
            return base, _pool["nb"], _pool["pages"]
    if key_cache.dim() == 3 and key_cache.shape[1] == num_heads and key_cache.shape[2] == lay["block"]:
        if not key_cache.is_contiguous():
            raise RuntimeError(f"{fn}: INT4 page buffer must be contiguous")
        if value_cache.data_ptr() != key_cache.data_ptr():
            raise RuntimeError(f"{fn}: pass the INT4 page buffer as both key_cache and value_cache")
        return key_cache.data_ptr(), key_cache.shape[0], key_cache
    return None


def _attention_desc(query, key_cache, value_cache, block_tables, context_lens, max_seq_len, window_size,
                    num_sink_tokens, causal, key_scales, value_scales, kv_layout, out, alloc_workspace=True):
    """Validate like src/csrc/attention.cu:383-439 and fill an AttnDesc.

    Returns (desc, out, workspace, keepalive) or (None, out, None, ()) for empty shapes.
    """
    # (A message with values in it is formatted only when it is raised: on a
    # small decode the host side of the call is longer than its kernels.)
    fn = "dynamic_sparse_attention"
    for t, n in ((query, "query"), (key_cache, "key_cache"), (value_cache, "value_cache"),
                 (block_tables, "block_tables"), (context_lens, "context_lens")):
        if not (isinstance(t, torch.Tensor) and t.is_cuda):
            raise RuntimeError(f"{n} must be a CUDA tensor")
    for t, n in ((query, "query"), (block_tables, "block_tables"), (context_lens, "context_lens")):
        if not t.is_contiguous():
            raise RuntimeError(f"{n} must be contiguous")
    q_shape, bt_shape, cl_shape = query.shape, block_tables.shape, context_lens.shape
    _require(len(q_shape) == 4, "query must be 4-D [batch, q_len, num_heads, head_dim]")
    _require(len(bt_shape) == 2, "block_tables must be 2-D [batch, max_blocks_per_seq]")
    _require(len(cl_shape) == 1, "context_lens must be 1-D [batch]")
    _require(query.dtype == torch.float16, "query must be fp16")
    _require(block_tables.dtype == torch.int32, "block_tables must be int32")
    _require(context_lens.dtype == torch.int32, "context_lens must be int32")
    B, Lq, H, D = q_shape
    _require(bt_shape[0] == B, "block_tables batch dimension mismatch")
    _require(cl_shape[0] == B, "context_lens batch dimension mismatch")
    if out is None:
        out = torch.empty_like(query)
    elif not (out.shape == q_shape and out.dtype == torch.float16 and out.is_contiguous() and out.is_cuda):
        raise RuntimeError(f"{fn}: out must be a contiguous fp16 CUDA tensor shaped like query")
    keep = (query, key_cache, value_cache, block_tables, context_lens, key_scales, value_scales)
    fmt = KV_FP16
    sc = (0, 0, 0)
    sdt = 0
    kv = (0, 0, 0)
    base_k, base_v = key_cache.data_ptr(), value_cache.data_ptr()
    if key_cache.dtype == torch.uint8:
        _require(value_cache.dtype == torch.uint8, "value_cache must match key_cache (INT4 codes)")
        _require(D % 64 == 0, "dynamic_sparse_attention: INT4 caches need head_dim % 64 == 0")
        pages = _int4_pages_base(key_cache, value_cache, H, D) if kv_layout in (None, "pages") else None
        if pages is not None:
            fmt = KV_INT4
            base_k, nb, buf = pages
            base_v = base_k
            bs = 16
            keep = keep + (buf,)
        else:
            _require(kv_layout in (None, "token_major"), "dynamic_sparse_attention: not an INT4 page buffer")
            _require(key_cache.dim() == 4 and value_cache.shape == key_cache.shape and value_cache.is_contiguous(),
                     "key_cache must be 4-D [num_kv_blocks, block_size, num_heads, head_dim/2] (INT4 codes)")
            _require(key_scales is not None and value_scales is not None,
                     "dynamic_sparse_attention: INT4 caches need key/value scales")
            for t, n in ((key_scales, "key_scales"), (value_scales, "value_scales")):
                if not (t.is_cuda and t.is_contiguous()):
                    raise RuntimeError(f"{n} must be a contiguous CUDA tensor")
            _require(key_scales.dtype == value_scales.dtype and key_scales.shape == value_scales.shape,
                     "dynamic_sparse_attention: key/value scales mismatch")
            fmt = KV_INT4_ROWS
            bs, nb, kv, sc, sdt = _int4_rows_layout(key_cache, key_scales, H, D)
    else:
        for t, n in ((key_cache, "key_cache"), (value_cache, "value_cache")):
            if not t.is_contiguous():
                raise RuntimeError(f"{n} must be contiguous")
        k_shape, v_shape = key_cache.shape, value_cache.shape
        _require(len(k_shape) == 4, "key_cache must be 4-D [num_kv_blocks, block_size, num_heads, head_dim]")
        _require(len(v_shape) == 4, "value_cache must be 4-D [num_kv_blocks, block_size, num_heads, head_dim]")
        _require(key_cache.dtype == torch.float16, "key_cache must be fp16")
        _require(value_cache.dtype == torch.float16, "value_cache must be fp16")
        nb, bs = k_shape[0], k_shape[1]
        if k_shape[2] != H:
            raise RuntimeError(f"key_cache num_heads {k_shape[2]} != query num_heads {H}")
        if k_shape[3] != D:
            raise RuntimeError(f"key_cache head_dim {k_shape[3]} != query head_dim {D}")
        _require(v_shape[1] == bs, "value_cache block_size mismatch")
        _require(v_shape[2] == H, "value_cache num_heads mismatch")
        _require(v_shape[3] == D, "value_cache head_dim mismatch")
        kv = (bs * H * D, D, H * D)
    if B == 0 or Lq == 0 or H == 0 or D == 0:
        return None, out, None, ()
    rows = fmt == KV_INT4_ROWS
    d = AttnDesc(query.data_ptr(), out.data_ptr(), B, Lq, H, D, fmt, base_k, base_v,
                 key_scales.data_ptr() if rows else None, value_scales.data_ptr() if rows else None, sdt, bs, nb,
                 *kv, *sc, block_tables.data_ptr(), bt_shape[1], context_lens.data_ptr(), int(max_seq_len),
                 int(window_size), int(num_sink_tokens), int(bool(causal)))
    need = _i64()
    _check(_c_ws(ctypes.byref(d), ctypes.byref(need)))
    ws = None
    if need.value > 0 and alloc_workspace:
        # A decode workspace holds split-K arrival counters, which must start
        # from zero (later calls may reuse it without clearing); a
        # multi-query workspace may hold anything.
        alloc = torch.zeros if Lq == 1 else torch.empty
        ws = alloc(need.value, dtype=torch.uint8, device=query.device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), need.value
    return d, out, ws, keep


def dynamic_sparse_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                             block_tables: torch.Tensor, context_lens: torch.Tensor, max_seq_len: int,
                             window_size: int, *, num_sink_tokens: int = 0, causal: bool = False,
                             key_scales: Optional[torch.Tensor] = None, value_scales: Optional[torch.Tensor] = None,
                             kv_layout: Optional[str] = None) -> torch.Tensor:
    """Paged sparse attention; returns fp16 [batch, q_len, H, D].

    Reference semantics for fp16 caches with the default keywords:
    non-causal, keys [max(0, ctx-W), ctx), pages with block_tables < 0
    skipped, W <= 0 or W > max_seq_len -> max_seq_len, scale 1/sqrt(D),
    no visible key -> 0. uint8 caches are INT4: either the INT4 page pool
    (its code views from ``get_pool_tensors()``, or a page buffer
    [nb, H, 16*D + 64*D/64] passed as both caches; scales live in the
    pages), or token-major codes [nb, bs, H, D/2] from
    ``quantize_kv_cache_int4`` of an fp16 pool together with their
    ``key_scales`` / ``value_scales`` (``kv_layout="token_major"``).
    """
    _require(isinstance(query, torch.Tensor) and query.is_cuda, "query must be a CUDA tensor")
    with _on(query.device):
        d, out, ws, _keep = _attention_desc(query, key_cache, value_cache, block_tables, context_lens,
                                            max_seq_len, window_size, num_sink_tokens, causal, key_scales,
                                            value_scales, kv_layout, None)
        if d is not None:
            _check(_c_attn(ctypes.byref(d), _stream(query)))
    return out


class PreparedAttention:
    """A validated ``dynamic_sparse_attention`` call bound to fixed tensors.

    Construction does the argument checks and workspace allocation once;
    each call launches on the current stream with a single C-ABI call and
    returns ``out`` (overwritten in place). Intended for decode loops where
    only the tensor *contents* change between steps.

    ``no_alloc=True`` allocates no workspace and launches through
    ``memopt_paged_attention_noalloc``, whose split-K partials live in a
    static per-GPU scratch array; no call allocates device memory, which suits
    capture into a HIP graph. Calls sharing that array must not overlap on
    one GPU.
    """

    def __init__(self, query, key_cache, value_cache, block_tables, context_lens, max_seq_len, window_size, *,
                 num_sink_tokens=0, causal=False, key_scales=None, value_scales=None, kv_layout=None, out=None,
                 no_alloc=False):
        _require(isinstance(query, torch.Tensor) and query.is_cuda, "query must be a CUDA tensor")
        self.device = query.device
        with _on(self.device):
            self._d, self.out, self._ws, self._keep = _attention_desc(
                query, key_cache, value_cache, block_tables, context_lens, max_seq_len, window_size,
                num_sink_tokens, causal, key_scales, value_scales, kv_layout, out, alloc_workspace=not no_alloc)
        self._dp = ctypes.byref(self._d) if self._d is not None else None
        self._fn = _c_attn_noalloc if no_alloc else _c_attn

    @property
    def workspace_bytes(self) -> int:
        """Device workspace held for the call (split-K partials or staged K/V)."""
        return 0 if self._ws is None else self._ws.numel() * self._ws.element_size()

    def __call__(self, stream: Optional[int] = None) -> torch.Tensor:
        if self._dp is not None:
            s = stream if stream is not None else torch._C._cuda_getCurrentRawStream(self.device.index)
            _check(self._fn(self._dp, s))
        return self.out


# ---------------------------------------------------------------------------
# Packed batches: grouped heads, sequences of different lengths (no
# counterparts in the reference)
# ---------------------------------------------------------------------------

# (On the smallest calls the host side takes longer than the kernels, so the
# checks below read each property of a tensor once and format messages only
# when they raise.)
def _device_tensors(fn: str, device: torch.device, names: Tuple[str, ...], *tensors) -> None:
    """Raises for the first of ``tensors`` that is not a CUDA tensor on ``device`` (one of CUDA)."""
    for t in tensors:
        if not (isinstance(t, torch.Tensor) and t.device == device):
            name = next(n for n, x in zip(names, tensors) if x is t)
            if not (isinstance(t, torch.Tensor) and t.is_cuda):
                raise RuntimeError(f"{fn}: {name} must be a CUDA tensor")
            raise RuntimeError(f"{fn}: {name} on a different device")


def _int32(fn: str, t: torch.Tensor, name: str, shape: Tuple[int, ...]) -> None:
    if not (t.dtype is torch.int32 and t.shape == shape and t.is_contiguous()):
        raise RuntimeError(f"{fn}: {name} must be a contiguous int32 tensor of shape {list(shape)}")


def _no_grad(fn: str, requires_grad: bool) -> None:
    if requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{fn}: no gradients are computed; call it under torch.no_grad()")


_FAR = 2 ** 23  # token stride from which the prompt kernel's 31-bit tile ranges no longer hold keys and values


def _rows(t: torch.Tensor, far: int = 2 ** 63) -> Tuple[torch.Tensor, int, int, int]:
    """(tensor, address, token stride, head stride) of ``t`` itself where its
    last dimension is contiguous, its rows are 16-byte aligned (views of a
    fused projection are) and its tokens less than ``far`` elements apart,
    else of a contiguous copy."""
    ts, hs, ds = t.stride()
    p = t.data_ptr()
    if ds == 1 and not (ts % 8 or hs % 8 or p % 16) and t.shape[2] <= ts < far:
        return t, p, ts, hs
    t = t.contiguous()  # (itself, where it is that already but off the alignment)
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t, t.data_ptr(), t.shape[1] * t.shape[2], t.shape[2]


def _out_rows(fn: str, out: Optional[torch.Tensor], query: torch.Tensor,
              width: Optional[int] = None) -> Tuple[torch.Tensor, int, int, int]:
    """(out, address, token stride, head stride); a fresh tensor for ``None``. ``width``: its last dimension, where
    that is not query's."""
    if out is None:
        if width is None:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)  # (half the time of torch.empty)
        else:
            out = torch.empty((query.shape[0], query.shape[1], width), dtype=query.dtype, device=query.device)
        _, H, D = out.shape
        return out, out.data_ptr(), H * D, D
    _device_tensors(fn, query.device, ("out",), out)
    shape = query.shape if width is None else query.shape[:2] + (width,)
    if not (out.shape == shape and out.dtype == query.dtype):
        raise RuntimeError(f"{fn}: out must be shaped like query, with its dtype" if width is None else
                           f"{fn}: out must be {list(shape)}, with query's dtype")
    ts, hs, ds = out.stride()
    p = out.data_ptr()
    T, H, D = out.shape
    # (rows lie token by token or head by head: others would overwrite each other)
    if not (ds == 1 and not (ts % 8 or hs % 8 or p % 16) and ts >= D and (
            H == 1 or hs >= D and (ts >= (H - 1) * hs + D or hs >= (T - 1) * ts + D))):
        raise RuntimeError(f"{fn}: out must have contiguous 16-byte aligned rows that do not overlap")
    return out, p, ts, hs


# Descriptors as bytes, in native alignment (a quarter of the time that ctypes structures take):
# memopt_prompt_desc and memopt_advance_desc.
_PROMPT = struct.Struct("@4P6i8qP2i")
_ADVANCE = struct.Struct("@11P5i")
_c_prompt_bytes = _lib["memopt_prompt_attention"]
_c_prompt_bytes.argtypes = [ctypes.c_char_p, _vp]
_c_prompt_bytes.restype = _i32


def _count32(n: int) -> int:
    """``n`` as an int32, where any negative number means the same and any past 2^31 - 1 as that."""
    return n if n.__class__ is int and -1 <= n < 2 ** 31 else min(max(int(n), -1), 2 ** 31 - 1)


def prompt_attention(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, cu_seqlens: torch.Tensor,
                     window_size: int = -1, *, num_sink_tokens: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over whole prompts packed one behind the other; returns ``[T, Hq, D]``.

    ``query`` ``[T, Hq, D]``, ``keys`` / ``values`` ``[T, Hkv, D]``: fp16 or
    bf16, D 64 or 128, Hq a multiple of Hkv (query head h reads key head
    ``h // (Hq / Hkv)``); any strides whose rows are contiguous and 16-byte
    aligned, such as views of a fused projection, are read in place (keys and
    values less than 2^23 elements apart), others are copied.
    ``cu_seqlens``: int32 ``[B + 1]`` on the device, ascending; sequence b is
    rows ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1``. Row i of a sequence sees
    its rows ``j <= i`` with ``j < num_sink_tokens`` or ``j > i -
    window_size`` (``window_size <= 0``: all of them), scale 1/sqrt(D).
    Rows of no sequence are left as they are in ``out`` (a fresh ``out`` is
    not initialized there). ``out`` must not overlap the inputs.
    """
    fn = "prompt_attention"
    if not (isinstance(query, torch.Tensor) and query.is_cuda):
        raise RuntimeError(f"{fn}: query must be a CUDA tensor")
    device, dtype = query.device, query.dtype
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(device):
            return prompt_attention(query, keys, values, cu_seqlens, window_size, num_sink_tokens=num_sink_tokens,
                                    out=out)
    _device_tensors(fn, device, ("keys", "values", "cu_seqlens"), keys, values, cu_seqlens)
    _no_grad(fn, query.requires_grad or keys.requires_grad or values.requires_grad)
    shape, kshape, cshape = query.shape, keys.shape, cu_seqlens.shape
    if not (len(shape) == 3 and len(kshape) == 3 and values.dim() == 3):
        raise RuntimeError(f"{fn}: query, keys and values must be 3-D [tokens, heads, head_dim]")
    T, Hq, D = shape
    Hk = kshape[1]
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise RuntimeError(f"{fn}: query must be fp16 or bf16")
    if not (keys.dtype is dtype and values.dtype is dtype):
        raise RuntimeError(f"{fn}: keys and values must have query's dtype")
    if not (kshape == (T, Hk, D) and values.shape == kshape):
        raise RuntimeError(f"{fn}: keys and values must be [{T}, kv heads, {D}], got {list(kshape)} and "
                           f"{list(values.shape)}")
    if len(cshape) != 1 or cshape[0] < 1:
        raise RuntimeError(f"{fn}: cu_seqlens must be 1-D [batch + 1]")
    _int32(fn, cu_seqlens, "cu_seqlens", cshape)
    out, po, ots, ohs = _out_rows(fn, out, query)
    q, pq, qts, qhs = _rows(query)
    k, pk, kts, khs = _rows(keys, _FAR)
    v, pv, vts, vhs = _rows(values, _FAR)
    try:
        d = _PROMPT.pack(pq, pk, pv, po, 1 if dtype is torch.bfloat16 else 0, T, cshape[0] - 1, Hq, Hk, D, qts, qhs, kts,
                         khs, vts, vhs, ots, ohs, cu_seqlens.data_ptr(), _count32(window_size),
                         _count32(num_sink_tokens))
    except struct.error:
        raise RuntimeError(f"{fn}: sizes must fit 32 bits") from None
    _check(_c_prompt_bytes(d, torch._C._cuda_getCurrentRawStream(index)))
    return out


def packed_workspace_bytes(tokens: int, batch: int, num_heads: int, num_kv_heads: int, head_dim: int,
                           max_query_len: int, max_seq_len: int, max_blocks_per_seq: int, window_size: int = -1, *,
                           num_sink_tokens: int = 0, block_size: int = 16, kv_format: str = "int4") -> int:
    """Device workspace bytes a ``packed_attention`` call of these sizes
    allocates (``memopt_packed_workspace_size``); "int4" counts page buffers."""
    fmt = _FORMATS.get(kv_format)
    _require(fmt is not None, f"packed_workspace_bytes: kv_format must be one of {sorted(_FORMATS)}")
    d = PackedDesc(None, None, tokens, batch, num_heads, num_kv_heads, head_dim, 0, 0, 0, 0, fmt, None, None, block_size,
                   1, None, max_blocks_per_seq, None, None, _count32(max_query_len), _count32(max_seq_len),
                   _count32(window_size), _count32(num_sink_tokens))
    need, zeroed = _i64(), _i64()
    _check(_c_packed_ws(ctypes.byref(d), ctypes.byref(need), ctypes.byref(zeroed)))
    return need.value


def _packed_desc(query, key_cache, value_cache, block_tables, context_lens, cu_seqlens, max_query_len, max_seq_len,
                 window_size, num_sink_tokens, out):
    """Validated PackedDesc: (desc, out, workspace, keepalive)."""
    fn = "packed_attention"
    _device_tensors(fn, query.device, ("key_cache", "value_cache", "block_tables", "context_lens", "cu_seqlens"),
                    key_cache, value_cache, block_tables, context_lens, cu_seqlens)
    _no_grad(fn, query.requires_grad)
    _require(query.dim() == 3, "packed_attention: query must be 3-D [tokens, heads, head_dim]")
    _require(query.dtype == torch.float16, "packed_attention: query must be fp16")
    T, Hq, D = query.shape
    _require(cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1, "packed_attention: cu_seqlens must be 1-D [batch + 1]")
    B = cu_seqlens.shape[0] - 1
    _int32(fn, cu_seqlens, "cu_seqlens", (B + 1,))
    _int32(fn, context_lens, "context_lens", (B,))
    _require(block_tables.dim() == 2, "packed_attention: block_tables must be 2-D [batch, max_blocks_per_seq]")
    _int32(fn, block_tables, "block_tables", (B, block_tables.shape[1]))
    _require(max_query_len >= 0, "packed_attention: max_query_len must not be negative")
    keep = (query, key_cache, value_cache, block_tables, context_lens, cu_seqlens)
    if key_cache.dtype == torch.uint8:
        _require(D in (64, 128), "packed_attention: head_dim must be 64 or 128")
        _require(key_cache.dim() == 3 and value_cache.dim() == 3 and key_cache.shape[1] > 0,
                 "packed_attention: INT4 caches are the pool's code views or its page buffer [pages, heads, bytes]")
        Hk = key_cache.shape[1]
        pages = _int4_pages_base(key_cache, value_cache, Hk, D, fn)
        _require(pages is not None, "packed_attention: not an INT4 page buffer of this head_dim")
        base_k, nb, buf = pages
        _require(buf.device == query.device, "packed_attention: key_cache on a different device")
        fmt, bs, base_v, keep = KV_INT4, 16, None, keep + (buf,)
    else:
        _require(key_cache.dtype == torch.float16 and value_cache.dtype == torch.float16,
                 "packed_attention: caches must be fp16 or INT4 pages")
        _require(key_cache.dim() == 4 and key_cache.shape == value_cache.shape and key_cache.shape[3] == D,
                 "packed_attention: caches must be 4-D [num_kv_blocks, block_size, kv heads, head_dim]")
        _require(key_cache.is_contiguous() and value_cache.is_contiguous(),
                 "packed_attention: caches must be contiguous")
        nb, bs, Hk = key_cache.shape[:3]
        fmt, base_k, base_v = KV_FP16, key_cache.data_ptr(), value_cache.data_ptr()
    out, po, ots, ohs = _out_rows(fn, out, query)
    q, pq, qts, qhs = _rows(query)
    # (the C side holds 32-bit sizes)
    d = PackedDesc(pq, po, T, B, Hq, Hk, D, qts, qhs, ots, ohs, fmt, base_k, base_v, bs, nb, block_tables.data_ptr(),
                   block_tables.shape[1], context_lens.data_ptr(), cu_seqlens.data_ptr(),
                   _count32(max_query_len), _count32(max_seq_len), _count32(window_size), _count32(num_sink_tokens))
    need, zeroed = _i64(), _i64()
    _check(_c_packed_ws(ctypes.byref(d), ctypes.byref(need), ctypes.byref(zeroed)))
    ws = None
    if need.value > 0:
        ws = torch.empty(need.value, dtype=torch.uint8, device=query.device)
        ws[:zeroed.value].zero_()  # arrival counters; the partial sums may hold anything
        d.workspace, d.workspace_bytes = ws.data_ptr(), need.value
    return d, out, ws, keep + (q,)


def packed_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                     block_tables: torch.Tensor, context_lens: torch.Tensor, cu_seqlens: torch.Tensor,
                     max_query_len: int, max_seq_len: int, window_size: int = -1, *, num_sink_tokens: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of packed queries over the paged cache with grouped heads; returns fp16 ``[T, Hq, D]``.

    Sequence b's queries are rows ``cu_seqlens[b] .. cu_seqlens[b + 1] - 1``
    of ``query`` ``[T, Hq, D]`` (fp16; strides as in ``prompt_attention``):
    the last positions of its ``context_lens[b]`` tokens, whose K/V are in the
    cache already. Each sequence may bring any number of them (decode: one);
    ``max_query_len`` bounds it. Caches: INT4 pages (the pool's code views,
    or a page buffer passed as both) or fp16 pools, with Hkv heads that divide
    Hq. Masks, windows and sinks are those of ``dynamic_sparse_attention(...,
    causal=True)``; a row that sees no key gives 0. Rows of no sequence are
    left as they are in ``out``.
    """
    _require(isinstance(query, torch.Tensor) and query.is_cuda, "packed_attention: query must be a CUDA tensor")
    with _on(query.device):
        d, out, ws, _keep = _packed_desc(query, key_cache, value_cache, block_tables, context_lens, cu_seqlens,
                                         max_query_len, max_seq_len, window_size, num_sink_tokens, out)
        _check(_c_packed(ctypes.byref(d), _stream(query)))
    return out


class PreparedPackedAttention:
    """A validated ``packed_attention`` call bound to fixed tensors.

    Construction checks the arguments, allocates the workspace and waits until
    its counters are cleared, so that calls may come on any stream; each call
    launches on the current stream (or the raw handle ``stream``) and returns
    ``out`` (overwritten in place). For loops in which only the tensors'
    contents change. Calls of one plan share its workspace and must not
    overlap. A plan made while a stream is captured has its counters cleared
    by that graph: it is for calls in that graph.
    """

    def __init__(self, query, key_cache, value_cache, block_tables, context_lens, cu_seqlens, max_query_len,
                 max_seq_len, window_size=-1, *, num_sink_tokens=0, out=None):
        _require(isinstance(query, torch.Tensor) and query.is_cuda, "packed_attention: query must be a CUDA tensor")
        self.device = query.device
        _require(query.dim() == 3 and _rows(query)[0] is query,
                 "PreparedPackedAttention: query's rows must be contiguous and 16-byte aligned (it is read in place)")
        with _on(self.device):
            self._d, self.out, self._ws, self._keep = _packed_desc(
                query, key_cache, value_cache, block_tables, context_lens, cu_seqlens, max_query_len, max_seq_len,
                window_size, num_sink_tokens, out)
            if self._ws is not None and not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()
        self._dp = ctypes.byref(self._d)

    @property
    def workspace_bytes(self) -> int:
        return 0 if self._ws is None else self._ws.numel()

    def __call__(self, stream: Optional[int] = None) -> torch.Tensor:
        with _on(self.device):
            s = stream if stream is not None else torch._C._cuda_getCurrentRawStream(self.device.index)
            _check(_c_packed(self._dp, s))
        return self.out


class BatchStep:
    """What ``advance_batch`` writes (int32, contiguous, on one device):
    ``context_lens`` ``[B]``, ``free_span`` ``[2]``, ``cu_seqlens`` ``[B +
    1]``, ``slots`` and ``positions`` ``[rows]``, ``status`` ``[B]``. The
    tensors are checked here once, and kept: another set is another step
    (``replace``)."""

    FIELDS = ("context_lens", "free_span", "cu_seqlens", "slots", "positions", "status")
    __slots__ = FIELDS + ("device", "_args")

    def __init__(self, context_lens, free_span, cu_seqlens, slots, positions, status):
        fn = "advance_batch"
        tensors = (context_lens, free_span, cu_seqlens, slots, positions, status)
        keep = super().__setattr__
        keep("device", getattr(context_lens, "device", None))
        _require(getattr(context_lens, "is_cuda", False), "advance_batch: context_lens must be a CUDA tensor")
        _device_tensors(fn, self.device, self.FIELDS, *tensors)
        _require(context_lens.dim() == 1 and slots.dim() == 1, "advance_batch: context_lens and slots must be 1-D")
        B, rows = context_lens.shape[0], slots.shape[0]
        for n, t, k in zip(self.FIELDS, tensors, (B, 2, B + 1, rows, rows, B)):
            _int32(fn, t, n, (k,))
            keep(n, t)
        keep("_args", tuple(t.data_ptr() for t in tensors))

    def __setattr__(self, name, value):
        raise AttributeError(f"BatchStep: {name} cannot be assigned; replace({name}=...) gives another step")

    def replace(self, **tensors) -> "BatchStep":
        """The same buffers with some of them exchanged."""
        return BatchStep(**{**{n: getattr(self, n) for n in self.FIELDS}, **tensors})


def advance_batch_buffers(num_requests: int, num_rows: int, device) -> BatchStep:
    """Buffers for ``advance_batch(..., out=)``."""
    sizes = (num_requests, 2, num_requests + 1, num_rows, num_rows, num_requests)
    return BatchStep(*(torch.empty(n, dtype=torch.int32, device=device) for n in sizes))


def advance_batch(new_tokens: torch.Tensor, context_lens: torch.Tensor, block_tables: torch.Tensor,
                  free_pages: torch.Tensor, free_span: torch.Tensor, block_size: int, num_rows: Optional[int] = None, *,
                  out: Optional[BatchStep] = None) -> BatchStep:
    """The index tensors of a batch's next step, built on the GPU (nothing is read back).

    Request b holds ``context_lens[b]`` tokens in the pages of
    ``block_tables[b]`` (int32 ``[B, M]``, its new entries are written in
    place) and asks for ``new_tokens[b]`` more. ``free_pages`` int32 ``[C]``
    is a ring whose free pages start at ``free_span[0]``, ``free_span[1]`` of
    them; they are taken in request order. Requests are served in order while
    what the valid ones so far ask for fits the free pages and ``num_rows``
    (one that needs no page is not refused for pages); the others stay as
    they were. ``status`` is 0 for a served request, 1 for an invalid count,
    2 where the page of its last token was evicted, 3 and 4 where pages or
    rows did not last. ``slots`` (for ``write_cache``) and ``positions`` hold
    the rows request by request, -1 behind the last.

    ``out``: buffers to write into (``advance_batch_buffers``); its
    ``context_lens`` and ``free_span`` may be the inputs, which are then
    advanced in place. Calls on one batch must not overlap.
    """
    fn = "advance_batch"
    if not (isinstance(new_tokens, torch.Tensor) and new_tokens.is_cuda):
        raise RuntimeError(f"{fn}: new_tokens must be a CUDA tensor")
    device = new_tokens.device
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(device):
            return advance_batch(new_tokens, context_lens, block_tables, free_pages, free_span, block_size, num_rows,
                                 out=out)
    _device_tensors(fn, device, ("context_lens", "block_tables", "free_pages", "free_span"), context_lens, block_tables,
                    free_pages, free_span)
    nshape, tshape, fshape = new_tokens.shape, block_tables.shape, free_pages.shape
    if not (len(nshape) == 1 and len(tshape) == 2 and len(fshape) == 1):
        raise RuntimeError(f"{fn}: new_tokens and free_pages must be 1-D, block_tables 2-D")
    if not (0 < block_size < 2 ** 31 and fshape[0] < 2 ** 31):
        raise RuntimeError(f"{fn}: sizes must be positive and fit 32 bits")
    B, = nshape
    M, C = tshape[1], fshape[0]
    _int32(fn, new_tokens, "new_tokens", nshape)
    _int32(fn, context_lens, "context_lens", nshape)
    _int32(fn, block_tables, "block_tables", (B, M))
    _int32(fn, free_pages, "free_pages", fshape)
    _int32(fn, free_span, "free_span", (2,))
    if out is None:
        _require(num_rows is not None and num_rows >= 0, "advance_batch: num_rows or out must be given")
        out = advance_batch_buffers(B, num_rows, device)
    rows, = out.slots.shape
    if num_rows is not None and num_rows != rows:
        raise RuntimeError(f"{fn}: num_rows differs from out's rows")
    if out.device != device or out.context_lens.shape != nshape:
        raise RuntimeError(f"{fn}: out holds buffers of another device or number of requests")
    d = _ADVANCE.pack(new_tokens.data_ptr(), context_lens.data_ptr(), block_tables.data_ptr(), free_pages.data_ptr(),
                      free_span.data_ptr(), *out._args, B, M, C, block_size, rows)
    _check(_c_advance(d, torch._C._cuda_getCurrentRawStream(index)))
    return out


# ---------------------------------------------------------------------------
# A cache that is kept small: weights per token, compaction (no counterparts in
# the reference)
# ---------------------------------------------------------------------------

_SCORES = struct.Struct("@3P5i2qiPiqPiPP5iPq")  # memopt_scores_desc


def _paged_call(fn: str, query, context_lens, cu_seqlens, block_tables) -> Tuple[int, int]:
    """(batch, max_blocks_per_seq) of the checked index tensors of packed queries over pages."""
    if not (cu_seqlens.dim() == 1 and cu_seqlens.shape[0] >= 1):
        raise RuntimeError(f"{fn}: cu_seqlens must be 1-D [batch + 1]")
    if block_tables.dim() != 2:
        raise RuntimeError(f"{fn}: block_tables must be 2-D [batch, max_blocks_per_seq]")
    B, M = cu_seqlens.shape[0] - 1, block_tables.shape[1]
    _int32(fn, cu_seqlens, "cu_seqlens", (B + 1,))
    _int32(fn, context_lens, "context_lens", (B,))
    _int32(fn, block_tables, "block_tables", (B, M))
    return B, M


def _near_rows(t: torch.Tensor, group: int) -> Tuple[torch.Tensor, int, int, int]:
    """``_rows`` of ``t``, copied too where 31 token strides and ``group`` head strides pass 2^29 elements."""
    r = _rows(t)
    if 31 * r[2] + group * r[3] >= 2 ** 29:
        r = _rows(t.clone(memory_format=torch.contiguous_format))
    return r


def attention_scores(query: torch.Tensor, key_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, cu_seqlens: torch.Tensor, max_query_len: int, max_seq_len: int,
                     window_size: int = -1, *, num_sink_tokens: int = 0, scores: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention weights that packed queries give the cached tokens, added up; returns f32 ``[B, Hkv, L]``.

    ``out[b, h, j] = scores[b, h, j]`` plus the softmax weights of token j in
    sequence b, summed over the sequence's query rows and the query heads of
    key head h: the scores that ``evict_tokens`` and ``compact_cache`` go by.
    ``query``, index tensors and masks are those of ``packed_attention``;
    ``key_cache``: INT4 pages (the pool's key view or a page buffer) or the
    fp16 key pool. A row that sees no key adds nothing. ``scores``: f32
    ``[B, Hkv, L]``, contiguous (``None``: zeros, L = ``max_seq_len``);
    ``out`` may be ``scores`` itself, else must not overlap it. Tokens from
    ``max_seq_len`` on are not looked at. The sums' order is fixed.
    """
    fn = "attention_scores"
    if not (isinstance(query, torch.Tensor) and query.is_cuda):
        raise RuntimeError(f"{fn}: query must be a CUDA tensor")
    device = query.device
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(device):
            return attention_scores(query, key_cache, block_tables, context_lens, cu_seqlens, max_query_len, max_seq_len,
                                    window_size, num_sink_tokens=num_sink_tokens, scores=scores, out=out)
    _device_tensors(fn, device, ("key_cache", "block_tables", "context_lens", "cu_seqlens"), key_cache, block_tables,
                    context_lens, cu_seqlens)
    _no_grad(fn, query.requires_grad)
    if query.dim() != 3 or query.dtype is not torch.float16:
        raise RuntimeError(f"{fn}: query must be fp16 [tokens, heads, head_dim]")
    T, Hq, D = query.shape
    B, M = _paged_call(fn, query, context_lens, cu_seqlens, block_tables)
    if max_query_len < 0 or max_seq_len < 0:
        raise RuntimeError(f"{fn}: max_query_len and max_seq_len must not be negative")
    if key_cache.dtype is torch.uint8:
        if D not in (64, 128):
            raise RuntimeError(f"{fn}: head_dim must be 64 or 128")
        if not (key_cache.dim() == 3 and key_cache.shape[1] > 0):
            raise RuntimeError(f"{fn}: INT4 caches are the pool's key view or its page buffer [pages, heads, bytes]")
        Hk = key_cache.shape[1]
        pages = _int4_pages_base(key_cache, key_cache, Hk, D, fn)
        if pages is None:
            raise RuntimeError(f"{fn}: not an INT4 page buffer of this head_dim")
        pk, nb, _ = pages
        fmt, bs = KV_INT4, 16
    else:
        if key_cache.dtype is not torch.float16:
            raise RuntimeError(f"{fn}: key_cache must be fp16 or INT4 pages")
        if not (key_cache.dim() == 4 and key_cache.shape[3] == D and key_cache.is_contiguous()):
            raise RuntimeError(f"{fn}: key_cache must be contiguous [num_kv_blocks, block_size, kv heads, {D}]")
        nb, bs, Hk = key_cache.shape[:3]
        fmt, pk = KV_FP16, key_cache.data_ptr()
    if scores is not None:
        _device_tensors(fn, device, ("scores",), scores)
        if not (scores.dim() == 3 and scores.shape[:2] == (B, Hk) and scores.dtype is torch.float32 and
                scores.is_contiguous()):
            raise RuntimeError(f"{fn}: scores must be contiguous f32 [{B}, {Hk}, positions]")
        _no_grad(fn, scores.requires_grad)
        L = scores.shape[2]
    else:
        L = max_seq_len if out is None else out.shape[-1]
    if out is None:
        out = torch.empty((B, Hk, L), dtype=torch.float32, device=device)
    else:
        _device_tensors(fn, device, ("out",), out)
        if not (out.shape == (B, Hk, L) and out.dtype is torch.float32 and out.is_contiguous()):
            raise RuntimeError(f"{fn}: out must be contiguous f32 {[B, Hk, L]}")
        _no_grad(fn, out.requires_grad)
    q, pq, qts, qhs = _near_rows(query, Hq // max(1, Hk))
    head = (pq, 0 if scores is None else scores.data_ptr(), out.data_ptr(), T, B, Hq, Hk, D, qts, qhs, fmt, pk, bs, nb,
            block_tables.data_ptr(), M, context_lens.data_ptr(), cu_seqlens.data_ptr(), _count32(max_query_len),
            _count32(max_seq_len), _count32(window_size), _count32(num_sink_tokens), L)
    _launch(fn, _SCORES, head, _c_scores_ws, _c_scores, device)
    return out


def _launch(fn: str, packed: struct.Struct, head: tuple, size, call, device: torch.device) -> None:
    """One call of a C entry whose descriptor ends in a workspace: ``head`` (numbers) and then a fresh one of ``size``'s
    bytes (any content) from torch's caching allocator, on the current stream of ``device``, which is current."""
    try:
        d = packed.pack(*head, 0, 0)
    except struct.error:
        raise RuntimeError(f"{fn}: sizes must fit 32 bits") from None
    need = _i64()
    rc = size(d, need)
    if rc:
        _check(rc)
    n = need.value
    if n:
        ws = torch.empty(n, dtype=torch.uint8, device=device)
        d = d[:-16] + _WORKSPACE.pack(ws.data_ptr(), n)
    rc = call(d, torch._C._cuda_getCurrentRawStream(device.index))
    if rc:
        _check(rc)


_WORKSPACE = struct.Struct("@Pq")


class CompactStep:
    """What ``compact_cache`` writes (contiguous, on one device; int32 but for
    ``scores``, f32): ``block_tables`` ``[N, M]``, ``context_lens`` ``[N]``,
    ``free_span`` ``[2]``, ``scores`` ``[N, Hkv, L]``, ``kept`` ``[N, Hkv,
    max_keep]``, ``status`` ``[N]``. The tensors are checked here once, and kept."""

    FIELDS = ("block_tables", "context_lens", "free_span", "scores", "kept", "status")
    __slots__ = FIELDS + ("device", "_args", "_sizes")

    def __init__(self, block_tables, context_lens, free_span, scores, kept, status):
        fn = "compact_cache"
        tensors = (block_tables, context_lens, free_span, scores, kept, status)
        keep = super().__setattr__
        keep("device", getattr(block_tables, "device", None))
        _require(getattr(block_tables, "is_cuda", False), "compact_cache: block_tables must be a CUDA tensor")
        _device_tensors(fn, self.device, self.FIELDS, *tensors)
        _require(block_tables.dim() == 2 and scores.dim() == 3 and kept.dim() == 3,
                 "compact_cache: block_tables must be 2-D, scores and kept 3-D")
        N, M = block_tables.shape
        Hk, L, K = scores.shape[1], scores.shape[2], kept.shape[2]
        for n, t, shape in zip(self.FIELDS, tensors, ((N, M), (N,), (2,), None, (N, Hk, K), (N,))):
            if shape is not None:
                _int32(fn, t, n, shape)
            elif not (t.dtype is torch.float32 and t.is_contiguous() and t.shape[0] == N):
                raise RuntimeError(f"{fn}: scores must be contiguous f32 [{N}, kv heads, positions]")
            keep(n, t)
        keep("_sizes", (N, Hk, M, L, K))
        keep("_args", tuple(t.data_ptr() for t in tensors))

    def __setattr__(self, name, value):
        raise AttributeError(f"CompactStep: {name} cannot be assigned")


def compact_cache_buffers(num_requests: int, num_kv_heads: int, max_blocks_per_seq: int, scores_len: int, max_keep: int,
                          device) -> CompactStep:
    """Buffers for ``compact_cache(..., out=)``."""
    def i32(*shape):
        return torch.empty(shape, dtype=torch.int32, device=device)

    N, Hk = num_requests, num_kv_heads
    return CompactStep(i32(N, max_blocks_per_seq), i32(N), i32(2),
                       torch.empty((N, Hk, scores_len), dtype=torch.float32, device=device), i32(N, Hk, max_keep), i32(N))


_COMPACT = struct.Struct("@3Pi2Pq9P10iPq")  # memopt_compact_desc


def compact_cache(scores: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, keep: torch.Tensor, free_pages: torch.Tensor, free_span: torch.Tensor, *,
                  num_sink_tokens: int = 4, num_recent_tokens: int = 0, max_keep: Optional[int] = None,
                  out: Optional[CompactStep] = None) -> CompactStep:
    """Tokens of least weight leave the cache; the others move to fresh pages and the old pages come back.

    Request b's ``context_lens[b]`` tokens lie in the pages of
    ``block_tables[b]`` (int32 ``[N, M]``). Every key head keeps ``n =
    min(keep[b], linked tokens)`` of them: the first ``num_sink_tokens``, the
    last ``num_recent_tokens``, and of the others those with the largest
    ``scores[b, h]`` (f32 ``[N, Hkv, L]``, L at least the longest context;
    ties: the first; NaN: last). They keep their order, as tokens ``0 .. n -
    1`` of pages from the front of the ring ``free_pages`` / ``free_span``
    (``advance_batch``); the old pages go to its end, in place. Unlike
    ``evict_tokens``, which zeroes rows, this takes them out of every later
    softmax. Queries after it stand at positions from n on: rotary positions
    are the caller's (``kept`` has the old ones).

    Caches: INT4 pages (the pool's code views, or a page buffer passed as
    both) or fp16 pools, changed in place (only in fresh pages). Results are
    new tensors, or ``out``'s (``compact_cache_buffers``), which must not
    overlap the inputs (but for ``free_span`` itself) nor each other; ``status``: 0 compacted, 1 invalid
    (length past table or scores, ``keep`` past ``max_keep``), 2 left (it may
    keep all it has; a negative ``keep``: always), 3 pages did not last (what
    a call gives back serves the next one), 4 a page is listed twice (by an
    invalid request, whose status stays 1, too).
    ``max_keep`` is needed without ``out``. Calls on one batch must not
    overlap.
    """
    fn = "compact_cache"
    if not (isinstance(scores, torch.Tensor) and scores.is_cuda):
        raise RuntimeError(f"{fn}: scores must be a CUDA tensor")
    device = scores.device
    if torch._C._cuda_getDevice() != device.index:
        with torch.cuda.device(device):
            return compact_cache(scores, key_cache, value_cache, block_tables, context_lens, keep, free_pages, free_span,
                                 num_sink_tokens=num_sink_tokens, num_recent_tokens=num_recent_tokens, max_keep=max_keep,
                                 out=out)
    _device_tensors(fn, device, ("key_cache", "value_cache", "block_tables", "context_lens", "keep", "free_pages",
                                 "free_span"), key_cache, value_cache, block_tables, context_lens, keep, free_pages,
                    free_span)
    if not (scores.dim() == 3 and scores.dtype is torch.float32 and scores.is_contiguous()):
        raise RuntimeError(f"{fn}: scores must be contiguous f32 [requests, kv heads, positions]")
    if block_tables.dim() != 2 or free_pages.dim() != 1:
        raise RuntimeError(f"{fn}: block_tables must be 2-D, free_pages 1-D")
    N, Hk, L = scores.shape
    M, C = block_tables.shape[1], free_pages.shape[0]
    _int32(fn, block_tables, "block_tables", (N, M))
    _int32(fn, context_lens, "context_lens", (N,))
    _int32(fn, keep, "keep", (N,))
    _int32(fn, free_pages, "free_pages", (C,))
    _int32(fn, free_span, "free_span", (2,))
    if key_cache.dtype is torch.uint8:
        if not (key_cache.dim() == 3 and value_cache.dim() == 3 and key_cache.shape[1] == Hk):
            raise RuntimeError(f"{fn}: INT4 caches are the pool's code views or its page buffer [pages, {Hk}, bytes]")
        pages = None
        for D in (64, 128):
            pages = pages or _int4_pages_base(key_cache, value_cache, Hk, D, fn)
            if pages is not None:
                break
        if pages is None:
            raise RuntimeError(f"{fn}: not an INT4 page buffer of head_dim 64 or 128")
        pk, nb, _ = pages
        fmt, bs, pv = KV_INT4, 16, 0
    else:
        if not (key_cache.dtype is torch.float16 and value_cache.dtype is torch.float16):
            raise RuntimeError(f"{fn}: caches must be fp16 or INT4 pages")
        if not (key_cache.dim() == 4 and key_cache.shape == value_cache.shape and key_cache.shape[2] == Hk and
                key_cache.is_contiguous() and value_cache.is_contiguous()):
            raise RuntimeError(f"{fn}: caches must be contiguous [num_kv_blocks, block_size, {Hk}, head_dim]")
        nb, bs, _, D = key_cache.shape
        fmt, pk, pv = KV_FP16, key_cache.data_ptr(), value_cache.data_ptr()
    if out is None:
        if max_keep is None or max_keep < 0:
            raise RuntimeError(f"{fn}: max_keep or out must be given")
        out = compact_cache_buffers(N, Hk, M, L, max_keep, device)
    K = out.kept.shape[2]
    if max_keep is not None and max_keep != K:
        raise RuntimeError(f"{fn}: max_keep differs from out's")
    if out.device != device or out._sizes[:4] != (N, Hk, M, L):
        raise RuntimeError(f"{fn}: out holds buffers of another device or of other sizes")
    bt_o, cl_o, span_o, sc_o, kept, status = out._args
    head = (scores.data_ptr(), sc_o, kept, fmt, pk, pv, nb, block_tables.data_ptr(), context_lens.data_ptr(),
            keep.data_ptr(), bt_o, cl_o, status, free_pages.data_ptr(), free_span.data_ptr(), span_o, N, Hk, D, M, bs, C, L,
            K, _count32(num_sink_tokens), _count32(num_recent_tokens))
    _launch(fn, _COMPACT, head, _c_compact_ws, _c_compact, device)
    return out


# ---------------------------------------------------------------------------
# Latent attention: one cached vector per token for all heads (no counterparts
# in the reference)
# ---------------------------------------------------------------------------

_LATENT = struct.Struct("@3P6i4qiqPiPP4ifPq")  # memopt_latent_desc


def _latent_cache(fn: str, cache: torch.Tensor, width: int) -> Tuple[int, int]:
    """(pages, tokens per page) of a latent cache of rows of ``width`` elements."""
    if not (cache.dim() == 3 and cache.shape[2] == width and cache.is_contiguous()):
        raise RuntimeError(f"{fn}: cache must be contiguous [num_kv_blocks, block_size, {width}]")
    return cache.shape[0], cache.shape[1]


def write_latent(latents: torch.Tensor, rope_keys: torch.Tensor, slot_mapping: torch.Tensor, cache: torch.Tensor) -> None:
    """Write tokens' latents ``[T, rank]`` and rotary keys ``[T, rope_dim]`` into a latent cache.

    ``cache`` ``[num_kv_blocks, block_size, rank + rope_dim]`` (contiguous,
    fp16 or bf16 like the rows); token t's row goes to slot
    ``slot_mapping[t]`` (int32; page * block_size + offset, as for
    ``write_cache``); slots outside the cache, -1 among them, are skipped.
    No two tokens may have one slot (pieces of both rows could stay).
    ``rank`` and ``rope_dim`` are multiples of 8. Rows may be views (of a
    fused projection): they are read in place where they are 16-byte aligned.
    """
    fn = "write_latent"
    if not (isinstance(latents, torch.Tensor) and latents.is_cuda):
        raise RuntimeError(f"{fn}: latents must be a CUDA tensor")
    device, dtype = latents.device, latents.dtype
    if torch._C._cuda_getDevice() != device.index:
        with torch.cuda.device(device):
            return write_latent(latents, rope_keys, slot_mapping, cache)
    _device_tensors(fn, device, ("rope_keys", "slot_mapping", "cache"), rope_keys, slot_mapping, cache)
    _no_grad(fn, latents.requires_grad or rope_keys.requires_grad)
    if not (latents.dim() == 2 and rope_keys.dim() == 2 and latents.shape[0] == rope_keys.shape[0]):
        raise RuntimeError(f"{fn}: latents and rope_keys must be 2-D [tokens, elements] of the same tokens")
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise RuntimeError(f"{fn}: latents must be fp16 or bf16")
    if not (rope_keys.dtype is dtype and cache.dtype is dtype):
        raise RuntimeError(f"{fn}: rope_keys and cache must have latents' dtype")
    T, R = latents.shape
    P = rope_keys.shape[1]
    nb, bs = _latent_cache(fn, cache, R + P)
    _int32(fn, slot_mapping, "slot_mapping", (T,))
    c, pc, cts, _ = _rows(latents[:, None])
    r, pr, rts, _ = _rows(rope_keys[:, None])
    if T > 2 ** 31 - 1:
        raise RuntimeError(f"{fn}: sizes must fit 32 bits")
    _check(_c_write_latent(pc, cts, pr, rts, T, R, P, slot_mapping.data_ptr(), cache.data_ptr(), nb * bs,
                           torch._C._cuda_getCurrentRawStream(device.index)))


def latent_attention(query: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, context_lens: torch.Tensor,
                     cu_seqlens: torch.Tensor, max_query_len: int, max_seq_len: int, scale: float, rank: int,
                     window_size: int = -1, *, num_sink_tokens: int = 0,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of packed queries over a paged latent cache (absorbed form); returns ``[T, Hq, rank]``.

    ``cache`` ``[num_kv_blocks, block_size, rank + rope_dim]``: a token's one
    row is the key of every head, its first ``rank`` elements the value.
    ``query`` ``[T, Hq, rank + rope_dim]`` holds each head's query times its
    key projection, then its rotary part; the caller multiplies the result
    with the heads' value projections. Scores are multiplied by ``scale``
    (one over the root of the width that a head's keys have when expanded).
    fp16 or bf16, one type for all; ``rank`` 128, 256 or 512, ``rope_dim`` 32
    or 64, pages of a multiple of 16 tokens. Index tensors, masks, strides and
    rows of no sequence are as in ``packed_attention``; tokens from
    ``max_seq_len`` on are not looked at. ``out`` must not overlap the inputs.
    """
    fn = "latent_attention"
    if not (isinstance(query, torch.Tensor) and query.is_cuda):
        raise RuntimeError(f"{fn}: query must be a CUDA tensor")
    device, dtype = query.device, query.dtype
    if torch._C._cuda_getDevice() != device.index:
        with torch.cuda.device(device):
            return latent_attention(query, cache, block_tables, context_lens, cu_seqlens, max_query_len, max_seq_len, scale,
                                    rank, window_size, num_sink_tokens=num_sink_tokens, out=out)
    _device_tensors(fn, device, ("cache", "block_tables", "context_lens", "cu_seqlens"), cache, block_tables, context_lens,
                    cu_seqlens)
    _no_grad(fn, query.requires_grad or cache.requires_grad)
    if query.dim() != 3:
        raise RuntimeError(f"{fn}: query must be 3-D [tokens, heads, rank + rope_dim]")
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise RuntimeError(f"{fn}: query must be fp16 or bf16")
    if cache.dtype is not dtype:
        raise RuntimeError(f"{fn}: cache must have query's dtype")
    T, Hq, W = query.shape
    if not 0 < rank < W:
        raise RuntimeError(f"{fn}: rank must be less than the query's width {W}")
    nb, bs = _latent_cache(fn, cache, W)
    B, M = _paged_call(fn, query, context_lens, cu_seqlens, block_tables)
    if max_query_len < 0 or max_seq_len < 0:
        raise RuntimeError(f"{fn}: max_query_len and max_seq_len must not be negative")
    out, po, ots, ohs = _out_rows(fn, out, query, rank)
    q, pq, qts, qhs = _rows(query)
    head = (pq, cache.data_ptr(), po, 1 if dtype is torch.bfloat16 else 0, T, B, Hq, rank, W - rank, qts, qhs, ots, ohs, bs,
            nb, block_tables.data_ptr(), M, context_lens.data_ptr(), cu_seqlens.data_ptr(), _count32(max_query_len),
            _count32(max_seq_len), _count32(window_size), _count32(num_sink_tokens), float(scale))
    _launch(fn, _LATENT, head, _c_latent_ws, _c_latent, device)
    return out


_LATENT_PROMPT = struct.Struct("@5P6i9qP2if")  # memopt_latent_prompt_desc (4 bytes of padding follow)


def latent_prompt_attention(query: torch.Tensor, keys: torch.Tensor, rope_keys: torch.Tensor, values: torch.Tensor,
                            cu_seqlens: torch.Tensor, window_size: int = -1, *, num_sink_tokens: int = 0,
                            scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over whole packed prompts of a latent model (expanded form); returns ``[T, H, D]``.

    Head h's key of a token is its row of ``keys`` ``[T, H, D]`` and, shared
    by all heads, that of ``rope_keys`` ``[T, P]``; ``query`` ``[T, H, D +
    P]`` holds the matching parts side by side, ``values`` are ``[T, H, D]``.
    fp16 or bf16, D 64 or 128, P 32 or 64; ``scale`` defaults to one over the
    root of D + P. Prompts, masks, strides and rows of no sequence are as in
    ``prompt_attention``: views (of the up-projection's output, say) are read
    in place. ``out`` must not overlap the inputs.
    """
    fn = "latent_prompt_attention"
    if not (isinstance(query, torch.Tensor) and query.is_cuda):
        raise RuntimeError(f"{fn}: query must be a CUDA tensor")
    device, dtype = query.device, query.dtype
    index = device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(device):
            return latent_prompt_attention(query, keys, rope_keys, values, cu_seqlens, window_size,
                                           num_sink_tokens=num_sink_tokens, scale=scale, out=out)
    _device_tensors(fn, device, ("keys", "rope_keys", "values", "cu_seqlens"), keys, rope_keys, values, cu_seqlens)
    _no_grad(fn, query.requires_grad or keys.requires_grad or rope_keys.requires_grad or values.requires_grad)
    if not (query.dim() == 3 and keys.dim() == 3 and rope_keys.dim() == 2 and values.dim() == 3):
        raise RuntimeError(f"{fn}: query, keys and values must be 3-D [tokens, heads, elements], rope_keys 2-D")
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise RuntimeError(f"{fn}: query must be fp16 or bf16")
    if not (keys.dtype is dtype and rope_keys.dtype is dtype and values.dtype is dtype):
        raise RuntimeError(f"{fn}: keys, rope_keys and values must have query's dtype")
    T, H, W = query.shape
    D, P = keys.shape[2], rope_keys.shape[1]
    if not (keys.shape == (T, H, D) and values.shape == keys.shape and rope_keys.shape[0] == T and D + P == W):
        raise RuntimeError(f"{fn}: keys and values must be [{T}, {H}, D] and rope_keys [{T}, P] with D + P = {W}, got "
                           f"{list(keys.shape)}, {list(values.shape)} and {list(rope_keys.shape)}")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise RuntimeError(f"{fn}: cu_seqlens must be 1-D [batch + 1]")
    _int32(fn, cu_seqlens, "cu_seqlens", cu_seqlens.shape)
    out, po, ots, ohs = _out_rows(fn, out, query, D)
    q, pq, qts, qhs = _rows(query)
    k, pk, kts, khs = _rows(keys, _FAR)
    rts, rds = rope_keys.stride()
    r, pr = rope_keys, rope_keys.data_ptr()
    if not (rds == 1 and not (rts % 8 or pr % 16) and P <= rts < _FAR):
        r, pr, rts, _ = _rows(rope_keys[:, None], _FAR)
    v, pv, vts, vhs = _rows(values, _FAR)
    try:
        d = _LATENT_PROMPT.pack(pq, pk, pr, pv, po, 1 if dtype is torch.bfloat16 else 0, T, cu_seqlens.shape[0] - 1, H, D, P,
                                qts, qhs, kts, khs, rts, vts, vhs, ots, ohs, cu_seqlens.data_ptr(), _count32(window_size),
                                _count32(num_sink_tokens), W ** -0.5 if scale is None else float(scale))
    except struct.error:
        raise RuntimeError(f"{fn}: sizes must fit 32 bits") from None
    _check(_c_latent_prompt(d + b"\0\0\0\0", torch._C._cuda_getCurrentRawStream(index)))
    return out
