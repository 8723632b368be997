"""Serving a batch of requests of different lengths from one paged KV cache:
the step's block tables and slot maps, the cache write through the slot map and
the attention over a shared prefix and the requests' own blocks.

A decode step of a serving loop is the three in turn; lengths and tables stay
on the GPU, so the step can be captured into a graph:

    q_start, kv_lens, slots, cursor = paged_tables(
        lens, new, free_blocks, cursor, block_table, block_rows=16, max_tokens=n)
    kv_cache_write_paged(k, v, k_cache, v_cache, slots)
    out = attention_paged(q, k_cache, v_cache, q_start, kv_lens, block_table,
                          prefix_table=prefix_table, prefix_len=2000, max_q_len=1)

The reference's KV-cache models keep one length and one contiguous cache per
batch (integration_tests/models/kv_cache.py:91-112).
"""
from __future__ import annotations

import contextlib

import torch

from . import _native
from ._native import check
from .dispatch import _require

_NO_GUARD = contextlib.nullcontext()


def _on(device: torch.device):
    """A guard that makes `device` current for a call (nothing to do on it)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _NO_GUARD
    return torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _ints(name: str, t: torch.Tensor, dtype: torch.dtype, numel: int, device: torch.device) -> int:
    """Data pointer of a contiguous integer tensor of at least `numel` elements."""
    if t.dtype != dtype or t.device != device or t.numel() < numel or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of at least {numel} elements "
                         f"on {device}")
    return t.data_ptr()


def _table(t: torch.Tensor, device: torch.device) -> tuple[int, int, int]:
    """(pointer, row pitch, columns) of a block table."""
    if t.dim() != 2 or t.dtype != torch.int32 or t.device != device or \
            (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"block_table must be a 2-D int32 tensor with unit inner stride on {device}")
    cols = t.shape[1]
    return t.data_ptr(), (t.stride(0) if t.shape[0] > 1 else cols), cols


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(blocks, KV heads, rows per block, head dim, block stride) of a cache."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or \
            k_cache.dtype != torch.float16 or v_cache.dtype != torch.float16:
        raise ValueError("k_cache / v_cache must be f16 [blocks, kv_heads, block_rows, head_dim]")
    n, h, p, d = k_cache.shape
    stride = k_cache.stride()
    if v_cache.stride() != stride or stride[1:] != (p * d, d, 1):
        raise ValueError("the blocks of k_cache / v_cache must be contiguous, with one stride")
    _require(k_cache.is_cuda and v_cache.device == k_cache.device,
             "k_cache / v_cache must be on one CUDA device")
    return n, h, p, d, (stride[0] if n > 1 else h * p * d)


def paged_tables(cached_lens: torch.Tensor, new_lens: torch.Tensor, free_blocks: torch.Tensor,
                 cursor: torch.Tensor, block_table: torch.Tensor, *, block_rows: int,
                 max_tokens: int | None = None, q_start: torch.Tensor | None = None,
                 kv_lens: torch.Tensor | None = None, slots: torch.Tensor | None = None,
                 cursor_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The tables of one step on the GPU (hxb_paged_tables): for int32
    `cached_lens` / `new_lens` [batch], writes the entries of the blocks begun in
    this step into `block_table` (taken from `free_blocks` at `cursor`[0]) and
    returns (q_start [batch + 1], kv_lens [batch], slots [max_tokens] int64 with
    -1 behind the last token, cursor_out [2]: the next cursor and how many
    blocks were missing). Outputs may be given: `kv_lens` may be `cached_lens`
    and `cursor_out` may be `cursor` (of 2 elements). `max_tokens` is needed
    unless `slots` is given, whose length it then is."""
    lib = _native.load()
    dev = cached_lens.device
    _require(cached_lens.is_cuda, "cached_lens must be a CUDA tensor")
    B = cached_lens.numel()
    i32 = torch.int32
    cached_p = _ints("cached_lens", cached_lens, i32, B, dev)
    new_p = _ints("new_lens", new_lens, i32, B, dev)
    free_p = _ints("free_blocks", free_blocks, i32, 0, dev)
    cursor_p = _ints("cursor", cursor, i32, 1, dev)
    table_p, ld, cols = _table(block_table, dev)
    _require(block_table.shape[0] == B, "block_table must have one row per request")
    _require(new_lens.numel() == B, "cached_lens and new_lens must have one entry per request")
    if slots is None:
        _require(max_tokens is not None, "max_tokens or slots is needed")
        slots = torch.empty(max_tokens, dtype=torch.int64, device=dev)
    n = slots.numel() if max_tokens is None else int(max_tokens)
    if q_start is None:
        q_start = torch.empty(B + 1, dtype=i32, device=dev)
    if kv_lens is None:
        kv_lens = torch.empty(B, dtype=i32, device=dev)
    if cursor_out is None:
        cursor_out = torch.empty(2, dtype=i32, device=dev)
    with _on(dev):
        check(lib.hxb_paged_tables(
            cached_p, new_p, B, block_rows, free_p, free_blocks.numel(), cursor_p, table_p, ld,
            cols, _ints("q_start", q_start, i32, B + 1, dev), _ints("kv_lens", kv_lens, i32, B, dev),
            _ints("slots", slots, torch.int64, n, dev), n,
            _ints("cursor_out", cursor_out, i32, 2, dev), _stream(dev)))
    return q_start, kv_lens, slots, cursor_out


def kv_cache_write_paged(k_src: torch.Tensor, v_src: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """k_cache[slots[t] // block_rows, h, slots[t] % block_rows] = k_src[t,
    h*D:(h+1)*D] (and V) for every source row t; a negative slot writes nothing.
    Sources are [tokens, kv_heads * D] f16 views of one row pitch (e.g. column
    blocks of a fused QKV output), caches [blocks, kv_heads, block_rows, D]."""
    lib = _native.load()
    blocks, heads, rows, D, stride = _cache(k_cache, v_cache)
    dev = k_cache.device
    if k_src.dim() != 2 or k_src.shape != v_src.shape or k_src.stride() != v_src.stride() or \
            k_src.dtype != torch.float16 or v_src.dtype != torch.float16 or \
            k_src.shape[1] != heads * D or k_src.stride(1) != 1:
        raise ValueError("k_src / v_src must be f16 [tokens, kv_heads * head_dim] views of one layout "
                         "with unit inner stride")
    _require(k_src.device == dev and v_src.device == dev, "sources and caches must share a device")
    n = k_src.shape[0]
    ld = k_src.stride(0) if n > 1 else heads * D
    with _on(dev):
        check(lib.hxb_kv_cache_write_paged_f16(
            k_src.data_ptr(), v_src.data_ptr(), ld, _ints("slots", slots, torch.int64, n, dev), n,
            k_cache.data_ptr(), v_cache.data_ptr(), stride, blocks, heads, rows, D, _stream(dev)))


def attention_paged_workspace_bytes(total_q: int, q_heads: int, head_dim: int,
                                    prefix_len: int = 0) -> int:
    """Bytes of workspace attention_paged needs on the current device."""
    return int(_native.load().hxb_attention_paged_workspace_bytes(total_q, q_heads, head_dim,
                                                                  prefix_len))


def attention_paged(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    q_start: torch.Tensor, kv_lens: torch.Tensor, block_table: torch.Tensor, *,
                    prefix_table: torch.Tensor | None = None, prefix_len: int = 0,
                    max_q_len: int | None = None, scale: float | None = None,
                    causal: bool = True, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Grouped-query attention of `query` [tokens, Hq, D] (rows
    [q_start[b], q_start[b+1]) belong to request b; rows may be further apart than
    Hq * D) over `prefix_len` rows of a prefix that all requests share (block ids
    in `prefix_table`) and the first kv_lens[b] rows of each request's own blocks
    (`block_table` [batch, columns]), caches [blocks, Hkv, block_rows, D]. The
    prefix is visible to every token; `causal` makes the tokens of a request its
    last cached rows. `max_q_len` is the most tokens a request is expected to
    have (a hint; by default all of them). Rows of `out` behind q_start[batch]
    are left as they are. `workspace`: a device buffer of
    attention_paged_workspace_bytes, allocated here if None."""
    lib = _native.load()
    blocks, Hkv, rows, D, stride = _cache(k_cache, v_cache)
    dev = k_cache.device
    if query.dim() != 3 or query.dtype != torch.float16 or query.device != dev or \
            query.shape[2] != D or query.stride(2) != 1 or query.stride(1) != D:
        raise ValueError("query must be f16 [tokens, q_heads, head_dim] with contiguous heads on the "
                         "caches' device")
    n, Hq, _ = query.shape
    if out is None:
        out = torch.empty((n, Hq, D), dtype=torch.float16, device=dev)
    elif out.shape != query.shape or out.dtype != torch.float16 or out.device != dev or \
            out.stride(2) != 1 or out.stride(1) != D:
        raise ValueError("out must match query's shape, type and device, with contiguous heads")
    B = kv_lens.numel()
    table_p, ld, cols = _table(block_table, dev)
    _require(block_table.shape[0] == B, "block_table must have one row per request")
    prefix_len = int(prefix_len)
    prefix_p = None
    if prefix_len:
        _require(prefix_table is not None, "prefix_len needs prefix_table")
        prefix_p = _ints("prefix_table", prefix_table, torch.int32, -(-prefix_len // rows), dev)
    row = Hq * D
    with _on(dev):
        if workspace is None:
            workspace = torch.empty(
                lib.hxb_attention_paged_workspace_bytes(n, Hq, D, prefix_len), dtype=torch.uint8,
                device=dev)
        else:
            _require(workspace.device == dev and workspace.is_contiguous(),
                     "workspace must be a contiguous buffer on the caches' device")
        check(lib.hxb_attention_paged_f16(
            query.data_ptr(), query.stride(0) if n > 1 else row, out.data_ptr(),
            out.stride(0) if n > 1 else row, _ints("q_start", q_start, torch.int32, B + 1, dev),
            _ints("kv_lens", kv_lens, torch.int32, B, dev), B, n,
            n if max_q_len is None else max_q_len, k_cache.data_ptr(), v_cache.data_ptr(), stride,
            blocks, rows, table_p, ld, cols, prefix_p, prefix_len, Hq, Hkv, D,
            D ** -0.5 if scale is None else float(scale), int(causal), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _stream(dev)))
    return out
