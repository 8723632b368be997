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
import functools
import struct

import torch

from . import _native
from ._native import check

# The entries' argument records (the structures of _native): packing one is
# several times cheaper than converting its fields one by one.
_TABLES = struct.Struct("=QQqqQqQQqqQQQqQ")
_WRITE = struct.Struct("=QQqQqQQqqqqq")
_ATTENTION = struct.Struct("=QqQqQQqqqQQqqqQqqQqqqqfiQQ")
_NO_GUARD = contextlib.nullcontext()
_I32, _I64, _F16 = torch.int32, torch.int64, torch.float16


def _raw_stream(index: int) -> int:
    """Handle of the device's current stream (torch.cuda.current_stream makes an
    object first: 1.3 us instead of 0.1, of a call of 6 to 13)."""
    return torch._C._cuda_getCurrentRawStream(index)


def _on(device: torch.device):
    """A guard that makes `device` current for a call (nothing to do on it)."""
    if device.index == torch.cuda.current_device():
        return _NO_GUARD
    return torch.cuda.device(device)


def _ints(name: str, t: torch.Tensor, dtype: torch.dtype, numel: int, index: int) -> int:
    """Data pointer of a contiguous integer tensor of at least `numel` elements."""
    if t.dtype is not dtype or t.get_device() != index or t.numel() < numel or \
            not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of at least {numel} elements "
                         f"on cuda:{index}")
    return t.data_ptr()


def _pitches(t: torch.Tensor) -> tuple[int, ...]:
    """Strides of `t`, 0 for an axis of one element, where any is as good."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape, t.stride()))


def _table(t: torch.Tensor, rows: int, index: int) -> tuple[int, int, int]:
    """(pointer, row pitch, columns) of a block table."""
    if t.dim() != 2 or t.dtype is not _I32 or t.get_device() != index or t.shape[0] != rows or \
            (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"block_table must be a 2-D int32 tensor with one row per request ({rows}) and "
                         f"unit inner stride on cuda:{index}")
    cols = t.shape[1]
    return t.data_ptr(), (t.stride(0) if rows > 1 else cols), cols


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int, int, int, int]:
    """(device index, blocks, KV heads, rows per block, head dim, block stride)
    of a cache."""
    shape = k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape or k_cache.dtype is not _F16 or \
            v_cache.dtype is not _F16:
        raise ValueError("k_cache / v_cache must be f16 [blocks, kv_heads, block_rows, head_dim]")
    n, h, p, d = shape
    stride = k_cache.stride()
    if (v_cache.stride() != stride or stride[1:] != (p * d, d, 1)) and \
            (_pitches(v_cache) != _pitches(k_cache) or
             _pitches(k_cache)[1:] != tuple(s if m > 1 else 0 for m, s in
                                            ((h, p * d), (p, d), (d, 1)))):
        raise ValueError("the blocks of k_cache / v_cache must be contiguous, with one stride")
    index = k_cache.get_device()
    if index < 0 or v_cache.get_device() != index:
        raise ValueError("k_cache / v_cache must be on one CUDA device")
    return index, n, h, p, d, (stride[0] if n > 1 else h * p * d)


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
    unless `slots` is given, whose length it then is; of a longer `slots` its
    first max_tokens entries are written and returned."""
    lib = _native.load()
    index = cached_lens.get_device()
    if index < 0 or block_rows < 1:
        raise ValueError("cached_lens must be a CUDA tensor and block_rows >= 1")
    B = cached_lens.numel()
    if new_lens.numel() != B:
        raise ValueError("cached_lens and new_lens must have one entry per request")
    if slots is None:
        if max_tokens is None:
            raise ValueError("max_tokens or slots is needed")
        slots = cached_lens.new_empty(max_tokens, dtype=_I64)
    n = slots.numel() if max_tokens is None else int(max_tokens)
    if q_start is None:
        q_start = cached_lens.new_empty(B + 1)
    if kv_lens is None:
        kv_lens = cached_lens.new_empty(B)
    if cursor_out is None:
        cursor_out = cached_lens.new_empty(2)
    table_p, ld, cols = _table(block_table, B, index)
    with _on(cached_lens.device):
        check(lib.hxb_paged_tables(_TABLES.pack(
            _ints("cached_lens", cached_lens, _I32, B, index),
            _ints("new_lens", new_lens, _I32, B, index), B, block_rows,
            _ints("free_blocks", free_blocks, _I32, 0, index), free_blocks.numel(),
            _ints("cursor", cursor, _I32, 1, index), table_p, ld, cols,
            _ints("q_start", q_start, _I32, B + 1, index), _ints("kv_lens", kv_lens, _I32, B, index),
            _ints("slots", slots, _I64, n, index), n,
            _ints("cursor_out", cursor_out, _I32, 2, index)), _raw_stream(index)))
    # (what lies behind them is an earlier step's: not for this step's cache write)
    return q_start, kv_lens, slots if slots.numel() == n else slots.view(-1)[:n], cursor_out


def kv_cache_write_paged(k_src: torch.Tensor, v_src: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """k_cache[slots[t] // block_rows, h, slots[t] % block_rows] = k_src[t,
    h*D:(h+1)*D] (and V) for every source row t; a negative slot writes nothing,
    the others must differ. Sources are [tokens, kv_heads * D] f16 views of one
    row pitch (e.g. column blocks of a fused QKV output), caches
    [blocks, kv_heads, block_rows, D]."""
    lib = _native.load()
    index, blocks, heads, rows, D, stride = _cache(k_cache, v_cache)
    shape, src_stride = k_src.shape, k_src.stride()
    if len(shape) != 2 or shape[1] != heads * D or shape != v_src.shape or src_stride[1] != 1 or \
            (src_stride != v_src.stride() and _pitches(k_src) != _pitches(v_src)) or \
            k_src.dtype is not _F16 or v_src.dtype is not _F16:
        raise ValueError("k_src / v_src must be f16 [tokens, kv_heads * head_dim] views of one layout "
                         "with unit inner stride")
    if k_src.get_device() != index or v_src.get_device() != index:
        raise ValueError("sources and caches must share a device")
    n = shape[0]
    with _on(k_cache.device):
        check(lib.hxb_kv_cache_write_paged_f16(_WRITE.pack(
            k_src.data_ptr(), v_src.data_ptr(), src_stride[0] if n > 1 else heads * D,
            _ints("slots", slots, _I64, n, index), n, k_cache.data_ptr(), v_cache.data_ptr(), stride,
            blocks, heads, rows, D), _raw_stream(index)))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(index: int, total_q: int, q_heads: int, head_dim: int, prefix: bool) -> int:
    with torch.cuda.device(index):
        return attention_paged_workspace_bytes(total_q, q_heads, head_dim, int(prefix))


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
    have, a hint that chooses kernels: give 1 for a decode step (by default all the
    tokens, for which a batch of more than 16 query rows per KV head takes the
    kernel of prompt chunks). Own rows within a length must be finite where a token
    may not see them. Rows of `out` outside [q_start[0], q_start[batch]) are left as
    they are; `out` must not overlap an input. `workspace`: a device buffer of
    attention_paged_workspace_bytes (44 MB at D = 128, 22 MB at 64, and more with the
    tokens), allocated here if None."""
    lib = _native.load()
    index, blocks, Hkv, rows, D, stride = _cache(k_cache, v_cache)
    shape, q_stride = query.shape, query.stride()
    if len(shape) != 3 or shape[2] != D or q_stride[2] != 1 or \
            (q_stride[1] != D and shape[1] > 1) or \
            query.dtype is not _F16 or query.get_device() != index:
        raise ValueError("query must be f16 [tokens, q_heads, head_dim] with contiguous heads on the "
                         "caches' device")
    n, Hq, _ = shape
    if out is None:
        out = k_cache.new_empty(shape)
        o_stride = out.stride()
    else:
        o_stride = out.stride()
        if out.shape != shape or o_stride[2] != 1 or (o_stride[1] != D and shape[1] > 1) or \
                out.dtype is not _F16 or out.get_device() != index:
            raise ValueError("out must match query's shape, type and device, with contiguous heads")
    if n == 0:
        return out
    B = kv_lens.numel()
    table_p, ld, cols = _table(block_table, B, index)
    prefix_len = int(prefix_len)
    prefix_p = 0
    if prefix_len > 0:
        if prefix_table is None:
            raise ValueError("prefix_len needs prefix_table")
        prefix_p = _ints("prefix_table", prefix_table, _I32, -(-prefix_len // rows), index)
    row = Hq * D
    with _on(k_cache.device):
        if workspace is None:
            nbytes = _workspace_bytes(index, n, Hq, D, prefix_len > 0)
            workspace = kv_lens.new_empty(nbytes >> 2)
        else:
            if workspace.get_device() != index or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous buffer on the caches' device")
            nbytes = workspace.numel() * workspace.element_size()
        check(lib.hxb_attention_paged_f16(_ATTENTION.pack(
            query.data_ptr(), q_stride[0] if n > 1 else row, out.data_ptr(),
            o_stride[0] if n > 1 else row, _ints("q_start", q_start, _I32, B + 1, index),
            _ints("kv_lens", kv_lens, _I32, B, index), B, n,
            n if max_q_len is None else max_q_len, k_cache.data_ptr(), v_cache.data_ptr(), stride,
            blocks, rows, table_p, ld, cols, prefix_p, prefix_len, Hq, Hkv, D,
            D ** -0.5 if scale is None else scale, bool(causal), workspace.data_ptr(), nbytes),
            _raw_stream(index)))
    return out
