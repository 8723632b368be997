"""Refusals of the paged-cache entries: bad arguments are answered on the host,
before any device access (no GPU needed; the pointers are never followed)."""
from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest

from conftest import REPO

A = 0x100000  # an aligned address


def attention(pkg, **kw):
    a = pkg._native.AttentionPaged(
        q=A, ldq=1024, out=A, ldo=1024, q_start=A, kv_lens=A, batch=2, total_q=2, max_q_len=1, k_cache=A,
        v_cache=A, block_stride=2 * 16 * 128, num_blocks=8, block_rows=16, block_table=A, table_ld=4,
        table_cols=4, prefix_table=A, prefix_len=20, q_heads=8, kv_heads=2, head_dim=128, scale=0.1,
        causal=1, workspace=A, workspace_bytes=1 << 40)
    return pkg._native.load().hxb_attention_paged_f16(filled(a, kw), None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(head_dim=96), 2, b"head dim 96"),
    (dict(block_rows=48), 2, b"power of two"),
    (dict(block_rows=8), 2, b"power of two"),
    (dict(block_rows=2048, block_stride=2 * 2048 * 128), 2, b"power of two"),
    (dict(q_heads=9), 1, b"multiple of kv_heads"),
    (dict(q_heads=0), 1, b"multiple of kv_heads"),
    (dict(kv_heads=0), 1, b"cache extents"),
    (dict(q_heads=258), 2, b"query heads per KV head"),
    (dict(batch=0), 1, b"batch"),
    (dict(total_q=-1), 1, b"batch"),
    (dict(prefix_len=-1), 1, b"extents"),
    (dict(table_cols=5), 1, b"extents"),
    (dict(table_cols=0), 1, b"extents"),
    (dict(scale=0.0), 1, b"scale"),
    (dict(scale=float("inf")), 1, b"scale"),
    (dict(scale=float("nan")), 1, b"scale"),
    (dict(block_stride=2 * 16 * 128 - 8), 1, b"block_stride"),
    (dict(block_stride=2 * 16 * 128 + 4), 1, b"block_stride"),
    (dict(k_cache=A + 8), 1, b"16-byte"),
    (dict(v_cache=None), 1, b"null cache"),
    (dict(q=None), 1, b"null"),
    (dict(prefix_table=None), 1, b"null"),
    (dict(q=A + 2), 1, b"16-byte"),
    (dict(ldq=1028), 1, b"16-byte"),
    (dict(ldo=512), 1, b"16-byte"),
    (dict(total_q=1 << 29), 1, b"extents"),
    (dict(num_blocks=0), 1, b"cache extents"),
    (dict(kv_heads=40000, q_heads=40000, ldq=40000 * 128, ldo=40000 * 128,
          block_stride=40000 * 16 * 128), 1, b"extents"),
])
def test_attention_paged_refuses(pkg, kw, status, text):
    lib = pkg._native.load()
    assert attention(pkg, **kw) == status
    assert text in lib.hxb_last_error_message()


def test_attention_paged_without_tokens_is_nothing(pkg):
    assert attention(pkg, total_q=0, q=None, out=None, workspace=None, workspace_bytes=0) == 0


@pytest.mark.parametrize("packed,structure,entry", [
    ("_TABLES", "PagedTables", "hxb_paged_tables"),
    ("_WRITE", "KvCacheWritePaged", "hxb_kv_cache_write_paged_f16"),
    ("_ATTENTION", "AttentionPaged", "hxb_attention_paged_f16"),
])
def test_argument_records_have_the_layout_of_the_wrappers(pkg, packed, structure, entry):
    """The Python entries pack the argument records by themselves."""
    packed, structure = getattr(pkg.paged, packed), getattr(pkg._native, structure)
    assert packed.size == ctypes.sizeof(structure)
    values = [0.5 if f[0] == "scale" else i + 1 for i, f in enumerate(structure._fields_)]
    got = structure.from_buffer_copy(packed.pack(*values))
    assert [getattr(got, f[0]) for f in structure._fields_] == values
    assert getattr(pkg._native.load(), entry)(None, None) == 1


def filled(structure, kw):
    for name, value in kw.items():
        assert hasattr(structure, name)
        setattr(structure, name, value)
    return ctypes.byref(structure)


def tables(pkg, **kw):
    a = pkg._native.PagedTables(
        cached_lens=A, new_lens=A, batch=2, block_rows=16, free_blocks=A, num_free=4, cursor=A,
        block_table=A, table_ld=4, table_cols=4, q_start=A, kv_lens=A, slots=A, max_tokens=8,
        cursor_out=A)
    return pkg._native.load().hxb_paged_tables(filled(a, kw), None)


@pytest.mark.parametrize("kw,text", [
    (dict(batch=0), b"requests"), (dict(batch=16385), b"requests"), (dict(block_rows=0), b"extents"),
    (dict(table_cols=0), b"extents"), (dict(table_cols=5), b"extents"),
    (dict(max_tokens=-1), b"extents"), (dict(num_free=-1), b"extents"),
    (dict(block_rows=1 << 20, table_cols=1 << 12, table_ld=1 << 12), b"extents"),
    (dict(cached_lens=None), b"null"), (dict(free_blocks=None), b"null"), (dict(slots=None), b"null"),
    (dict(cursor_out=None), b"null"),
])
def test_paged_tables_refuses(pkg, kw, text):
    assert tables(pkg, **kw) == 1
    assert text in pkg._native.load().hxb_last_error_message()


def write(pkg, **kw):
    a = pkg._native.KvCacheWritePaged(
        k_src=A, v_src=A, ld_src=256, slots=A, tokens=3, k_cache=A, v_cache=A,
        block_stride=2 * 16 * 128, num_blocks=8, kv_heads=2, block_rows=16, head_dim=128)
    return pkg._native.load().hxb_kv_cache_write_paged_f16(filled(a, kw), None)


@pytest.mark.parametrize("kw,status,text", [
    (dict(block_rows=24), 2, b"power of two"), (dict(head_dim=12), 2, b"head_dim"),
    (dict(head_dim=2048), 2, b"head_dim"), (dict(tokens=-1), 1, b"token count"),
    (dict(k_src=None), 1, b"null"), (dict(slots=None), 1, b"null"),
    (dict(ld_src=255), 1, b"16-byte"), (dict(ld_src=248), 1, b"16-byte"),
    (dict(v_src=A + 8), 1, b"16-byte"), (dict(k_cache=A + 8), 1, b"16-byte"),
    (dict(block_stride=128), 1, b"block_stride"), (dict(kv_heads=0), 1, b"cache extents"),
])
def test_kv_cache_write_paged_refuses(pkg, kw, status, text):
    assert write(pkg, **kw) == status
    assert text in pkg._native.load().hxb_last_error_message()


def test_workspace_query_of_invalid_extents_is_zero(pkg):
    lib = pkg._native.load()
    assert lib.hxb_attention_paged_workspace_bytes(0, 8, 128, 0) == 0
    assert lib.hxb_attention_paged_workspace_bytes(4, 8, 96, 0) == 0
    assert lib.hxb_attention_paged_workspace_bytes(4, 0, 128, 0) == 0
    assert lib.hxb_attention_paged_workspace_bytes(4, 8, 128, -1) == 0


def test_python_entries_refuse_before_the_library(pkg):
    import torch
    f16 = dict(dtype=torch.float16)
    cache = torch.zeros(2, 1, 16, 64, **f16)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.kv_cache_write_paged(torch.zeros(1, 64, **f16), torch.zeros(1, 64, **f16), cache, cache,
                                 torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="contiguous"):
        pkg.kv_cache_write_paged(torch.zeros(1, 64, **f16), torch.zeros(1, 64, **f16),
                                 cache.transpose(2, 3), cache.transpose(2, 3),
                                 torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="f16"):
        pkg.kv_cache_write_paged(torch.zeros(1, 64), torch.zeros(1, 64), cache.float(), cache.float(),
                                 torch.zeros(1, dtype=torch.int64))
    ints = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        pkg.paged_tables(ints, ints, ints, ints, ints[None], block_rows=16, max_tokens=1)


def test_package_imports_on_a_torch_without_cuda_bindings():
    """The streams of a call are looked up by the call, not by the import."""
    program = ("import torch\n"
               "for name in [n for n in vars(torch._C) if n.startswith('_cuda_')]:\n"
               "    delattr(torch._C, name)\n"
               "import __graft_entry__\n"
               "assert callable(__graft_entry__.load_package().attention_paged)\n")
    r = subprocess.run([sys.executable, "-c", program], cwd=REPO, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
