"""C ABI of the page operations and of shared-prefix decode: the ctypes structs
are laid out as the header's, and bad arguments are refused before any launch (no
kernel runs here)."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from flashattntile_amd import _hip

HEADER = Path(__file__).resolve().parents[1] / "include" / "fat_abi.h"
STRUCTS = {"fat_shared_args": _hip.SharedArgs, "fat_pool": _hip.Pool, "fat_copy_pages_args": _hip.CopyPagesArgs,
           "fat_fork_args": _hip.ForkArgs, "fat_free_args": _hip.FreeArgs, "fat_compact_args": _hip.CompactArgs,
           "fat_check_args": _hip.CheckArgs}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layout_matches_ctypes(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for struct, cls in STRUCTS.items():
        lines.append(f'  printf("{struct} size %zu\\n", sizeof({struct}));')
        for n, _ in cls._fields_:
            lines.append(f'  printf("{struct} {n} %zu\\n", offsetof({struct}, {n}));')
    for n in ("COPY", "FORK", "FREE", "SHARED"):
        lines.append(f'  printf("kind {n} %d\\n", FAT_CHECK_{n});')
    lines.append("  return 0; }")
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(src)], check=True)
    got = {}
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        struct, name, val = line.split()
        got[(struct, name)] = int(val)
    for struct, cls in STRUCTS.items():
        assert got[(struct, "size")] == ctypes.sizeof(cls), struct
        for n, _ in cls._fields_:
            assert got[(struct, n)] == getattr(cls, n).offset, (struct, n)
    assert [got[("kind", n)] for n in ("COPY", "FORK", "FREE", "SHARED")] == [
        _hip.CHECK_COPY, _hip.CHECK_FORK, _hip.CHECK_FREE, _hip.CHECK_SHARED]


def _refused(fn, args, error, code=None):
    rc = fn(None if args is None else ctypes.byref(args), None)
    message = _hip.lib().fat_last_error().decode()
    assert rc != 0 and (code is None or rc == code), (rc, message)
    assert error in message, message


def _pool(p):
    p.k_cache, p.v_cache = 0x1000, 0x2000
    p.num_pages, p.page_size, p.num_kv_heads, p.head_dim, p.dtype = 8, 16, 2, 64, _hip.DT_F16
    for n in "kv":
        setattr(p, f"{n}_stride_page", 16 * 2 * 64)
        setattr(p, f"{n}_stride_slot", 2 * 64)
        setattr(p, f"{n}_stride_head", 64)


def test_pool_errors():
    fn = _hip.lib().fat_copy_pages
    _refused(fn, None, "required")
    a = _hip.CopyPagesArgs(count=1)
    _refused(fn, a, "src and dst are required")
    a.src, a.dst = 0x3000, 0x4000
    _refused(fn, a, "k_cache and v_cache are required")
    _pool(a.pool)
    for field, value, error in (("num_pages", 0, "must be positive"), ("page_size", -1, "must be positive"),
                                ("num_kv_heads", 0, "must be positive"), ("head_dim", 0, "must be positive"),
                                ("dtype", 17, "unknown dtype 17"), ("page_size", 1 << 30, "more than 1 GiB"),
                                ("k_stride_page", 0, "strides"), ("v_stride_slot", -128, "strides"),
                                ("quant_k_cache", 0x5000, "in pairs"), ("k_scale", 0x5000, "in pairs")):
        kept = getattr(a.pool, field)
        setattr(a.pool, field, value)
        _refused(fn, a, error)
        setattr(a.pool, field, kept)
    a.count = -1
    _refused(fn, a, "count must be")
    a.count = 1 << 31
    _refused(fn, a, "count must be")
    a.count = 0
    assert fn(ctypes.byref(a), None) == 0  # nothing to copy: no launch


def test_fork_errors():
    fn = _hip.lib().fat_fork_sequences
    _refused(fn, None, "required")
    a = _hip.ForkArgs(count=1)
    _refused(fn, a, "required")
    for f in ("parents", "children", "pages", "page_table", "seq_lens"):
        setattr(a, f, 0x1000)
    _refused(fn, a, "k_cache and v_cache are required")
    _pool(a.pool)
    a.batch, a.max_pages, a.page_table_stride = 4, 3, 3
    for field, value, error in (("count", -1, "invalid"), ("batch", 0, "invalid"), ("max_pages", 0, "invalid"),
                                ("page_table_stride", 2, "invalid"), ("count", 5, "at most")):
        kept = getattr(a, field)
        setattr(a, field, value)
        _refused(fn, a, error, 1)
        setattr(a, field, kept)
    a.count = 0
    assert fn(ctypes.byref(a), None) == 0


def test_free_and_compact_errors():
    lib = _hip.lib()
    _refused(lib.fat_free_sequences, None, "required")
    a = _hip.FreeArgs(count=1)
    _refused(lib.fat_free_sequences, a, "required")
    for f in ("rows", "pages", "num_free"):
        setattr(a, f, 0x1000)
    _refused(lib.fat_free_sequences, a, "pointer is NULL")
    for f in ("seq_lens", "page_table", "workspace"):
        setattr(a, f, 0x1000)
    a.batch, a.max_pages, a.num_pages, a.page_size, a.page_table_stride = 2, 3, 8, 16, 3
    for field, value in (("batch", -1), ("max_pages", 0), ("num_pages", 0), ("num_pages", (1 << 30) + 1),
                         ("page_size", 0), ("page_table_stride", 2), ("workspace", 0x1008)):
        kept = getattr(a, field)
        setattr(a, field, value)
        _refused(lib.fat_free_sequences, a, "invalid", 1)
        setattr(a, field, kept)
    a.count = -1
    _refused(lib.fat_free_sequences, a, "count must be", 1)

    _refused(lib.fat_compact_pages, None, "required")
    c = _hip.CompactArgs()
    _refused(lib.fat_compact_pages, c, "required")
    c.remap, c.num_used = 0x1000, 0x1000
    _refused(lib.fat_compact_pages, c, "k_cache and v_cache")
    _pool(c.pool)
    _refused(lib.fat_compact_pages, c, "pointer is NULL")
    for f in ("seq_lens", "page_table", "workspace"):
        setattr(c, f, 0x1000)
    c.batch, c.max_pages, c.page_table_stride = 2, 3, 2
    _refused(lib.fat_compact_pages, c, "invalid", 1)


def test_pages_workspace():
    size = _hip.lib().fat_pages_workspace_bytes
    assert size(0) == 0 and size(-5) == 0
    # flags (1 byte) and three lists (4 bytes each) of whole groups of 4096 ids; a count per group and one more
    for pages, groups in ((1, 1), (4096, 1), (4097, 2), (1 << 30, 1 << 18)):
        assert size(pages) == groups * 4096 * 13 + 4 * (groups + 1)


def test_shared_decode_errors():
    lib = _hip.lib()
    fn = lib.fat_paged_decode_shared
    _refused(fn, None, "NULL")
    a = _hip.SharedArgs()
    _refused(fn, a, "NULL")
    for f in ("q", "k_cache", "v_cache", "page_table", "seq_lens", "cu_groups", "prefix_lens", "out", "workspace"):
        setattr(a, f, 0x1000)
    a.batch, a.groups, a.max_group, a.num_heads, a.num_kv_heads, a.head_dim = 2, 1, 2, 4, 2, 128
    a.page_size, a.num_pages, a.max_pages, a.q_len, a.page_table_stride = 16, 8, 4, 1, 4
    a.q_dtype = a.kv_dtype = _hip.DT_F16
    a.q_stride_b, a.q_stride_t, a.q_stride_h = 512, 512, 128
    a.out_stride_b, a.out_stride_t, a.out_stride_h = 512, 512, 128
    for n in "kv":
        setattr(a, f"{n}_stride_page", 16 * 2 * 128)
        setattr(a, f"{n}_stride_slot", 2 * 128)
        setattr(a, f"{n}_stride_head", 128)
    a.prefix_split, a.prefix_chunk, a.split, a.chunk = 2, 32, 1, 32
    a.softmax_scale = 0.1
    a.workspace_bytes = 1 << 20
    for field, value in (("batch", 0), ("groups", 0), ("max_group", 0), ("num_heads", 3), ("num_kv_heads", 0),
                         ("page_size", 0), ("num_pages", 0), ("max_pages", 0), ("q_len", 65), ("q_len", 0),
                         ("prefix_split", 0), ("prefix_split", 65), ("split", 0), ("split", 65), ("prefix_chunk", 31),
                         ("chunk", 0), ("row_blocks", 2), ("workspace_bytes", 16), ("head_dim", 96),
                         ("q_dtype", _hip.DT_F32), ("kv_dtype", _hip.DT_BF16), ("kv_dtype", _hip.DT_I8),
                         ("k_stride_slot", 3), ("k_cache", 0x1008)):
        kept = getattr(a, field)
        setattr(a, field, value)
        _refused(fn, a, "")
        setattr(a, field, kept)
    # (acc, m, l) in fp32 per query row, head and partial
    assert lib.fat_paged_decode_shared_workspace_bytes(2, 4, 128, 3) == 2 * 4 * 3 * 130 * 4
