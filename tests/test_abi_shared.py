"""C entry of shared-prefix decode: what it refuses, with which code and words.  A
launch that fails for lack of a device is another code (3), so no refusal here is one
by chance, and nothing here launches a kernel."""

from __future__ import annotations

import ctypes

import pytest

from flashattntile_amd import _hip

INVALID, UNSUPPORTED = 1, 2


def _args(**more):
    """A launch of two sequences of 4 / 2 heads whose buffers lie apart."""
    a = _hip.SharedArgs()
    for i, f in enumerate(("q", "k_cache", "v_cache", "page_table", "seq_lens", "cu_groups", "prefix_lens", "out")):
        setattr(a, f, 0x1000 * (i + 1))
    a.workspace, a.workspace_bytes = 0x100000, 1 << 20
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
    for f, value in more.items():
        setattr(a, f, value)
    return a


def _refused(a, code, error):
    rc = _hip.lib().fat_paged_decode_shared(ctypes.byref(a), None)
    message = _hip.lib().fat_last_error().decode()
    assert rc == code and error in message, (rc, message)


NEED = 2 * 4 * 3 * 130 * 4  # bytes of the launch's partials


@pytest.mark.parametrize("q_len", [0, 1])
@pytest.mark.parametrize("field", ["q", "k_cache", "v_cache", "page_table", "seq_lens", "cu_groups", "prefix_lens", "out"])
def test_a_workspace_on_top_of_another_buffer(field, q_len):
    """The partials are written while the others are read."""
    a = _args(q_len=q_len)
    base = getattr(a, field)
    for at in (base, (base - NEED + 16) // 16 * 16):
        _refused(_args(q_len=q_len, workspace=at + 0x1000000, **{field: base + 0x1000000}), INVALID, "overlaps")


def test_a_workspace_on_top_of_the_scales():
    for field in ("k_scale", "v_scale"):
        a = _args(kv_dtype=_hip.DT_I8, k_scale=0x200000, v_scale=0x300000)
        setattr(a, field, a.workspace + NEED - 16)
        _refused(a, INVALID, "overlaps")


@pytest.mark.parametrize("more,code,error", [
    ({"q": 0}, INVALID, "NULL"), ({"workspace": 0}, INVALID, "NULL"), ({"batch": 0}, INVALID, "must be positive"),
    ({"groups": 0}, INVALID, "must be positive"), ({"max_group": 0}, INVALID, "must be positive"),
    ({"num_kv_heads": 0}, INVALID, "must be positive"), ({"page_size": 0}, INVALID, "must be positive"),
    ({"num_heads": 3}, INVALID, "divisible"), ({"max_pages": 1 << 28}, INVALID, "overflows int32 positions"),
    ({"q_len": 65}, INVALID, "q_len 65"), ({"q_len": -1}, INVALID, "q_len -1"),
    ({"prefix_split": 0}, INVALID, "must be in [1, 64]"), ({"split": 65}, INVALID, "must be in [1, 64]"),
    ({"prefix_chunk": 31}, INVALID, "multiples of 32"), ({"chunk": 0}, INVALID, "multiples of 32"),
    ({"row_blocks": 2}, INVALID, "row_blocks"), ({"prefix_chunk": 1 << 30, "prefix_split": 2}, INVALID, "overflow"),
    ({"head_dim": 96}, UNSUPPORTED, "head_dim 64 or 128"), ({"q_dtype": _hip.DT_F32}, UNSUPPORTED, "fp16/bf16"),
    ({"kv_dtype": _hip.DT_BF16}, UNSUPPORTED, "fp16/bf16"), ({"kv_dtype": _hip.DT_I8}, INVALID, "k_scale and v_scale"),
    ({"k_stride_slot": 3}, INVALID, "16-byte aligned"), ({"q": 0x1008}, INVALID, "16-byte aligned"),
    ({"workspace": 0x100008}, INVALID, "16-byte aligned"), ({"workspace_bytes": 16}, INVALID, "bytes of workspace"),
    ({"workspace_bytes": NEED - 1}, INVALID, "bytes of workspace"),
    ({"k_stride_page": 1 << 31}, UNSUPPORTED, "below 4 GiB"), ({"page_size": 1 << 24, "max_pages": 1}, UNSUPPORTED, "strides"),
])
def test_refusals(more, code, error):
    _refused(_args(**more), code, error)


@pytest.mark.parametrize("batch,q_len,heads,kv_heads,code,error", [
    # batch x q_len = 2^31: the rows, and with them the bytes of workspace, were counted in 32 bits
    (1 << 25, 64, 1, 1, UNSUPPORTED, "query rows"), (1 << 30, 2, 1, 1, UNSUPPORTED, "query rows"),
    (2 ** 31 - 1, 64, 1, 1, UNSUPPORTED, "query rows"),
    # 2^31 rows of one KV head
    (1 << 24, 1, 128, 1, UNSUPPORTED, "query rows"), (1 << 20, 64, 64, 2, UNSUPPORTED, "query rows"),
    # 2^30 rows: their workspace is what is missing
    (1 << 24, 64, 1, 1, INVALID, "bytes of workspace"), (1 << 24, 1, 64, 1, INVALID, "bytes of workspace"),
])
def test_rows_beyond_32_bits(batch, q_len, heads, kv_heads, code, error):
    _refused(_args(batch=batch, max_group=1, q_len=q_len, num_heads=heads, num_kv_heads=kv_heads), code, error)
