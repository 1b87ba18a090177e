"""Decode of sequences that share a prefix: host side of ``csrc/decode_shared.hip``.

:func:`paged_decode_attention_shared` computes what
:func:`~flashattntile_amd.kernels.decode.paged_decode_attention`, its 8-bit and
its multi-token forms compute, for a batch whose sequences come in groups with
the same first keys (a system prompt, the samples of one prompt, questions about
one document): those keys are read once for all queries of the group instead of
once per sequence (the reference has no counterpart; its decode reads every
sequence's own table, ``kernels/decode.py:47-127``).

:func:`paged_decode_shared_launch` is the sync-free entry below the validation.
"""

from __future__ import annotations

import math

import torch

from .. import _hip
from ..paging import PagedKVCache, _check_layout
from .decode import (_QUANT_DTYPES, _decode, _dense_scales, _require_rocm, _resolve_config, _scale_of)

__all__ = ["paged_decode_attention_shared", "paged_decode_shared_launch", "shared_splits"]

# Partials of a launch: prefix_split chunks of prefix_chunk keys of a group's
# prefix, split chunks of chunk keys of a sequence's own; None: shared_splits.
# row_blocks: rows of a workgroup on a prefix, in 32s (1 or 4; None: by the rows).
_CONFIG_KEYS = ("prefix_split", "split", "row_blocks")


def _check_inputs(q, cache: PagedKVCache, cu_groups, prefix_lens, scales) -> None:
    """The host-only checks."""
    if not isinstance(cache, PagedKVCache):
        raise TypeError("cache must be a PagedKVCache")
    _check_layout(cache)
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [batch, heads, head_dim] or [batch, q_len, heads, head_dim], got {tuple(q.shape)}")
    if q.shape[0] != cache.batch_size:
        raise ValueError(f"q batch {q.shape[0]} != cache batch {cache.batch_size}")
    if q.shape[-1] != cache.head_dim:
        raise ValueError(f"q head_dim {q.shape[-1]} != cache head_dim {cache.head_dim}")
    if q.shape[-2] % cache.num_kv_heads != 0:
        raise ValueError(f"num_heads {q.shape[-2]} must be divisible by num_kv_heads {cache.num_kv_heads}")
    if q.dim() == 4 and not 1 <= q.shape[1] <= 64:
        raise ValueError(f"multi-token decode takes 1 to 64 tokens per sequence, got {q.shape[1]}")
    for name, t in (("cu_groups", cu_groups), ("prefix_lens", prefix_lens)):
        if t.dim() != 1 or t.dtype != torch.int32:
            raise ValueError(f"{name} must be a 1-D int32 tensor")
    if cu_groups.shape[0] != prefix_lens.shape[0] + 1 or prefix_lens.shape[0] == 0:
        raise ValueError(f"cu_groups must have one entry more than prefix_lens, at least two; got "
                         f"{cu_groups.shape[0]} and {prefix_lens.shape[0]}")
    device = q.device
    if not (cache.k_cache.device == device == cache.page_table.device == cu_groups.device == prefix_lens.device):
        raise ValueError("q, the cache, its page table, seq_lens, cu_groups and prefix_lens must live on one device")
    quantized = cache.k_cache.dtype in _QUANT_DTYPES
    if quantized != (scales is not None):
        raise ValueError("an int8/float8 cache needs scales, and only such a cache takes them")
    if quantized:
        if q.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"quantised decode requires fp16/bf16 queries, got {q.dtype}")
        k_scale = scales["k"] if isinstance(scales, dict) else scales.k
        v_scale = scales["v"] if isinstance(scales, dict) else scales.v
        expected = (cache.num_pages, cache.num_kv_heads)
        if tuple(k_scale.shape) != expected or tuple(v_scale.shape) != expected:
            raise ValueError(f"scales must have shape {expected}, got {tuple(k_scale.shape)}")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError("scales must be float32")
        if k_scale.device != q.device or v_scale.device != q.device:
            raise ValueError("scales must live on q's device")
    elif cache.k_cache.dtype != q.dtype:
        raise ValueError(f"q dtype {q.dtype} must match cache dtype {cache.k_cache.dtype}")


def _assess(r: list[int], q, cache: PagedKVCache) -> None:
    """The device-side checks on their numbers (``FAT_CHECK_SHARED``)."""
    tokens = q.shape[1] if q.dim() == 4 else 1
    flags = r[7]
    if r[3] != 0:
        raise ValueError("cu_groups must start at 0")
    if flags & 1:
        raise ValueError("cu_groups must be non-decreasing")
    if r[4] != cache.batch_size:
        raise ValueError(f"cu_groups must end at the batch size {cache.batch_size}, got {r[4]}")
    if flags & 2:
        raise ValueError("prefix_lens must be non-negative")
    if r[0] < 0:
        raise AssertionError("seq_lens must be non-negative")
    if r[1] > cache.capacity:
        raise AssertionError(f"seq_len {r[1]} exceeds page-table capacity {cache.capacity}")
    if r[0] < tokens:
        raise ValueError(f"decode requires every sequence to hold its {tokens} new token(s) (shortest seq_len {r[0]})")
    if flags & 4:
        raise ValueError("a group's prefix must be no longer than what the first new token of each of its sequences "
                         "sees (prefix_lens[g] <= seq_lens[b] - q_len + 1)")
    if flags & 8:
        raise ValueError("the sequences of a group must share the pages that its prefix fills")
    if r[12] < 0:
        raise AssertionError("page_table contains a negative page id")
    if r[13] >= cache.num_pages:
        raise AssertionError(f"page_table references page {r[13]} but cache has {cache.num_pages} pages")


def _takes(q, cache: PagedKVCache) -> bool:
    """Whether the shared-prefix kernel takes the launch."""
    if q.dtype not in (torch.float16, torch.bfloat16) or q.shape[-1] not in (64, 128):
        return False
    k, v, size = cache.k_cache, cache.v_cache, cache.page_size
    if size >= 2 ** 24 or cache.page_table.shape[1] * size > 2 ** 31 - 4097:
        return False
    eb = k.element_size()
    bits = k.data_ptr() | v.data_ptr()
    for t in (k, v):
        page, slot, head, _ = t.stride()
        if eb * page >= 2 ** 32 or eb * slot >= 2 ** 24 or eb * slot * size >= 2 ** 32:
            return False
        bits |= eb * (page | slot | head)
    return bits % 16 == 0


def _ordinary_takes(cache: PagedKVCache, tokens: int) -> bool:
    """Whether ordinary decode takes a 16-bit launch that the shared-prefix kernel
    takes: with several tokens its MFMA kernel, on power-of-two pages of at least
    the rows that one of its loads covers."""
    size = cache.page_size
    return tokens == 1 or (size & (size - 1) == 0 and size >= (4 if cache.head_dim == 128 else 8))


def _one_by_one(q, cache: PagedKVCache):
    """Every token of a multi-token call as a sequence of its own, for the kernels
    that take one query per sequence: token t sees the first len - T + 1 + t keys."""
    batch, tokens, heads, dim = q.shape
    lens = cache.seq_lens[:, None] + torch.arange(1 - tokens, 1, dtype=torch.int32, device=q.device)
    table = cache.page_table[:, None].expand(-1, tokens, -1).reshape(batch * tokens, -1)
    return q.view(batch * tokens, heads, dim), PagedKVCache(cache.k_cache, cache.v_cache, table, lens.view(-1),
                                                            cache.page_size)


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def shared_splits(num_kv_heads: int, group_rows: int, own_tiles: int, groups: float, max_prefix: int,
                  sequences: float, max_own: int, rows: int, batch: int | None = None) -> dict:
    """Partials of a launch: ``prefix_split`` x ``prefix_chunk`` keys of every
    prefix, ``split`` x ``chunk`` own keys of every sequence.

    ``group_rows``: query rows of the largest group and KV head; ``own_tiles``:
    32-row tiles of a sequence; ``rows``: query rows of all heads.  ``groups`` and
    ``sequences`` count those of the longest's length (the sum of all lengths by the
    longest): splits that fit the longest leave the chip to the others' few
    workgroups otherwise.  ``batch``: all sequences (default: ``sequences``), whose
    workgroups a split has too, keys or not.
    """
    # n chunks of K keys cost a chain of a K / n us, and n b for their partials (1040
    # bytes per row, written and read) and workgroups: least at sqrt(a K / b), a little
    # below as the chunks overlap.  No more workgroups than CUs.  Chunks taken, us at
    # 1 chunk, at them and at twice them (fp16, 8 KV heads): 1 group of 8 rows x 4096
    # keys 17: 52.5, 12.8, 14.2; of 256 x 1024 5: 35.3, 19.0, 21.2; 4 of 128 x 2048 5:
    # 59.9, 31.0, 37.2; 1 of 512 x 32768 8: 170 (16: 180).
    tile, per_key = (128, 0.022) if group_rows > 32 else (32, 0.0105)
    items = max(1.0, groups * num_kv_heads * -(-group_rows // tile))
    best = 0.8 * math.sqrt(per_key * max_prefix / (2.0e-4 * rows + 0.01 * items))
    prefix_split = max(1, min(round(min(best, 256 / items)), 64, max_prefix // 32))
    # Four workgroups of own keys per CU (128 sequences of 100 to 2000 keys on fp8: 1
    # chunk 66.6 us, 2 60.4, 4 62.7, 8 72.6), and as for prefixes: a chunk costs 1.7 ns
    # per workgroup, those without keys among them (bf16, one long sequence among short
    # ones of 100 keys, us at the chunks taken and at 64: 128 sequences, one of 32768
    # keys, 13: 104, 185; 256 of 4 tokens 9: 190, 355; 256 of 8, one of 65536, 13: 312,
    # 471).
    per_slot = num_kv_heads * own_tiles
    split = max(1, min(int(1024 / max(1.0, sequences * per_slot)), 64, max_own // 256))
    if split > 1:
        per_slot *= max(batch or 0, sequences)
        split = max(1, min(split, round(math.sqrt(0.0092 * max_own / (0.15 + 0.0017 * per_slot)))))
    # At most 512 MiB of partials, where two slots fit that (520 bytes a row at head_dim
    # 128; all 128 slots of 8065 rows do).
    if rows > 8000:
        slots = 2 ** 29 // (520 * rows)
        prefix_split = min(prefix_split, max(1, slots - 1))
        split = min(split, max(1, slots - prefix_split))
    return _chunks(prefix_split, split, max_prefix, max_own)


def _chunks(prefix_split: int, split: int, max_prefix: int, max_own: int) -> dict:
    return {"prefix_split": prefix_split, "prefix_chunk": _up(max(1, -(-max_prefix // prefix_split)), 32),
            "split": split, "chunk": _up(max(1, -(-max_own // split)), 32)}


def _block(q, cache, cu_groups, prefix_lens, scale, scales, out=None):
    """The argument block but for its splits, its output, and what has to live
    until the launch is enqueued."""
    if cache.k_cache.stride(-1) != 1 or cache.v_cache.stride(-1) != 1:
        raise ValueError("k_cache and v_cache need a contiguous head_dim axis")
    if out is None:
        out = torch.empty_like(q)
    sc = None if scales is None else _dense_scales(scales)
    a = _hip.shared_args(q, cache, cu_groups, prefix_lens, out, scale, *((sc["k"], sc["v"]) if sc else ()))
    return a, out, sc


def _dense_query(q: torch.Tensor) -> torch.Tensor:
    """``q`` with the strides of its shape (torch calls a tensor contiguous whatever
    those of its axes of one entry are), on a 16-byte boundary."""
    q = q.contiguous()
    if q.data_ptr() % 16:
        return q.clone(memory_format=torch.contiguous_format)
    return q.view(-1).view(q.shape) if 1 in q.shape else q


def _dense(cache: PagedKVCache, cu_groups, prefix_lens):
    """The cache, groups and prefixes with the table, lengths and lists that the
    kernels read (unit strides)."""
    pt, sl = cache.page_table, cache.seq_lens
    if pt.stride(1) != 1 or not sl.is_contiguous():
        cache = PagedKVCache(cache.k_cache, cache.v_cache, pt if pt.stride(1) == 1 else pt.contiguous(),
                             sl.contiguous(), cache.page_size)
    return cache, cu_groups.contiguous(), prefix_lens.contiguous()


def _launch(a, q, cfg: dict, max_group: int, workspace=None) -> None:
    rows = q.shape[0] * (q.shape[1] if q.dim() == 4 else 1)
    # fat_paged_decode_shared_workspace_bytes: (acc, m, l) per (query row, head, partial)
    need = 4 * rows * q.shape[-2] * (cfg["prefix_split"] + cfg["split"]) * (q.shape[-1] + 2)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    a.max_group = max_group
    a.prefix_split, a.prefix_chunk = cfg["prefix_split"], cfg["prefix_chunk"]
    a.split, a.chunk = cfg["split"], cfg["chunk"]
    a.row_blocks = cfg.get("row_blocks", 0)
    _hip.shared_with_args(a, workspace, _hip.current_stream_handle(q.device))


def paged_decode_shared_launch(q: torch.Tensor, cache: PagedKVCache, cu_groups: torch.Tensor,
                               prefix_lens: torch.Tensor, softmax_scale: float, max_prefix: int, max_own: int,
                               max_group: int | None = None, out: torch.Tensor | None = None,
                               workspace: torch.Tensor | None = None, scales=None,
                               config: dict | None = None) -> torch.Tensor:
    """Enqueue the shared-prefix decode without validation or synchronisation
    (capture, serving loops that validated once).

    ``max_prefix`` and ``max_own`` are the groups' longest prefix and the most
    keys behind one; they size the grid, and more keys than they say are still
    attended.  No group may have more sequences than ``max_group`` (default: the
    batch): the outputs of those beyond are undefined.  Lengths, table, groups
    and prefixes are read on the device at every run.
    ``q`` must be contiguous and begin on a 16-byte boundary (else it is copied);
    ``out`` (of ``q``'s shape, dtype and device, head_dim contiguous) and
    ``workspace`` (contiguous, 4 x rows x heads x partials x (head_dim + 2) bytes; a
    smaller one is left aside) may be passed in to avoid allocations; launches that
    may run at the same time, replays of two graphs among them, need a workspace each.
    Takes fp16/bf16 queries at head_dim 64 or 128, else raises.
    """
    with _hip.on_device(q.device):
        q = _dense_query(q)
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device
                                or out.stride(-1) != 1):
            raise ValueError(f"out must be a {q.dtype} tensor of q's shape {tuple(q.shape)} on its device, head_dim "
                             f"contiguous")
        if workspace is not None and (workspace.device != q.device or not workspace.is_contiguous()):
            raise ValueError("workspace must be a contiguous tensor on q's device")
        cache, cu_groups, prefix_lens = _dense(cache, cu_groups, prefix_lens)
        a, out, _keep = _block(q, cache, cu_groups, prefix_lens, softmax_scale, scales, out)
        cfg = _resolve(config, q, cache, max_prefix, max_own, max_group or q.shape[0], prefix_lens.shape[0],
                       q.shape[0])
        _launch(a, q, cfg, max_group or q.shape[0], workspace)
    return out


def _resolve(config, q, cache, max_prefix: int, max_own: int, max_group: int, groups: float,
             sequences: float) -> dict:
    per_seq = (q.shape[1] if q.dim() == 4 else 1) * q.shape[-2] // cache.num_kv_heads
    cfg = shared_splits(cache.num_kv_heads, max_group * per_seq, -(-per_seq // 32), groups, max_prefix, sequences,
                        max_own, q.shape[0] * per_seq * cache.num_kv_heads, q.shape[0])
    given = _given(config) if config else None
    if not given:
        return cfg
    row_blocks = given.pop("row_blocks", 0)
    cfg = _chunks(given.get("prefix_split", cfg["prefix_split"]), given.get("split", cfg["split"]), max_prefix,
                  max_own)
    cfg["row_blocks"] = row_blocks
    return cfg


def _given(config: dict | None) -> dict:
    """What ``config`` sets, checked."""
    unknown = set(config or ()) - set(_CONFIG_KEYS)
    if unknown:
        raise ValueError(f"unknown shared decode config keys: {sorted(unknown)}")
    given = {k: v for k, v in (config or {}).items() if v is not None}
    for k, v in given.items():
        if k == "row_blocks":
            if v not in (1, 4):
                raise ValueError(f"row_blocks must be None, 1 or 4, got {v}")
        elif not isinstance(v, int) or isinstance(v, bool) or not 1 <= v <= 64:
            raise ValueError(f"{k} must be an integer in [1, 64], got {v}")
    return given


def paged_decode_attention_shared(
    q: torch.Tensor,
    cache: PagedKVCache,
    cu_groups: torch.Tensor,
    prefix_lens: torch.Tensor,
    softmax_scale: float | None = None,
    config: dict | None = None,
    scales=None,
) -> torch.Tensor:
    """Paged decode of groups of sequences with the same first keys.

    ``q``: ``[batch, heads, head_dim]`` or, multi-token, ``[batch, q_len, heads,
    head_dim]``, as :func:`paged_decode_attention` and ``..._multi`` take it.
    ``cu_groups`` (int32 ``[groups + 1]``, from 0 to batch): sequences
    ``cu_groups[g] .. cu_groups[g + 1] - 1`` are group g.  ``prefix_lens`` (int32
    ``[groups]``): the keys they share, read through the table row of the
    group's first sequence; ``seq_lens`` counts them too.  A prefix of 0 and
    groups of one sequence are valid; one that ends inside a page too (every
    sequence then has its own copy of that page, as
    :func:`~flashattntile_amd.page_ops.fork_sequences` makes it), the pages it
    fills must be the same ids in all rows of the group.  ``scales`` selects an
    int8 / float8_e4m3fn cache, where that last page is read per sequence (its scale
    and codes depend on each one's own keys).  ``config``: ``prefix_split`` and ``split``,
    partials per prefix and per sequence (default: by the lengths).

    Shapes that the kernel isn't built for (fp32, other head_dims than 64 and
    128) run as ordinary decode, which reads the prefix once per sequence, and per
    token of a multi-token query, and so do batches without ``scales`` in which no
    two sequences share a key; ``config`` does not apply to the former.  K and V
    rows are 16-byte aligned, as for every decode.  On fp16 caches the softmax's
    numerators are rounded to fp16 (in bf16 and on 8-bit caches to two bf16 parts).
    Returns ``q``'s shape and dtype.
    """
    _check_inputs(q, cache, cu_groups, prefix_lens, scales)
    _require_rocm(q, cache, "paged_decode_attention_shared")
    if cache.batch_size == 0 or cache.page_table.numel() == 0:
        raise ValueError("decode requires every sequence to hold at least one cached token")
    tokens = q.shape[1] if q.dim() == 4 else 1
    given = _given(config)
    scale = _scale_of(q, softmax_scale)
    device = q.device
    with _hip.on_device(device):
        q = _dense_query(q)
        stream = _hip.current_stream_handle(device)
        cache, cu_groups, prefix_lens = _dense(cache, cu_groups, prefix_lens)
        check = _hip.check_begin(_hip.CHECK_SHARED, stream, device, cu_q=cu_groups, seq_lens=cache.seq_lens,
                                 page_table=cache.page_table, page_size=cache.page_size, ids=(prefix_lens,),
                                 tokens=tokens)
        # prepared while the check kernel runs
        block = _block(q, cache, cu_groups, prefix_lens, scale, scales) if _takes(q, cache) else None
        r = check.wait()
        _assess(r, q, cache)
        # Nothing is shared: 64 sequences of 4100 keys took 221 us here, 195 as ordinary
        # decode (which rounds an 8-bit cache's scaled values to bf16, and so isn't taken there).
        if block is None or (r[9] == r[11] and scales is None and not given and _ordinary_takes(cache, tokens)):
            pages, shape = r[2], q.shape
            if block is None and tokens > 1:
                q, cache = _one_by_one(q, cache)
                pages, tokens = pages * tokens, 1
            cfg = _resolve_config(None, q, cache, r[1], pages, q_len=tokens)
            return _decode(q, cache, scale, cfg, None, None if scales is None else _dense_scales(scales)).view(shape)
        a, out, keep = block
        prefix, own = r[6], r[8]
        groups, sequences = r[9] / max(1, prefix), r[10] / max(1, own)
        if scales is not None:  # a prefix's last page is among its sequences' own keys
            own = min(r[1], own + min(prefix, cache.page_size - 1))
            prefix -= prefix % cache.page_size
        cfg = _resolve(config, q, cache, prefix, own, max(1, r[5]), groups, sequences)
        _launch(a, q, cfg, max(1, r[5]))
        del keep
        return out
