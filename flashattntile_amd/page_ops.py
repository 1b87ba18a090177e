"""Operations on the pages of a paged cache: copy, fork, free and compact.

What an engine that shares pages among its sequences needs beside
:func:`~flashattntile_amd.paging.append_tokens` (the reference has none of it:
its engine allocates every sequence its own pages, ``paging.py:133-169``):

* :func:`copy_pages` copies pages of the pool to others;
* :func:`fork_sequences` makes empty batch rows forks of others, which share
  their parents' whole pages;
* :func:`free_sequences` empties rows and lists the pages no row uses any more;
* :func:`compact_pages` moves the pages in use to the front of the pool.

The tables and lengths say everything: a page is in use if a row's used columns
name it, however many do.  Row ``b`` uses its first ``ceil(seq_lens[b] /
page_size)`` columns; where an engine gives rows pages ahead of their tokens
(:func:`~flashattntile_amd.paging.allocate` does so for all of them), ``held``
(int32 ``[batch]``) says how many columns a row holds.  Columns behind are
neither counted nor renumbered.

Each takes the cache's 8-bit copy as ``quantized=(qcache, scales)``, as
``append_tokens`` does, and an int8 / float8_e4m3fn cache with its ``scales``;
what is given moves together, byte for byte.  Lists of ids are contiguous or
strided int32 vectors on the cache's device.  On a ROCm cache the work is HIP
kernels on the current stream (``csrc/pages.hip``) and the checks cost one
launch that the host polls; ``validate=False`` leaves them out (capture, serving
loops): pairs and rows that are out of range are then skipped on the device.
CPU caches take torch, always checked.  Bad arguments raise ``AssertionError``,
as the cache's other checks do, before anything is changed.
"""

from __future__ import annotations

import torch

from .paging import PagedKVCache, _assess_cache, _check_layout, _quant_pair, _require

__all__ = ["copy_pages", "fork_sequences", "free_sequences", "compact_pages"]


def _eight_bit(dtype: torch.dtype) -> bool:
    return dtype in (torch.int8, getattr(torch, "float8_e4m3fn", None))


def _parts(cache: PagedKVCache, quantized, scales, shared_table: bool):
    """Check the 8-bit copy and the scales; returns ``(copy, scales)``:
    ``(qk, qv, k_scale, v_scale)`` or None, and ``(k_scale, v_scale)`` or None."""
    _check_layout(cache)
    if quantized is not None:
        _require(scales is None, "scales belong to an 8-bit cache; those of an 8-bit copy come with it")
        _require(not _eight_bit(cache.k_cache.dtype), "an int8/float8 cache has no 8-bit copy")
        copy = _quant_pair(cache, quantized)
        _require(copy[2].stride() == copy[3].stride(), "k and v scales must share strides")
        if cache.k_cache.is_cuda:
            _require(copy[0].stride(3) == 1 and copy[1].stride(3) == 1,
                     "the head_dim axis of the quantised pages must be contiguous")
        qcache = quantized[0]
        if shared_table:
            for name in ("page_table", "seq_lens"):
                mine, theirs = getattr(cache, name), getattr(qcache, name)
                _require(mine.data_ptr() == theirs.data_ptr() and mine.shape == theirs.shape,
                         f"the 8-bit copy must share the cache's {name} (quantize_cache gives it the same tensor)")
        return copy, None
    _require(_eight_bit(cache.k_cache.dtype) == (scales is not None),
             "an int8/float8 cache needs scales, and only such a cache takes them")
    if scales is None:
        return None, None
    sk = scales["k"] if isinstance(scales, dict) else scales.k
    sv = scales["v"] if isinstance(scales, dict) else scales.v
    want = (cache.num_pages, cache.num_kv_heads)
    _require(tuple(sk.shape) == want and tuple(sv.shape) == want,
             f"scales must be [{want[0]}, {want[1]}], got {tuple(sk.shape)} / {tuple(sv.shape)}")
    _require(sk.dtype == torch.float32 and sv.dtype == torch.float32, "scales must be float32")
    _require(sk.device == cache.k_cache.device and sv.device == sk.device, "scales must live on the cache device")
    _require(sk.stride() == sv.stride(), "k and v scales must share strides")
    return None, (sk, sv)


def _ids(cache: PagedKVCache, name: str, t: torch.Tensor, count: int | None = None) -> torch.Tensor:
    _require(isinstance(t, torch.Tensor) and t.dim() == 1 and t.dtype == torch.int32,
             f"{name} must be a 1-D int32 tensor")
    _require(t.device == cache.k_cache.device, f"{name} must be on the cache device")
    _require(count is None or t.shape[0] == count, f"{name} must have {count} entries, got {t.shape[0]}")
    return t.contiguous()


def _held(cache: PagedKVCache, held: torch.Tensor | None, written: bool) -> torch.Tensor | None:
    if held is None:
        return None
    _require(held.dim() == 1 and held.dtype == torch.int32 and held.shape[0] == cache.batch_size,
             f"held must be int32 [{cache.batch_size}]")
    _require(held.device == cache.k_cache.device, "held must be on the cache device")
    _require(held.is_contiguous() or not written, "held must be contiguous (it is updated in place)")
    return held.contiguous()


def _check_rocm(cache: PagedKVCache) -> None:
    """The layout that the kernels read, for a ROCm cache."""
    dev = cache.k_cache.device
    _require(cache.page_table.device == dev and cache.seq_lens.device == dev,
             "page_table and seq_lens must live on the cache device")
    _require(cache.k_cache.stride(3) == 1 and cache.v_cache.stride(3) == 1, "the head_dim axis must be contiguous")
    _require(cache.page_table.stride(1) == 1, "page_table rows must be contiguous")
    _require(cache.seq_lens.is_contiguous(), "seq_lens must be contiguous")


def _copy_flags(flags: int, cache: PagedKVCache) -> None:
    _require(not flags & 1, f"src holds a page outside [0, {cache.num_pages})")
    _require(not flags & 2, f"dst holds a page outside [0, {cache.num_pages})")
    _require(not flags & 4, "dst holds a page twice")
    _require(not flags & 8, "dst holds a page that src holds too")


def _fork_flags(flags: int, cache: PagedKVCache) -> None:
    batch, pages = cache.batch_size, cache.num_pages
    _require(not flags & 1, f"parents holds a row outside [0, {batch})")
    _require(not flags & 2, f"children holds a row outside [0, {batch})")
    _require(not flags & 4, "children holds a row twice")
    _require(not flags & 8, "a row is both parent and child")
    _require(not flags & 16, "children must be empty rows (seq_lens 0: free_sequences them first)")
    _require(not flags & 32, f"a parent's seq_len is negative or exceeds page-table capacity {cache.capacity}")
    _require(not flags & 64, f"page_table maps a parent's last page outside [0, {pages})")
    _require(not flags & 128, f"pages holds a page outside [0, {pages})")
    _require(not flags & 256, "pages holds a page twice")
    _require(not flags & 512, "pages holds a page that a row uses")


def _outside(t: torch.Tensor, limit: int) -> bool:
    return bool(((t < 0) | (t >= limit)).any())


def _planes(cache: PagedKVCache, copy, scales) -> list[torch.Tensor]:
    """Everything that a page consists of (torch indexes no 8-bit floats on the
    CPU: their bits)."""
    planes = [cache.k_cache, cache.v_cache, *(copy or ()), *(scales or ())]
    return [t.view(torch.int8) if _eight_bit(t.dtype) else t for t in planes]


def copy_pages(cache: PagedKVCache, src: torch.Tensor, dst: torch.Tensor, *, quantized=None, scales=None,
               validate: bool = True) -> None:
    """Copy page ``src[i]`` of the pool to page ``dst[i]``, for every i: K and V,
    and the 8-bit copy and scales where given.

    For engines that keep their tables on the host (copy on write, swapping,
    defragmenting).  No page may be in ``dst`` twice, or in ``src`` and ``dst``
    (the copies have no order); a page may be in ``src`` any number of times.
    Table and lengths are not read.
    """
    copy, scales = _parts(cache, quantized, scales, shared_table=False)
    src = _ids(cache, "src", src)
    dst = _ids(cache, "dst", dst, src.shape[0])
    if src.shape[0] == 0:
        return
    _require(cache.num_pages > 0, "src holds a page outside [0, 0)")
    if not cache.k_cache.is_cuda:
        flags = _outside(src, cache.num_pages) | 2 * _outside(dst, cache.num_pages)
        flags |= 4 * (torch.unique(dst).numel() < dst.numel()) | 8 * bool(torch.isin(dst, src).any())
        _copy_flags(flags, cache)
        for t in _planes(cache, copy, scales):
            t[dst.long()] = t[src.long()]
        return

    from . import _hip

    dev = cache.k_cache.device
    _require(cache.k_cache.stride(3) == 1 and cache.v_cache.stride(3) == 1, "the head_dim axis must be contiguous")
    with _hip.on_device(dev):
        stream = _hip.current_stream_handle(dev)
        check = None
        if validate:
            check = _hip.check_begin(_hip.CHECK_COPY, stream, dev, ids=(src, dst), num_pages=cache.num_pages)
        args = _hip.copy_pages_args(cache, src, dst, copy, scales)  # prepared while the check kernel runs
        if check is not None:
            _copy_flags(check.wait()[7], cache)
        _hip.page_operation("fat_copy_pages", args, stream)


def fork_sequences(cache: PagedKVCache, parents: torch.Tensor, children: torch.Tensor, pages: torch.Tensor, *,
                   quantized=None, scales=None, validate: bool = True) -> None:
    """Make row ``children[i]`` a fork of row ``parents[i]``, for every i (the
    samples of a prompt, the beams of a search).

    The child gets the parent's length and page ids: whole pages are shared, and
    stay as they are, since an append goes behind them.  Where the parent's
    length is no multiple of ``page_size``, the child's last page is
    ``pages[i]``, into which the parent's is copied (K and V, and the 8-bit copy
    and scales where given); ``pages[i]`` isn't used where it is one.
    ``pages`` are pages that no row's tokens use, such as :func:`free_sequences`
    lists (not one that another row holds ahead, which this call can't see).
    Children must be empty rows and no child a parent; a parent may have any
    number of children.  Table columns behind the child's last page stay as they
    are.  ``page_table`` and ``seq_lens`` are updated in place, on the device.
    """
    copy, scales = _parts(cache, quantized, scales, shared_table=True)
    parents = _ids(cache, "parents", parents)
    n = parents.shape[0]
    children = _ids(cache, "children", children, n)
    pages = _ids(cache, "pages", pages, n)
    if n == 0:
        return
    _require(cache.num_pages > 0 and cache.page_table.numel() > 0, "the cache holds no pages")
    if not cache.k_cache.is_cuda:
        _fork_torch(cache, parents, children, pages, copy, scales)
        return

    from . import _hip

    _check_rocm(cache)
    dev = cache.k_cache.device
    with _hip.on_device(dev):
        stream = _hip.current_stream_handle(dev)
        check = None
        if validate:
            check = _hip.check_begin(_hip.CHECK_FORK, stream, dev, seq_lens=cache.seq_lens,
                                     page_table=cache.page_table, page_size=cache.page_size,
                                     ids=(parents, children, pages), num_pages=cache.num_pages)
        args = _hip.fork_args(cache, parents, children, pages, copy, scales)  # prepared while the check kernel runs
        if check is not None:
            _fork_flags(check.wait()[7], cache)
        _hip.page_operation("fat_fork_sequences", args, stream)


def _fork_torch(cache, parents, children, pages, copy, scales) -> None:
    batch, size, pool = cache.batch_size, cache.page_size, cache.num_pages
    flags = _outside(parents, batch) | 2 * _outside(children, batch)
    _fork_flags(flags, cache)  # the rest reads the rows
    par, chi = parents.long(), children.long()
    lens = cache.seq_lens[par].long()
    flags = 4 * (torch.unique(chi).numel() < chi.numel()) | 8 * bool(torch.isin(chi, par).any())
    flags |= 16 * bool((cache.seq_lens[chi] != 0).any()) | 32 * _outside(lens, cache.capacity + 1)
    _fork_flags(flags, cache)
    full = torch.div(lens, size, rounding_mode="floor")
    tail = (lens % size != 0).nonzero()[:, 0]
    fresh = pages[tail]
    last = cache.page_table[par[tail], full[tail]]
    flags = 64 * _outside(last, pool) | 128 * _outside(fresh, pool)
    _fork_flags(flags, cache)  # the rest reads the pages' use
    flags = 256 * (torch.unique(fresh).numel() < fresh.numel())
    _fork_flags(flags | 512 * bool(_used_torch(cache, None)[1][fresh.long()].any()), cache)
    rows = cache.page_table[par]
    rows[tail, full[tail]] = fresh
    column = torch.arange(cache.max_pages_per_seq, device=rows.device)
    used = column < torch.div(lens + size - 1, size, rounding_mode="floor")[:, None]
    cache.page_table[chi] = torch.where(used, rows, cache.page_table[chi])
    cache.seq_lens[chi] = lens.to(torch.int32)
    for t in _planes(cache, copy, scales):
        t[fresh.long()] = t[last.long()]


def _used_torch(cache: PagedKVCache, held: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
    """Used columns [batch, max_pages] and used pages [num_pages]."""
    lens = cache.seq_lens.long().clamp_min(0)
    n = torch.div(lens + cache.page_size - 1, cache.page_size, rounding_mode="floor")
    if held is not None:
        n = torch.maximum(n, held.long())
    table = cache.page_table
    columns = torch.arange(table.shape[1], device=table.device) < n[:, None]
    columns &= (table >= 0) & (table < cache.num_pages)
    used = torch.zeros(cache.num_pages, dtype=torch.bool, device=table.device)
    used[table[columns].long()] = True
    return columns, used


def _assess_used(cache: PagedKVCache, held: torch.Tensor | None, stats: tuple[int, int, int, int],
                 beyond: bool) -> None:
    """The checks of lengths, ``held`` and the columns that rows use, on their numbers."""
    _require(not beyond, f"held counts more columns than the page table has ({cache.max_pages_per_seq})")
    _assess_cache(cache, stats, check_pages=held is None)
    if held is not None:  # pages may be held where no row has tokens
        lo, hi = stats[2:]
        _require(lo >= 0, "page_table contains a negative page id")
        _require(hi < cache.num_pages, f"page_table references page {hi} but cache has {cache.num_pages} pages")


def _beyond(cache: PagedKVCache, held: torch.Tensor | None) -> bool:
    return held is not None and bool((held > cache.max_pages_per_seq).any())


def _used_stats(cache: PagedKVCache, held: torch.Tensor | None) -> tuple[int, int, int, int]:
    """Min and max length, and min and max page id of the columns that rows use
    (0, -1 where none does)."""
    lens = cache.seq_lens.long()
    if not lens.numel():
        return 0, 0, 0, -1
    n = torch.div(lens.clamp_min(0) + cache.page_size - 1, cache.page_size, rounding_mode="floor")
    if held is not None:
        n = torch.maximum(n, held.long())
    ids = cache.page_table[torch.arange(cache.page_table.shape[1], device=n.device) < n[:, None]]
    return (int(lens.min()), int(lens.max())) + ((int(ids.min()), int(ids.max())) if ids.numel() else (0, -1))


def free_sequences(cache: PagedKVCache, rows: torch.Tensor, *, held: torch.Tensor | None = None,
                   validate: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """Empty the rows ``rows`` and list the pool's pages that no row uses.

    Sets ``seq_lens`` (and ``held``) of the rows to 0, in place.  Returns
    ``(pages, count)``, on the device: the ids of all unused pages of the pool,
    ascending, in ``pages[:count]`` (int32 ``[num_pages]``, -1 behind), and
    their number (0-d int32).  A page that another row still uses isn't among
    them.  A row may be in ``rows`` twice; with none it lists the unused pages.
    """
    _check_layout(cache)
    rows = _ids(cache, "rows", rows)
    held = _held(cache, held, written=True)
    dev = cache.k_cache.device
    if not cache.k_cache.is_cuda or not cache.page_table.numel() or not cache.num_pages:
        _require(not _outside(rows, cache.batch_size), f"rows holds a row outside [0, {cache.batch_size})")
        _assess_used(cache, held, _used_stats(cache, held), _beyond(cache, held))
        cache.seq_lens[rows.long()] = 0
        if held is not None:
            held[rows.long()] = 0
        free = (~_used_torch(cache, held)[1]).nonzero()[:, 0].to(torch.int32)
        pages = torch.full((cache.num_pages,), -1, dtype=torch.int32, device=dev)
        pages[:free.shape[0]] = free
        return pages, torch.tensor(free.shape[0], dtype=torch.int32, device=dev)

    from . import _hip

    _check_rocm(cache)
    with _hip.on_device(dev):
        stream = _hip.current_stream_handle(dev)
        check = None
        if validate:
            check = _hip.check_begin(_hip.CHECK_FREE, stream, dev, seq_lens=cache.seq_lens,
                                     page_table=cache.page_table, page_size=cache.page_size, ids=(rows,),
                                     held=held)
        # prepared while the check kernel runs
        pages = torch.empty(cache.num_pages, dtype=torch.int32, device=dev)
        count = torch.empty((), dtype=torch.int32, device=dev)
        workspace = _hip.pages_workspace(cache.num_pages, dev)
        args = _hip.free_args(cache, rows, held, pages, count, workspace)
        if check is not None:
            r = check.wait()
            _assess_used(cache, held, _stats_of(r), bool(r[7] & 2))
            _require(not r[7] & 1, f"rows holds a row outside [0, {cache.batch_size})")
        _hip.page_operation("fat_free_sequences", args, stream)
    return pages, count


def _stats_of(r: list[int]) -> tuple[int, int, int, int]:
    """A check's results as :func:`~flashattntile_amd.paging.cache_stats` gives them."""
    none = r[12] == 2 ** 31 - 1  # of no used column
    return r[0], r[1], 0 if none else r[12], -1 if none else r[13]


def compact_pages(cache: PagedKVCache, *, held: torch.Tensor | None = None, quantized=None, scales=None,
                  validate: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the n pages that rows use to the pool's front, ids 0 to n - 1.

    Used pages with an id below n stay; the others, in ascending order, go to the
    unused ids below n, in ascending order; shared pages move once.  Moves K and
    V (and the 8-bit copy and scales where given) and renumbers the used columns
    of ``page_table``, in place.  Returns ``(remap, count)``, on the device:
    ``remap[id]`` is a page's new id, -1 where no row used it (int32
    ``[num_pages]``, for tables an engine keeps elsewhere), and ``count`` is n
    (0-d int32).  Pages from n on then belong to nobody and keep their bytes, so
    the pool can be cut there, copied out or given back.

    Columns that a row doesn't use keep their entries, which then name pages of
    others or of nobody: pass ``held`` where rows hold pages ahead of their
    tokens, as those of :func:`~flashattntile_amd.paging.allocate` do.
    """
    copy, scales = _parts(cache, quantized, scales, shared_table=True)
    held = _held(cache, held, written=False)
    dev = cache.k_cache.device
    if not cache.k_cache.is_cuda or not cache.page_table.numel() or not cache.num_pages:
        _assess_used(cache, held, _used_stats(cache, held), _beyond(cache, held))
        columns, used = _used_torch(cache, held)
        n = int(used.sum())
        ids = torch.arange(cache.num_pages, device=dev)
        src = (used & (ids >= n)).nonzero()[:, 0]
        dst = (~used & (ids < n)).nonzero()[:, 0]
        remap = torch.where(used, ids, torch.full_like(ids, -1)).to(torch.int32)
        remap[src] = dst.to(torch.int32)
        for t in _planes(cache, copy, scales):
            t[dst] = t[src]
        cache.page_table[columns] = remap[cache.page_table[columns].long()]
        return remap, torch.tensor(n, dtype=torch.int32, device=dev)

    from . import _hip

    _check_rocm(cache)
    with _hip.on_device(dev):
        stream = _hip.current_stream_handle(dev)
        check = None
        if validate:
            check = _hip.check_begin(_hip.CHECK_FREE, stream, dev, seq_lens=cache.seq_lens,
                                     page_table=cache.page_table, page_size=cache.page_size, held=held)
        # prepared while the check kernel runs
        remap = torch.empty(cache.num_pages, dtype=torch.int32, device=dev)
        count = torch.empty((), dtype=torch.int32, device=dev)
        workspace = _hip.pages_workspace(cache.num_pages, dev)
        args = _hip.compact_args(cache, held, remap, count, workspace, copy, scales)
        if check is not None:
            r = check.wait()
            _assess_used(cache, held, _stats_of(r), bool(r[7] & 2))
        _hip.page_operation("fat_compact_pages", args, stream)
    return remap, count
