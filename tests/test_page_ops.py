"""copy_pages, fork_sequences, free_sequences and compact_pages, on the CPU
(torch) and on the GPU (``csrc/pages.hip``), against plain Python over dicts of
pages.  Everything is bits and whole numbers, so every comparison is exact, of
the whole pool: pages that an operation doesn't name have to stay as they were.
"""

from __future__ import annotations

import math

import pytest
import torch

import flashattntile_amd as fat
from flashattntile_amd import (PagedKVCache, allocate, append_tokens, compact_pages, copy_pages, fork_sequences,
                               free_sequences, gather_contiguous, quantize_cache)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
device = pytest.mark.parametrize("dev", DEVICES)


def _ids(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _pool(pages, P, hkv, d, dtype, dev, layout="dense", seed=0):
    """Random bits of ``dtype`` as pages, in one of the layouts an engine may have."""
    g = torch.Generator().manual_seed(seed)

    def one():
        shape = {"dense": (pages, P, hkv, d), "heads_first": (pages, hkv, P, d), "padded": (pages, P, hkv + 1, d + 8),
                 "joint": (2, pages, P, hkv, d)}[layout]
        bits = torch.randint(-100, 100, shape, generator=g, dtype=torch.int32).to(torch.int8)
        t = bits.view(dtype) if dtype == torch.float8_e4m3fn else bits.to(dtype)
        t = t.to(dev)
        if layout == "heads_first":
            return t.transpose(1, 2)
        if layout == "padded":
            return t[:, :, :hkv, 3:3 + d] if d % 2 else t[:, :, :hkv, :d]
        return t

    if layout == "joint":  # K and V in one tensor, as the backend's cache shape has them
        t = one()
        return t[0], t[1]
    return one(), one()


def _cache(lens, P, hkv=2, d=16, dtype=torch.float16, dev="cpu", layout="dense", spare=5, width=None, seed=0,
           shared=0):
    """Scattered pages; the first ``shared`` columns name the same pages in all rows that are long enough."""
    g = torch.Generator().manual_seed(seed + 1)
    per = [math.ceil(n / P) for n in lens]
    pool = sum(per) + spare + shared
    perm = torch.randperm(pool, generator=g).tolist()
    common = [perm.pop() for _ in range(shared)]
    table = torch.full((len(lens), width or max(per + [1])), 0, dtype=torch.int32)
    for b, n in enumerate(per):
        for c in range(n):
            table[b, c] = common[c] if c < shared else perm.pop()
    k, v = _pool(pool, P, hkv, d, dtype, dev, layout, seed)
    return PagedKVCache(k, v, table.to(dev), _ids(lens, dev), P)


def _scales(pages, hkv, dev, seed=3):
    g = torch.Generator().manual_seed(seed)
    return {"k": torch.rand(pages, hkv, generator=g).to(dev), "v": torch.rand(pages, hkv, generator=g).to(dev)}


def _bits(t):
    t = t.detach().contiguous().cpu()
    return t.view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()]).clone()


def _planes(cache, quantized=None, scales=None):
    out = [cache.k_cache, cache.v_cache]
    if quantized is not None:
        q, scales = quantized
        out += [q.k_cache, q.v_cache]
    if scales is not None:
        out += [scales["k"], scales["v"]]
    return out


def _snapshot(cache, quantized=None, scales=None):
    return [_bits(t) for t in _planes(cache, quantized, scales)]


def _moved(before, moves):
    """The pool after page src of every (src, dst) was copied to page dst."""
    after = [t.clone() for t in before]
    for src, dst in moves:
        for a, b in zip(after, before):
            a[dst] = b[src]
    return after


def _same(got, want):
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def _mirror(cache, seed=9):
    """An 8-bit copy under the cache's own table and lengths."""
    k, v = _pool(cache.num_pages, cache.page_size, cache.num_kv_heads, cache.head_dim, torch.int8,
                 cache.k_cache.device, seed=seed)
    return (PagedKVCache(k, v, cache.page_table, cache.seq_lens, cache.page_size),
            _scales(cache.num_pages, cache.num_kv_heads, cache.k_cache.device))


def _parts(kind, pages, P, hkv, d, dev, layout="dense"):
    """A cache of a kind, its ``quantized`` and its ``scales``."""
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "mirror": torch.bfloat16,
             "int8": torch.int8, "fp8": torch.float8_e4m3fn}[kind]
    k, v = _pool(pages, P, hkv, d, dtype, dev, layout)
    cache = PagedKVCache(k, v, torch.zeros(1, 1, dtype=torch.int32, device=dev), _ids([0], dev), P)
    return (cache, _mirror(cache) if kind == "mirror" else None,
            _scales(pages, hkv, dev) if kind in ("int8", "fp8") else None)


# ---------------------------------------------------------------------------
# copy
# ---------------------------------------------------------------------------
@device
@pytest.mark.parametrize("kind", ["fp16", "bf16", "fp32", "mirror", "int8", "fp8"])
@pytest.mark.parametrize("P,hkv,d", [(16, 8, 128), (1, 1, 16), (7, 3, 20), (64, 2, 512), (1, 4, 7)])
def test_copy_pages_moves_every_plane(dev, kind, P, hkv, d):
    print(f"copy {dev} {kind} P{P} hkv{hkv} d{d}", flush=True)
    cache, quantized, scales = _parts(kind, 40, P, hkv, d, dev)
    g = torch.Generator().manual_seed(P)
    perm = torch.randperm(40, generator=g).tolist()
    src, dst = perm[:13] + perm[:4], perm[20:37]  # a source more than once
    before = _snapshot(cache, quantized, scales)
    copy_pages(cache, _ids(src, dev), _ids(dst, dev), quantized=quantized, scales=scales)
    _same(_snapshot(cache, quantized, scales), _moved(before, zip(src, dst)))


@device
@pytest.mark.parametrize("layout", ["heads_first", "padded", "joint"])
@pytest.mark.parametrize("kind,P,hkv,d", [("fp16", 16, 2, 64), ("fp32", 5, 3, 33), ("int8", 16, 4, 31), ("fp8", 1, 2, 64)])
def test_copy_pages_in_other_layouts(dev, layout, kind, P, hkv, d):
    print(f"copy {dev} {layout} {kind}", flush=True)
    cache, _, scales = _parts(kind, 12, P, hkv, d, dev, layout)
    if scales is not None:  # scales stored head by head
        scales = {n: t.t().contiguous().t() for n, t in scales.items()}
    before = _snapshot(cache, None, scales)
    copy_pages(cache, _ids([3, 0, 11], dev), _ids([1, 2, 5], dev), scales=scales)
    _same(_snapshot(cache, None, scales), _moved(before, [(3, 1), (0, 2), (11, 5)]))


@pytest.mark.gpu
def test_copy_pages_padding_between_rows_stays():
    """Bytes between the rows of a padded layout belong to somebody else."""
    whole = torch.arange(6 * 4 * 3 * 24, dtype=torch.float32, device="cuda").view(6, 4, 3, 24)
    other = whole.clone()
    cache = PagedKVCache(whole[:, :, :2, 4:20], other[:, :, :2, 4:20], _ids([[0]], "cuda"), _ids([0], "cuda"), 4)
    want = whole.clone()
    want[2, :, :2, 4:20] = whole[5, :, :2, 4:20]
    copy_pages(cache, _ids([5], "cuda"), _ids([2], "cuda"))
    assert torch.equal(whole, want) and torch.equal(other, want)


@device
def test_copy_pages_of_none(dev):
    cache, _, _ = _parts("fp16", 4, 16, 1, 16, dev)
    before = _snapshot(cache)
    copy_pages(cache, _ids([], dev), _ids([], dev))
    _same(_snapshot(cache), before)


@pytest.mark.gpu
def test_copy_pages_of_many_pairs_and_a_strided_list():
    print("copy of many", flush=True)
    cache, _, _ = _parts("fp16", 30000, 2, 1, 32, "cuda")
    perm = torch.randperm(30000, generator=torch.Generator().manual_seed(5)).to(torch.int32)
    before = _snapshot(cache)
    both = perm.view(-1, 2).cuda()  # columns of one tensor: stride 2
    copy_pages(cache, both[:, 0], both[:, 1])
    want = [t.clone() for t in before]
    for w, b in zip(want, before):
        w[perm.view(-1, 2)[:, 1].long()] = b[perm.view(-1, 2)[:, 0].long()]
    _same(_snapshot(cache), want)


@pytest.mark.gpu
def test_copy_pages_behind_4_gib():
    """Byte offsets past 32 bits on both sides."""
    print("copy behind 4 GiB", flush=True)
    pages = 2500
    k = torch.zeros(pages, 1024, 8, 128, dtype=torch.float16, device="cuda")  # 2 MiB a page, 4.9 GiB
    k[pages - 1] = 3.0
    k[1] = 5.0
    cache = PagedKVCache(k, k, _ids([[0]], "cuda"), _ids([0], "cuda"), 1024)
    copy_pages(cache, _ids([pages - 1, 1], "cuda"), _ids([0, pages - 2], "cuda"))
    assert bool((k[0] == 3.0).all()) and bool((k[pages - 2] == 5.0).all())
    assert not bool(k[2:pages - 2].any())


@device
@pytest.mark.parametrize("src,dst,error", [([0, 4], [1, 2], "src holds a page outside"),
                                           ([-1, 0], [1, 2], "src holds a page outside"),
                                           ([0, 3], [1, 4], "dst holds a page outside"),
                                           ([0, 3], [1, 1], "dst holds a page twice"),
                                           ([0, 3], [1, 0], "dst holds a page that src holds too"),
                                           ([2, 3], [2, 1], "dst holds a page that src holds too")])
def test_copy_pages_refusals(dev, src, dst, error):
    cache, _, _ = _parts("fp16", 4, 16, 1, 16, dev)
    before = _snapshot(cache)
    with pytest.raises(AssertionError, match=error):
        copy_pages(cache, _ids(src, dev), _ids(dst, dev))
    _same(_snapshot(cache), before)


@device
def test_argument_refusals(dev):
    cache, _, _ = _parts("fp16", 4, 16, 2, 16, dev)
    one = _ids([0], dev)
    for bad in (one.long(), one.view(1, 1), [0]):
        with pytest.raises(AssertionError, match="src must be a 1-D int32"):
            copy_pages(cache, bad, one)
    with pytest.raises(AssertionError, match="dst must have 1 entries"):
        copy_pages(cache, one, _ids([1, 2], dev))
    with pytest.raises(AssertionError, match="only such a cache takes them"):
        copy_pages(cache, one, one, scales=_scales(4, 2, dev))
    small, _, scales = _parts("int8", 4, 16, 2, 16, dev)
    with pytest.raises(AssertionError, match="needs scales"):
        compact_pages(small)
    with pytest.raises(AssertionError, match="scales must be \\[4, 2\\]"):
        copy_pages(small, one, one, scales=_scales(3, 2, dev))
    with pytest.raises(AssertionError, match="float32"):
        copy_pages(small, one, one, scales={n: t.half() for n, t in scales.items()})
    with pytest.raises(AssertionError, match="no 8-bit copy"):
        copy_pages(small, one, one, quantized=(small, scales))
    apart = PagedKVCache(small.k_cache, small.v_cache, small.page_table.clone(), small.seq_lens, 16)
    with pytest.raises(AssertionError, match="share the cache's page_table"):
        compact_pages(cache, quantized=(apart, scales))
    with pytest.raises(AssertionError, match="held must be int32"):
        compact_pages(cache, held=_ids([1, 2], dev))
    with pytest.raises(AssertionError, match="parents must be"):
        fork_sequences(cache, one.float(), one, one)


# ---------------------------------------------------------------------------
# fork
# ---------------------------------------------------------------------------
def _fork_ref(cache, parents, children, pages, before, table, lens):
    """Table, lengths and pool after the forks, in plain Python."""
    P, moves = cache.page_size, []
    table, lens = [list(r) for r in table], list(lens)
    for p, c, fresh in zip(parents, children, pages):
        n = lens[p]
        used = math.ceil(n / P)
        table[c][:used] = table[p][:used]
        if n % P:
            moves.append((table[p][used - 1], fresh))
            table[c][used - 1] = fresh
        lens[c] = n
    return table, lens, _moved(before, moves)


@device
@pytest.mark.parametrize("P", [1, 16, 12])
@pytest.mark.parametrize("kind", ["fp16", "mirror", "fp8"])
def test_fork_shares_whole_pages_and_copies_the_last(dev, P, kind):
    print(f"fork {dev} P{P} {kind}", flush=True)
    lens = [0, 5 * P, 3 * P + max(1, P // 2), 1, 0, 0, 0, 0, 0, 0, 0]
    dtype = {"fp16": torch.float16, "mirror": torch.bfloat16, "fp8": torch.float8_e4m3fn}[kind]
    cache = _cache(lens, P, hkv=3, d=32, dtype=dtype, dev=dev, spare=20, width=9)
    quantized = _mirror(cache) if kind == "mirror" else None
    scales = _scales(cache.num_pages, 3, dev) if kind == "fp8" else None
    cache.page_table[4:] = 77  # what columns behind a row's last page hold stays
    used = {int(x) for b, n in enumerate(lens) for x in cache.page_table[b, :math.ceil(n / P)]}
    fresh = [i for i in range(cache.num_pages) if i not in used]
    parents, children = [1, 2, 2, 3, 0, 2], [10, 4, 9, 5, 6, 8]
    pages = fresh[:6]
    before = _snapshot(cache, quantized, scales)
    table, lens2, pool = _fork_ref(cache, parents, children, pages, before, cache.page_table.tolist(), lens)
    fork_sequences(cache, _ids(parents, dev), _ids(children, dev), _ids(pages, dev), quantized=quantized,
                   scales=scales)
    assert cache.page_table.tolist() == table
    assert cache.seq_lens.tolist() == lens2
    _same(_snapshot(cache, quantized, scales), pool)


@pytest.mark.gpu
def test_fork_of_long_sequences_and_strided_tables():
    print("fork long", flush=True)
    lens = [8000, 4097, 1] + [0] * 60
    cache = _cache(lens, 1, hkv=1, d=16, dev="cuda", spare=70)
    wide = torch.full((63, 9000), -5, dtype=torch.int32, device="cuda")
    wide[:, 100:8100] = cache.page_table
    cache = PagedKVCache(cache.k_cache, cache.v_cache, wide[:, 100:8100], cache.seq_lens, 1)
    parents = [i % 3 for i in range(60)]
    children = list(range(3, 63))
    fork_sequences(cache, _ids(parents, "cuda"), _ids(children, "cuda"), _ids(list(range(60)), "cuda"))
    for i, p in enumerate(parents):
        assert torch.equal(cache.page_table[3 + i, :lens[p]], cache.page_table[p, :lens[p]])
        assert int(cache.page_table[3 + i, lens[p]:].abs().sum()) == 0  # behind: as it was
    assert cache.seq_lens.tolist() == lens[:3] + [lens[p] for p in parents]
    assert bool((wide[:, :100] == -5).all()) and bool((wide[:, 8100:] == -5).all())


@device
@pytest.mark.parametrize("parents,children,pages,error", [
    ([0], [9], [20], "children holds a row outside"),
    ([4], [2], [20], "parents holds a row outside"),
    ([-1], [2], [20], "parents holds a row outside"),
    ([0, 1], [2, 2], [20, 21], "children holds a row twice"),
    ([0, 2], [2, 3], [20, 21], "both parent and child"),
    ([0], [1], [20], "children must be empty"),
    ([0], [2], [99], "pages holds a page outside"),
    ([0, 0], [2, 3], [20, 20], "pages holds a page twice"),
])
def test_fork_refusals(dev, parents, children, pages, error):
    cache = _cache([21, 16, 0, 0], 16, dev=dev, spare=30)
    before = _snapshot(cache), cache.page_table.tolist(), cache.seq_lens.tolist()
    with pytest.raises(AssertionError, match=error):
        fork_sequences(cache, _ids(parents, dev), _ids(children, dev), _ids(pages, dev))
    _same(_snapshot(cache), before[0])
    assert (cache.page_table.tolist(), cache.seq_lens.tolist()) == before[1:]


@device
def test_fork_refuses_bad_parents(dev):
    for spoil, error in ((lambda c: c.seq_lens.__setitem__(0, 1000), "exceeds page-table capacity"),
                         (lambda c: c.seq_lens.__setitem__(0, -3), "negative"),
                         (lambda c: c.page_table[0].__setitem__(1, 500), "last page outside")):
        cache = _cache([21, 16, 0, 0], 16, dev=dev, spare=30)
        spoil(cache)
        before = _snapshot(cache), cache.page_table.tolist(), cache.seq_lens.tolist()
        with pytest.raises(AssertionError, match=error):
            fork_sequences(cache, _ids([0], dev), _ids([2], dev), _ids([20], dev))
        _same(_snapshot(cache), before[0])
        assert (cache.page_table.tolist(), cache.seq_lens.tolist()) == before[1:]


@pytest.mark.gpu
def test_fork_unused_page_ids_are_not_looked_at():
    """pages[i] of a parent that fills its last page may be anything, twice too."""
    cache = _cache([32, 48, 0, 0], 16, dev="cuda", width=3)
    fork_sequences(cache, _ids([0, 1], "cuda"), _ids([2, 3], "cuda"), _ids([-1, -1], "cuda"))
    assert cache.seq_lens.tolist() == [32, 48, 32, 48]
    assert torch.equal(cache.page_table[3], cache.page_table[1])


@pytest.mark.gpu
def test_without_validation_bad_entries_are_skipped_whole():
    print("unvalidated", flush=True)
    cache = _cache([21, 16, 0, 0, 0, 0, 0], 16, dev="cuda", spare=30)
    cache.seq_lens[1] = 9999
    before = _snapshot(cache)
    table, lens = cache.page_table.tolist(), cache.seq_lens.tolist()
    fork_sequences(cache, _ids([0, 50, 1, 0, -2], "cuda"), _ids([70, 2, 3, 4, 5], "cuda"),
                   _ids([20, 21, 22, 1 << 30, 23], "cuda"), validate=False)
    assert cache.page_table.tolist() == table and cache.seq_lens.tolist() == lens
    copy_pages(cache, _ids([0, -1, 1 << 20], "cuda"), _ids([1 << 20, 1, 2], "cuda"), validate=False)
    _same(_snapshot(cache), before)
    cache.seq_lens[1] = 16
    cache.page_table[1, 0] = 1 << 30  # used, and no page
    pages, count = free_sequences(cache, _ids([-1, 7, 1 << 30], "cuda"), validate=False)
    assert int(count) == cache.num_pages - 2 and cache.seq_lens.tolist()[:2] == [21, 16]
    compact_pages(cache, validate=False)
    assert int(cache.page_table[1, 0]) == 1 << 30


# ---------------------------------------------------------------------------
# free and compact
# ---------------------------------------------------------------------------
def _used(table, lens, P, pages, held=None):
    out = set()
    for b, n in enumerate(lens):
        cols = max(math.ceil(max(n, 0) / P), held[b] if held else 0)
        out |= {x for x in table[b][:cols] if 0 <= x < pages}
    return out


SIZES = [([0], 16, 3), ([1], 1, 0), ([5, 0, 33, 16], 16, 4), ([700, 1, 300, 0, 650], 1, 900),
         ([13, 77, 1, 40], 7, 2), ([64 * i for i in range(40)], 16, 5000)]


@device
@pytest.mark.parametrize("lens,P,spare", SIZES)
@pytest.mark.parametrize("shared", [0, 2])
def test_free_lists_what_no_row_uses(dev, lens, P, spare, shared):
    print(f"free {dev} P{P} rows{len(lens)} shared{shared}", flush=True)
    cache = _cache(lens, P, hkv=1, d=16, dev=dev, spare=spare, shared=shared)
    if not cache.num_pages:
        pytest.skip("an empty pool")
    rows = [b for b in range(len(lens)) if b % 3 == 2] * 2  # every row twice
    want_lens = [0 if b in rows else n for b, n in enumerate(lens)]
    used = _used(cache.page_table.tolist(), want_lens, P, cache.num_pages)
    free = [i for i in range(cache.num_pages) if i not in used]
    before, table = _snapshot(cache), cache.page_table.tolist()
    pages, count = free_sequences(cache, _ids(rows, dev))
    assert pages.dtype == torch.int32 and count.shape == () and count.dtype == torch.int32
    assert cache.seq_lens.tolist() == want_lens and cache.page_table.tolist() == table
    assert int(count) == len(free)
    assert pages.tolist() == free + [-1] * len(used)
    _same(_snapshot(cache), before)


@device
def test_free_with_pages_held_ahead(dev):
    cache = _cache([20, 40, 0, 1], 16, dev=dev, spare=8, width=5)
    cache.page_table[:, 3:] = torch.arange(8, dtype=torch.int32, device=dev).view(4, 2)  # held in rows 0 and 2
    held = _ids([5, 0, 5, -3], dev)
    pages, count = free_sequences(cache, _ids([0], dev), held=held)
    assert held.tolist() == [0, 0, 5, -3] and cache.seq_lens.tolist() == [0, 40, 0, 1]
    used = _used(cache.page_table.tolist(), [0, 40, 0, 1], 16, cache.num_pages, held.tolist())
    assert pages.tolist()[:int(count)] == [i for i in range(cache.num_pages) if i not in used]


@device
@pytest.mark.parametrize("rows", [[4], [-1], [0, 99]])
def test_free_refusals(dev, rows):
    cache = _cache([20, 40, 0, 1], 16, dev=dev)
    with pytest.raises(AssertionError, match="rows holds a row outside"):
        free_sequences(cache, _ids(rows, dev))
    assert cache.seq_lens.tolist() == [20, 40, 0, 1]
    cache.page_table[1, 0] = 1000
    for call in (lambda: free_sequences(cache, _ids([0], dev)), lambda: compact_pages(cache)):
        with pytest.raises(AssertionError, match="references page 1000"):
            call()
    assert cache.seq_lens.tolist() == [20, 40, 0, 1]


def _compact_ref(cache, lens, table, before, held=None):
    P, N = cache.page_size, cache.num_pages
    used = _used(table, lens, P, N, held)
    n = len(used)
    moves = list(zip(sorted(i for i in used if i >= n), sorted(i for i in range(n) if i not in used)))
    remap = [i if i in used else -1 for i in range(N)]
    for a, b in moves:
        remap[a] = b
    out = [list(r) for r in table]
    for b, length in enumerate(lens):
        cols = max(math.ceil(max(length, 0) / P), held[b] if held else 0)
        for c in range(min(cols, len(out[b]))):
            if 0 <= out[b][c] < N:
                out[b][c] = remap[out[b][c]]
    return n, remap, out, _moved(before, moves)


@device
@pytest.mark.parametrize("lens,P,spare", SIZES)
@pytest.mark.parametrize("kind,shared", [("fp16", 0), ("mirror", 2), ("int8", 1)])
def test_compact_moves_used_pages_to_the_front(dev, lens, P, spare, kind, shared):
    print(f"compact {dev} P{P} rows{len(lens)} {kind} shared{shared}", flush=True)
    dtype = {"fp16": torch.float16, "mirror": torch.bfloat16, "int8": torch.int8}[kind]
    cache = _cache(lens, P, hkv=2, d=16, dtype=dtype, dev=dev, spare=spare, shared=shared, width=None)
    quantized = _mirror(cache) if kind == "mirror" else None
    scales = _scales(cache.num_pages, 2, dev) if kind == "int8" else None
    before = _snapshot(cache, quantized, scales)
    n, want_remap, want_table, pool = _compact_ref(cache, lens, cache.page_table.tolist(), before)
    remap, count = compact_pages(cache, quantized=quantized, scales=scales)
    assert int(count) == n and count.shape == () and count.dtype == torch.int32
    assert remap.tolist() == want_remap and remap.dtype == torch.int32
    assert cache.page_table.tolist() == want_table
    assert cache.seq_lens.tolist() == lens
    _same(_snapshot(cache, quantized, scales), pool)


@device
def test_compact_with_pages_held_ahead(dev):
    """An allocate()d cache, half of it: its reserved pages move with it."""
    cache = allocate(6, 64, 2, 16, 16, device=dev)
    cache.page_table[0:3].copy_(cache.page_table[3:6].clone())  # rows 0-2 hold the pool's end
    cache.seq_lens[:2] = _ids([40, 5], dev)
    held = _ids([4, 4, 4, 0, 0, 0], dev)
    table = cache.page_table.tolist()
    before = _snapshot(cache)
    n, want_remap, want_table, pool = _compact_ref(cache, cache.seq_lens.tolist(), table, before, held.tolist())
    remap, count = compact_pages(cache, held=held)
    assert int(count) == n == 12 and remap.tolist() == want_remap and cache.page_table.tolist() == want_table
    assert held.tolist() == [4, 4, 4, 0, 0, 0]
    _same(_snapshot(cache), pool)


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [1, 4095, 4096, 4097, 40961])
@pytest.mark.parametrize("fill", ["none", "one", "half", "all", "front", "back"])
def test_compact_and_free_at_group_borders(pages, fill):
    """Pools of whole and broken groups of 4096 pages, and used pages lying at their ends."""
    print(f"borders {pages} {fill}", flush=True)
    g = torch.Generator().manual_seed(pages)
    ids = {"none": [], "one": [pages - 1], "half": torch.randperm(pages, generator=g)[:pages // 2].tolist(),
           "all": list(range(pages)), "front": list(range(pages // 3)),
           "back": list(range(pages - pages // 3, pages))}[fill]
    table = torch.zeros(1, max(1, pages), dtype=torch.int32)
    table[0, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
    k = torch.randint(-2 ** 15, 2 ** 15 - 1, (pages, 1, 1, 2), generator=g, dtype=torch.int32).to(torch.float32)
    cache = PagedKVCache(k.cuda(), -k.cuda(), table.cuda(), _ids([len(ids)], "cuda"), 1)
    free, count = free_sequences(cache, _ids([], "cuda"))
    left = sorted(set(range(pages)) - set(ids))
    assert int(count) == len(left) and free.tolist() == left + [-1] * len(ids)
    rows = k[table[0, :len(ids)].long(), 0, 0].tolist()
    remap, count = compact_pages(cache)
    n = len(ids)
    assert int(count) == n
    assert sorted(cache.page_table[0, :n].tolist()) == list(range(n))
    assert cache.k_cache[cache.page_table[0, :n].long(), 0, 0].tolist() == rows
    assert cache.v_cache[cache.page_table[0, :n].long(), 0, 0].neg().tolist() == rows
    got = remap.cpu()
    assert torch.equal(got[torch.tensor(ids, dtype=torch.long)], cache.page_table[0, :n].cpu())
    assert int((got >= 0).sum()) == n


@device
def test_empty_batches_and_tables(dev):
    k = torch.ones(5, 4, 1, 16, device=dev)
    for shape in ((0, 3), (2, 0)):
        cache = PagedKVCache(k, k.clone(), torch.zeros(shape, dtype=torch.int32, device=dev),
                             torch.zeros(shape[0], dtype=torch.int32, device=dev), 4)
        pages, count = free_sequences(cache, _ids([], dev))
        assert pages.tolist() == [0, 1, 2, 3, 4] and int(count) == 5
        remap, count = compact_pages(cache)
        assert remap.tolist() == [-1] * 5 and int(count) == 0


# ---------------------------------------------------------------------------
# Together, and as an engine runs them
# ---------------------------------------------------------------------------
@device
@pytest.mark.parametrize("mode", [None, "int8"])
def test_a_run_of_all_of_them_keeps_every_sequence(dev, mode):
    """Prompts, forks, appends that grow into free pages, ends, compaction, and a
    pool cut at its new end: every row holds the tokens a row of its own would."""
    print(f"run of all {dev} {mode}", flush=True)
    P, hkv, d = 4, 2, 16
    pages, rows = 60, 6
    g = torch.Generator().manual_seed(1)
    cache = PagedKVCache(torch.zeros(pages, P, hkv, d, dtype=torch.float16, device=dev),
                         torch.zeros(pages, P, hkv, d, dtype=torch.float16, device=dev),
                         torch.zeros(rows, 9, dtype=torch.int32, device=dev), _ids([0] * rows, dev), P)
    quantized = quantize_cache(cache, mode=mode) if mode else None
    free = list(range(pages - 1, -1, -1))  # the engine's own list
    tokens = [[] for _ in range(rows)]

    def step(live):
        """One token for every row of ``live``; the others' write is dropped."""
        nonlocal cache
        lens = cache.seq_lens.tolist()
        for b in live:
            if lens[b] % P == 0:
                cache.page_table[b, lens[b] // P] = free.pop()
        new = torch.randn(rows, hkv, d, generator=g).half()
        sub = PagedKVCache(cache.k_cache, cache.v_cache, cache.page_table[live].contiguous(),
                           cache.seq_lens[live].contiguous(), P)
        pair = None
        if quantized:
            pair = (PagedKVCache(quantized[0].k_cache, quantized[0].v_cache, sub.page_table, sub.seq_lens, P),
                    {"k": quantized[1].k, "v": quantized[1].v})
        append_tokens(sub, new[live].to(dev), (-new[live]).to(dev), quantized=pair)
        cache.seq_lens[live] = sub.seq_lens
        for b in live:
            tokens[b].append(new[b])

    def check():
        k, v = gather_contiguous(cache)
        for b in range(rows):
            want = torch.stack(tokens[b]) if tokens[b] else torch.zeros(0, hkv, d).half()
            assert torch.equal(k[b, :len(tokens[b])].cpu(), want), b
            assert torch.equal(v[b, :len(tokens[b])].cpu(), -want), b
        if quantized:
            fresh, scales = quantize_cache(cache, mode=mode)
            ids = sorted(_used(cache.page_table.tolist(), cache.seq_lens.tolist(), P, cache.num_pages))
            for a, b in ((quantized[0].k_cache, fresh.k_cache), (quantized[0].v_cache, fresh.v_cache),
                         (quantized[1].k, scales.k), (quantized[1].v, scales.v)):
                assert torch.equal(_bits(a)[ids], _bits(b)[ids])

    for _ in range(10):
        step([0, 1])
    step([1])
    take = [free.pop() for _ in range(3)]
    fork_sequences(cache, _ids([0, 0, 1], dev), _ids([2, 3, 4], dev), _ids(take, dev), quantized=quantized)
    for p, c in ((0, 2), (0, 3), (1, 4)):
        tokens[c] = list(tokens[p])
    check()
    for _ in range(7):
        step([0, 1, 2, 4])
    check()
    pages_left, count = free_sequences(cache, _ids([0, 4], dev))
    tokens[0], tokens[4] = [], []
    free = pages_left[:int(count)].tolist()[::-1]
    check()
    remap, count = compact_pages(cache, quantized=quantized)
    n = int(count)
    used = _used(cache.page_table.tolist(), cache.seq_lens.tolist(), P, cache.num_pages)
    assert used == set(range(n)) and n < pages
    check()
    # the pool's end is given back
    cache = PagedKVCache(cache.k_cache[:n + 8].clone(), cache.v_cache[:n + 8].clone(), cache.page_table,
                         cache.seq_lens, P)
    if quantized:
        q, s = quantized
        quantized = (PagedKVCache(q.k_cache[:n + 8].clone(), q.v_cache[:n + 8].clone(), cache.page_table,
                                  cache.seq_lens, P),
                     fat.QuantScales(k=s.k[:n + 8].clone(), v=s.v[:n + 8].clone(), mode=s.mode))
    free = list(range(n + 7, n - 1, -1))
    for _ in range(5):
        step([1, 2, 3])
    check()


@pytest.mark.gpu
def test_captured_and_replayed_with_eager_work_between():
    """fork, free and compact without validation in one graph; every replay
    starts from other lengths and matches the eager calls."""
    print("capture", flush=True)
    P = 4
    lens = [9, 22, 4, 0, 0, 13]
    cache = _cache(lens, P, dev="cuda", spare=12, width=8)
    twin = _cache(lens, P, dev="cuda", spare=12, width=8)
    start = cache.page_table.clone(), cache.k_cache.clone(), cache.v_cache.clone()
    parents, children, rows = _ids([1, 0], "cuda"), _ids([3, 4], "cuda"), _ids([5], "cuda")

    def work(c, fresh, out):
        fork_sequences(c, parents, children, fresh, validate=False)
        pages, count = free_sequences(c, rows, validate=False)
        remap, used = compact_pages(c, validate=False)
        for o, t in zip(out, (pages, count, remap, used)):
            o.copy_(t)

    fresh = _ids([0, 0], "cuda")
    outs = [[torch.zeros(n, dtype=torch.int32, device="cuda") for n in (cache.num_pages, 1, cache.num_pages, 1)]
            for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            work(cache, fresh, outs[0])
    torch.cuda.current_stream().wait_stream(side)
    for seed, now in enumerate([[9, 22, 4, 0, 0, 13], [1, 3, 4, 0, 0, 0], [12, 8, 4, 0, 0, 32], [9, 22, 4, 0, 0, 13]]):
        width = max(math.ceil(n / P) for n in now)
        for c in (cache, twin):
            c.page_table.copy_(start[0])
            c.page_table[5] = torch.arange(c.num_pages - 8, c.num_pages, dtype=torch.int32, device="cuda")
            c.k_cache.copy_(start[1])
            c.v_cache.copy_(start[2])
            c.seq_lens.copy_(_ids(now, "cuda"))
        assert width <= 8
        used = _used(cache.page_table.tolist(), now, P, cache.num_pages)
        fresh.copy_(_ids([i for i in range(cache.num_pages) if i not in used][:2], "cuda"))
        graph.replay()
        work(twin, fresh, outs[1])
        torch.cuda.synchronize()
        for a, b in zip(outs[0], outs[1]):
            assert torch.equal(a, b), seed
        _same(_snapshot(cache), _snapshot(twin))
        assert torch.equal(cache.page_table, twin.page_table) and torch.equal(cache.seq_lens, twin.seq_lens)


@pytest.mark.gpu
def test_on_streams_of_their_own():
    print("streams", flush=True)
    lens = [64 * i + 3 for i in range(20)]
    caches = [_cache(lens, 16, dev="cuda", spare=40, seed=s) for s in range(4)]
    want = [_compact_ref(c, lens, c.page_table.tolist(), _snapshot(c)) for c in caches]
    streams = [torch.cuda.Stream() for _ in caches]
    torch.cuda.synchronize()
    got = []
    for c, s in zip(caches, streams):
        with torch.cuda.stream(s):
            got.append(compact_pages(c, validate=False))
    torch.cuda.synchronize()
    for c, (remap, count), (n, want_remap, table, pool) in zip(caches, got, want):
        assert int(count) == n and remap.tolist() == want_remap and c.page_table.tolist() == table
        _same(_snapshot(c), pool)


@pytest.mark.gpu
def test_validated_page_operations_are_refused_under_capture():
    cache = _cache([9, 0], 4, dev="cuda")
    graph = torch.cuda.CUDAGraph()
    before = cache.page_table.clone()
    with pytest.raises(RuntimeError, match="capturing"):
        with torch.cuda.graph(graph):
            compact_pages(cache)
    torch.cuda.synchronize()
    assert torch.equal(cache.page_table, before)


@pytest.mark.gpu
@pytest.mark.parametrize("P,hkv,d", [(5, 4, 128), (1, 4, 128), (11, 4, 128), (8, 1, 64), (32, 4, 64), (100, 2, 256)])
@pytest.mark.parametrize("pairs", [1, 2, 7, 65])
def test_copy_of_pages_of_whole_chunks(P, hkv, d, pairs):
    """Pages of 1, 5, 11, 16 and 100 KiB: a wave's eight chunks begin and end anywhere in them."""
    print(f"chunks {P} {hkv} {d} {pairs}", flush=True)
    cache = _cache([1], P, hkv, d, torch.float16, "cuda", spare=2 * pairs + 3, seed=pairs)
    order = torch.randperm(cache.num_pages, generator=torch.Generator().manual_seed(pairs)).tolist()
    src, dst = order[:pairs], order[pairs:2 * pairs]
    before = _snapshot(cache)
    copy_pages(cache, _ids(src, "cuda"), _ids(dst, "cuda"))
    _same(_snapshot(cache), _moved(before, list(zip(src, dst))))


def _huge(pages, rows=3, width=4, P=1):
    """A pool of many tiny pages."""
    k = torch.arange(pages * 2, dtype=torch.int32, device="cuda").view(pages, P, 1, 2).to(torch.float32)
    table = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
    return PagedKVCache(k, -k, table, _ids([0] * rows, "cuda"), P)


@pytest.mark.gpu
def test_ids_of_pools_that_take_several_turns_of_the_bitmap():
    """Repetitions and overlaps on both sides of every 2^19 ids."""
    turn = 1 << 19
    pages = 2 * turn + 100
    cache = _huge(pages)
    print("several turns", flush=True)
    src = [0, turn - 1, turn + 1, 2 * turn + 99, turn - 1]
    dst = [turn, 2 * turn, 5, 2 * turn - 1, 7]
    before = _snapshot(cache)
    copy_pages(cache, _ids(src, "cuda"), _ids(dst, "cuda"))
    _same(_snapshot(cache), _moved(before, list(zip(src, dst))))
    for bad, error in ((turn, "twice"), (2 * turn, "twice"), (turn - 1, "src holds too"), (turn + 1, "src holds too"),
                       (2 * turn + 99, "src holds too"), (pages, "dst holds a page outside"), (-1, "dst holds a page")):
        with pytest.raises(AssertionError, match=error):
            copy_pages(cache, _ids(src, "cuda"), _ids(dst[:4] + [bad], "cuda"))
    cache.page_table.copy_(_ids([[2 * turn + 98, 0, 0, 0], [turn + 3, 9, 0, 0], [0, 0, 0, 0]], "cuda"))
    cache = PagedKVCache(cache.k_cache.view(pages // 2, 2, 1, 2), cache.v_cache.view(pages // 2, 2, 1, 2),
                         torch.zeros(4, 2, dtype=torch.int32, device="cuda"), _ids([1, 1, 0, 0], "cuda"), 2)
    cache.page_table[0, 0], cache.page_table[1, 0] = pages // 2 - 1, 3
    for take in ([turn, turn], [pages // 2 - 7] * 2):
        with pytest.raises(AssertionError, match="pages holds a page twice"):
            fork_sequences(cache, _ids([0, 1], "cuda"), _ids([2, 3], "cuda"), _ids(take, "cuda"))
    fork_sequences(cache, _ids([0, 1], "cuda"), _ids([2, 3], "cuda"), _ids([turn, 0], "cuda"))
    assert cache.page_table[2:, 0].tolist() == [turn, 0] and cache.seq_lens.tolist() == [1, 1, 1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("pages,rows,width", [(65536, 4, 8192), (65537, 4, 8192), (65536, 4, 8193), (70, 1, 32768),
                                              (70, 32768, 1), (70, 17, 5), (200, 33, 3)])
def test_free_and_compact_where_one_workgroup_ends(pages, rows, width):
    """Pools and tables at the largest that one workgroup lists, and one beyond."""
    print(f"one workgroup {pages} {rows} {width}", flush=True)
    g = torch.Generator().manual_seed(pages + width)
    cache = _huge(pages, rows, width)
    table = torch.randint(0, pages, (rows, width), generator=g, dtype=torch.int32)
    lens = torch.randint(0, width + 1, (rows,), generator=g, dtype=torch.int32)
    cache.page_table.copy_(table)
    cache.seq_lens.copy_(lens)
    gone = sorted({0, rows // 2, rows - 1}) if rows > 1 else []
    got, count = free_sequences(cache, _ids(gone, "cuda"))
    lens[gone] = 0
    assert torch.equal(cache.seq_lens.cpu(), lens)
    used = torch.zeros(pages, dtype=torch.bool)
    seen = torch.arange(width)[None] < lens[:, None]
    used[table[seen].long()] = True
    free = (~used).nonzero()[:, 0].to(torch.int32)
    assert int(count) == len(free) and torch.equal(got[:len(free)].cpu(), free)
    assert bool((got[len(free):] == -1).all())
    before = _snapshot(cache)
    remap, n = compact_pages(cache)
    n = int(n)
    assert n == int(used.sum())
    ids = torch.arange(pages)
    src, dst = ids[used & (ids >= n)], ids[~used & (ids < n)]
    want = torch.where(used, ids, torch.full_like(ids, -1))
    want[src] = dst
    assert torch.equal(remap.cpu().long(), want)
    _same(_snapshot(cache), _moved(before, list(zip(src.tolist(), dst.tolist()))))
    table[seen] = want[table[seen].long()].to(torch.int32)
    assert torch.equal(cache.page_table.cpu(), table)
