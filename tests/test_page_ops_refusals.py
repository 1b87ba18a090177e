"""What the operations on pages refuse, beyond test_page_ops: on the CPU and the GPU
alike, before anything is changed."""

from __future__ import annotations

import pytest
import torch

from test_page_ops import _cache, _ids, _mirror, _same, _snapshot, device

from flashattntile_amd import PagedKVCache, compact_pages, copy_pages, fork_sequences, free_sequences


def _state(cache):
    return cache.page_table.tolist(), cache.seq_lens.tolist()


# ---------------------------------------------------------------------------
# fork: pages that a row uses
# ---------------------------------------------------------------------------
# rows: a parent of 2 pages, the last part full; one of 1 part full page; one of 2 whole pages; a bystander; empty ones
LENS = [21, 5, 32, 40, 0, 0]


@device
@pytest.mark.parametrize("parents,children,taken", [
    ([0], [4], [(0, 1)]),             # the parent's own last page
    ([0], [4], [(0, 0)]),             # a whole page of the parent's
    ([0, 1], [4, 5], [(1, 0), None]),  # the page that another fork of the call copies from
    ([0, 1], [4, 5], [None, (0, 1)]),
    ([0], [4], [(3, 2)]),             # a bystander's last page
    ([0], [4], [(3, 0)]),
    ([1], [5], [(2, 1)]),
])
def test_fork_refuses_pages_in_use(dev, parents, children, taken):
    cache = _cache(LENS, 16, dev=dev, spare=30)
    table = cache.page_table.tolist()
    used = {p for b, n in enumerate(LENS) for p in table[b][:-(-n // 16)]}
    fresh = [p for p in range(cache.num_pages) if p not in used]
    pages = [fresh[i] if at is None else table[at[0]][at[1]] for i, at in enumerate(taken)]
    before = _snapshot(cache), _state(cache)
    with pytest.raises(AssertionError, match="pages holds a page that a row uses"):
        fork_sequences(cache, _ids(parents, dev), _ids(children, dev), _ids(pages, dev))
    _same(_snapshot(cache), before[0])
    assert _state(cache) == before[1]


@device
def test_fork_takes_pages_that_only_unused_columns_name(dev):
    """A child's own column, one behind a row's end; and what a whole parent's entry names is not looked at."""
    cache = _cache(LENS, 16, dev=dev, spare=30, width=4)
    used = {p for b, n in enumerate(LENS) for p in cache.page_table[b, :-(-n // 16)].tolist()}
    fresh = [p for p in range(cache.num_pages) if p not in used]
    cache.page_table[4, 1] = fresh[0]
    cache.page_table[3, 3] = fresh[1]
    cache.page_table[5, 0] = fresh[1]
    last = int(cache.page_table[2, 1])
    fork_sequences(cache, _ids([0, 2], dev), _ids([4, 5], dev), _ids([fresh[0], last], dev))
    assert cache.page_table[4, 1] == fresh[0] and cache.page_table[5, :2].tolist() == cache.page_table[2, :2].tolist()
    fork_sequences(cache, _ids([], dev), _ids([], dev), _ids([], dev))


@device
def test_fork_with_bad_rows_beside_it(dev):
    """Lengths and ids of rows that the call doesn't name are not its business."""
    cache = _cache(LENS, 16, dev=dev, spare=30)
    named = set(cache.page_table.flatten().tolist())  # a length beyond the table uses all of its columns
    fresh = [p for p in range(cache.num_pages) if p not in named]
    cache.seq_lens[2], cache.seq_lens[1] = 9999, -7
    cache.page_table[3, 0], cache.page_table[3, 1] = -1, 1 << 30
    fork_sequences(cache, _ids([0], dev), _ids([4], dev), _ids([fresh[0]], dev))
    assert int(cache.seq_lens[4]) == 21


@device
@pytest.mark.parametrize("rows,width,pages", [(40, 3000, 200000), (3000, 40, 200000), (5, 70, (1 << 19) + 5),
                                              (300, 900, (1 << 20) + 77)])
def test_fork_looks_at_every_column_of_large_tables(dev, rows, width, pages):
    """Tables of many workgroups, and pools beyond one bitmap: the one column that names a page, anywhere."""
    if dev == "cpu" and rows * width > 200000:
        pytest.skip("the same on the GPU")
    print(f"fork on a large table {dev} {rows} {width} {pages}", flush=True)
    P = 2
    g = torch.Generator().manual_seed(rows)
    k = torch.zeros(pages, P, 1, 2, device=dev)
    table = torch.randint(100, pages, (rows + 1, width), generator=g, dtype=torch.int32)
    lens = torch.randint(0, P * width + 1, (rows + 1,), generator=g, dtype=torch.int32)
    lens[0], lens[rows] = 3, 0
    table[0, :2] = torch.tensor([101, 102], dtype=torch.int32)
    for where in ((rows - 1, width - 1), (rows // 2, width // 2), (1, 0), None):
        for page in (7, pages - 1):
            t, n = table.clone(), lens.clone()
            t[t == page] = page - 1
            if where is not None:
                t[where[0], where[1]] = page
                n[where[0]] = P * where[1] + 1  # the column is just used
            cache = PagedKVCache(k, k, t.to(dev), n.to(dev), P)
            call = lambda: fork_sequences(cache, _ids([0], dev), _ids([rows], dev), _ids([page], dev))
            if where is None:
                call()
                assert cache.page_table[rows, :2].tolist() == [101, page]
                continue
            with pytest.raises(AssertionError, match="that a row uses"):
                call()
            cache.seq_lens[where[0]] = P * where[1]  # and now just not
            call()
            assert int(cache.seq_lens[rows]) == 3


# ---------------------------------------------------------------------------
# held
# ---------------------------------------------------------------------------
@device
@pytest.mark.parametrize("name", ["free", "compact"])
def test_held_columns_are_checked(dev, name):
    """Columns that only `held` covers name pages too, and are columns of the table."""
    def run(cache, held):
        if name == "free":
            return free_sequences(cache, _ids([0], dev), held=held)
        return compact_pages(cache, held=held)

    lens = [20, 40, 0, 1]
    for row, column, value, error in ((2, 3, 1 << 20, "references page 1048576"), (0, 4, -3, "negative page id"),
                                      (3, 1, None, "references page"), (2, 0, -1, "negative page id")):
        cache = _cache(lens, 16, dev=dev, spare=8, width=5)
        cache.page_table[row, column] = cache.num_pages if value is None else value
        held = _ids([5, 3, 4, 2], dev)
        before = _snapshot(cache), _state(cache)
        with pytest.raises(AssertionError, match=error):
            run(cache, held)
        _same(_snapshot(cache), before[0])
        assert _state(cache) == before[1] and held.tolist() == [5, 3, 4, 2]
        held[row] = column  # the columns before it
        run(cache, held)
    for many in (6, 2 ** 31 - 1):
        cache = _cache(lens, 16, dev=dev, spare=8, width=5)
        before = _snapshot(cache), _state(cache)
        with pytest.raises(AssertionError, match="held counts more columns than the page table has \\(5\\)"):
            run(cache, _ids([0, many, 0, 0], dev))
        _same(_snapshot(cache), before[0])
        assert _state(cache) == before[1]
        run(cache, _ids([0, 5, -1, -2 ** 31], dev))  # less than its tokens' columns: those


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(40, 3000), (3000, 40), (5000, 3)])
def test_held_columns_of_large_tables_are_checked(rows, width):
    print(f"held {rows} {width}", flush=True)
    k = torch.zeros(50, 2, 1, 2, device="cuda")
    for where in ((rows - 1, width - 1), (0, 0), (rows // 2, width // 2)):
        table = torch.zeros(rows, width, dtype=torch.int32, device="cuda")
        table[where] = 50
        cache = PagedKVCache(k, k.clone(), table, torch.zeros(rows, dtype=torch.int32, device="cuda"), 2)
        held = torch.zeros(rows, dtype=torch.int32, device="cuda")
        held[where[0]] = where[1] + 1
        with pytest.raises(AssertionError, match="references page 50"):
            free_sequences(cache, _ids([], "cuda"), held=held)
        with pytest.raises(AssertionError, match="references page 50"):
            compact_pages(cache, held=held)
        held[where[0]] = where[1]
        pages, count = free_sequences(cache, _ids([], "cuda"), held=held)
        assert int(count) == (49 if where[1] else 50)


@pytest.mark.gpu
def test_held_of_one_call_is_not_the_next_one_s():
    """On one device and thread the checks share a block of arguments."""
    cache = _cache([20, 40, 0, 1], 16, dev="cuda", spare=8, width=5)
    cache.page_table[2, 3] = -1
    for call in (free_sequences, lambda c, rows, **more: compact_pages(c, **more)):
        with pytest.raises(AssertionError, match="negative page id"):
            call(cache, _ids([], "cuda"), held=_ids([0, 0, 4, 0], "cuda"))
        call(cache, _ids([], "cuda"))


# ---------------------------------------------------------------------------
# The 8-bit copy's layout
# ---------------------------------------------------------------------------
@device
@pytest.mark.parametrize("name", ["copy", "fork", "compact"])
@pytest.mark.parametrize("spread", ["k_cache", "v_cache"])
def test_an_8_bit_copy_whose_rows_are_not_contiguous(dev, name, spread):
    """The kernels read head_dim with a unit stride: refused on the GPU, as append_tokens does."""
    cache = _cache([21, 5, 32, 0], 16, dtype=torch.bfloat16, dev=dev, spare=30)
    copy, scales = _mirror(cache)
    wide = torch.zeros(*copy.k_cache.shape, 2, dtype=torch.int8, device=dev)
    wide[..., 0] = getattr(copy, spread)
    setattr(copy, spread, wide[..., 0])
    used = set(cache.page_table.flatten().tolist())
    fresh = [p for p in range(cache.num_pages) if p not in used]
    call = {"copy": lambda: copy_pages(cache, _ids([0], dev), _ids([fresh[0]], dev), quantized=(copy, scales)),
            "fork": lambda: fork_sequences(cache, _ids([0], dev), _ids([3], dev), _ids([fresh[0]], dev),
                                           quantized=(copy, scales)),
            "compact": lambda: compact_pages(cache, quantized=(copy, scales))}[name]
    before = _snapshot(cache, (copy, scales)), _state(cache)
    if dev == "cpu":
        call()  # torch takes any strides
        return
    with pytest.raises(AssertionError, match="head_dim axis of the quantised pages must be contiguous"):
        call()
    _same(_snapshot(cache, (copy, scales)), before[0])
    assert _state(cache) == before[1]
