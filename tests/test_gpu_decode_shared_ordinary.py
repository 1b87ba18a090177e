"""paged_decode_attention_shared where ordinary decode could run in its place:
batches in which nothing is shared, several tokens per sequence on pages and types
that ordinary multi-token decode doesn't take, and queries of any alignment.

Tolerance: test_gpu_decode_shared's, whose terms cover ordinary decode too (its
kernels for one query keep P in fp32)."""

from __future__ import annotations

import pytest
import torch

from test_gpu_decode_shared import DTYPES, _check, _ints, _reference, _run, _setup

import flashattntile_amd as fat
from flashattntile_amd import PagedKVCache, paged_decode_attention_shared
from flashattntile_amd.kernels.shared import paged_decode_shared_launch

pytestmark = pytest.mark.gpu

# nothing shared: groups of one sequence, and groups without a prefix
APART = {"one each": [(40, [5]), (3, [70]), (33, [4])], "no prefix": [(0, [45, 4, 130]), (0, [9])]}


@pytest.mark.parametrize("name", list(APART))
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("P", [1, 2, 4, 12, 16])
@pytest.mark.parametrize("tokens", [2, 4])
def test_several_tokens_where_nothing_is_shared(name, dtype, d, P, tokens):
    """A loop that verifies drafts keeps running when its last shared group is down to one sequence."""
    label = f"{name} {dtype} D{d} P{P} T{tokens}"
    print(label, flush=True)
    case = _setup(APART[name], P, 2, d, DTYPES[dtype], tokens, 8, seed=P + tokens)
    out = _run(case)
    _check(out, *_reference(case["q"], case["cache"]), label)
    if P & (P - 1) == 0 and P >= (4 if d == 128 else 8):  # ordinary decode's own shapes
        assert torch.equal(out, fat.paged_decode_attention_multi(case["q"], case["cache"]))


@pytest.mark.parametrize("kv", ["int8", "fp8"])
@pytest.mark.parametrize("P", [1, 12])
def test_several_tokens_of_8_bit_caches_where_nothing_is_shared(kv, P):
    print(f"{kv} P{P}", flush=True)
    case = _setup(APART["one each"], P, 2, 128, torch.bfloat16, 3, 8, kv, seed=P)
    _check(_run(case), *_reference(case["q"], case["cache"], case["scales"]), f"{kv} {P}")


def _one_by_one(q, cache):
    """Every token as a sequence of its own: (queries, cache)."""
    batch, tokens = q.shape[:2]
    lens = [n - tokens + 1 + t for n in cache.seq_lens.tolist() for t in range(tokens)]
    table = torch.stack([row for row in cache.page_table for _ in range(tokens)])
    return q.reshape(batch * tokens, *q.shape[2:]), PagedKVCache(cache.k_cache, cache.v_cache, table, _ints(lens),
                                                                 cache.page_size)


@pytest.mark.parametrize("dtype,d,kv,heads,P", [("fp32", 64, "same", 4, 16), ("fp32", 128, "same", 4, 1),
                                                ("fp16", 256, "same", 4, 16), ("bf16", 32, "same", 4, 12),
                                                ("bf16", 16, "same", 2, 16), ("fp16", 512, "same", 2, 16),
                                                ("fp16", 256, "int8", 4, 16), ("bf16", 32, "fp8", 4, 16)])
@pytest.mark.parametrize("tokens", [2, 5])
def test_several_tokens_of_shapes_that_run_as_ordinary_decode(dtype, d, kv, heads, P, tokens):
    label = f"ordinary {dtype} D{d} {kv} P{P} T{tokens}"
    print(label, flush=True)
    groups = [(96, [5, 30, 64, 7])] if kv == "same" else [(96, [16, 32]), (48, [5])]
    case = _setup(groups, P, 2, d, DTYPES[dtype], tokens, heads, kv, seed=9)
    out = _run(case)
    q, cache = _one_by_one(case["q"], case["cache"])
    if kv == "same":
        _check(out, *_reference(case["q"], case["cache"]), label)
        assert torch.equal(out.view(q.shape), fat.paged_decode_attention(q, cache))
    else:
        assert torch.equal(out.view(q.shape), fat.paged_decode_attention_fp8(q, cache, case["scales"]))


@pytest.mark.parametrize("tokens", [0, 1, 3])
@pytest.mark.parametrize("groups", [[(32, [20])], [(48, [5, 9])], [(0, [7, 40])]])
def test_queries_behind_any_address(tokens, groups):
    """Queries that begin between 16-byte boundaries, and those whose axes of one
    entry have odd strides (torch calls both contiguous)."""
    print(f"addresses {tokens} {groups}", flush=True)
    for heads, hkv in ((8, 2), (1, 1)):
        case = _setup(groups, 16, hkv, 64, torch.float16, tokens, heads, seed=tokens)
        q = case["q"]
        want = _run(case)
        _check(want, *_reference(q, case["cache"]), "as it was")
        room = torch.zeros(q.numel() + 40, dtype=q.dtype, device="cuda")
        views = []
        for offset in (1, 3, 8):
            flat = room.clone()
            flat[offset:offset + q.numel()] = q.flatten()
            views.append(flat[offset:offset + q.numel()].view(q.shape))
        odd = q.clone()
        views.append(odd.as_strided(q.shape, [s if n > 1 else s + 13 for n, s in zip(q.shape, q.stride())]))
        for i, view in enumerate(views):
            assert view.is_contiguous()
            out = paged_decode_attention_shared(view, case["cache"], case["cu_groups"], case["prefix_lens"])
            assert torch.equal(out, want), i
        config = {"prefix_split": 2, "split": 2}
        a, b = (paged_decode_shared_launch(x, case["cache"], case["cu_groups"], case["prefix_lens"], 0.125, 48, 40,
                                           config=config) for x in (q, views[-1]))
        assert torch.equal(a, b)


def test_a_page_id_that_is_the_smallest_number():
    """-2^31 in a used column is a negative page, not a page that isn't shared."""
    case = _setup([(48, [5, 9]), (32, [20])], 16, 2, 64, torch.float16, 0, 8, seed=10)
    table = case["cache"].page_table.clone()
    table[2, 1] = -2 ** 31
    cache = PagedKVCache(case["cache"].k_cache, case["cache"].v_cache, table, case["cache"].seq_lens, 16)
    with pytest.raises(AssertionError, match="negative page id"):
        paged_decode_attention_shared(case["q"], cache, case["cu_groups"], case["prefix_lens"])
