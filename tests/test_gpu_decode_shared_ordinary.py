"""paged_decode_attention_shared where ordinary decode could run in its place:
batches in which nothing is shared, and several tokens per sequence on types and
head_dims that ordinary multi-token decode doesn't take.

Tolerance: test_gpu_decode_shared's, whose terms cover ordinary decode too (its
kernels for one query keep P in fp32)."""

from __future__ import annotations

import pytest
import torch

from test_gpu_decode_shared import DTYPES, _check, _ints, _reference, _run, _setup

import flashattntile_amd as fat
from flashattntile_amd import PagedKVCache

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
