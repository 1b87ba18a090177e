"""paged_decode_attention_shared where ordinary decode could run in its place:
batches in which nothing is shared.

Tolerance: test_gpu_decode_shared's, whose terms cover ordinary decode too (its
kernels for one query keep P in fp32)."""

from __future__ import annotations

import pytest
import torch

from test_gpu_decode_shared import DTYPES, _check, _reference, _run, _setup

import flashattntile_amd as fat

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
