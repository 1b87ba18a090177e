"""8-bit caches behind prefixes that end inside a page.  A page has one scale per KV
head for all of its slots, so the page that a prefix ends in holds other codes of the
same first keys in every sequence (each has requantised its own), and each row sees
its own.  Reference and tolerance: test_gpu_decode_shared's, on code times scale over
each sequence's own table."""

from __future__ import annotations

import pytest
import torch

from test_gpu_decode_shared import DEV, DTYPES, GROUPS, _check, _ints, _reference, _run, _setup

from flashattntile_amd import PagedKVCache, append_tokens, fork_sequences, paged_decode_attention_shared, quantize_cache
from flashattntile_amd.kernels.shared import paged_decode_shared_launch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["ragged", "edges"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kv", ["int8", "fp8"])
@pytest.mark.parametrize("d,heads,hkv", [(128, 8, 2), (64, 48, 1)])
def test_every_row_sees_its_own_last_page(name, dtype, kv, d, heads, hkv):
    for tokens, P in ((0, 16), (0, 64), (3, 16), (0, 12), (4, 128)):
        if any(own < tokens for _, owns in GROUPS[name] for own in owns):
            continue
        case = _setup(GROUPS[name], P, hkv, d, DTYPES[dtype], tokens, heads, kv, seed=P + tokens)
        ref = _reference(case["q"], case["cache"], case["scales"])
        for config in (None, {"row_blocks": 1, "prefix_split": 3, "split": 2}, {"row_blocks": 4, "prefix_split": 2}):
            label = f"{name} {dtype} {kv} D{d} {heads}/{hkv} T{tokens} P{P} {config}"
            print(label, flush=True)
            _check(_run(case, config=config), *ref, label)


@pytest.mark.parametrize("kv", ["int8", "fp8"])
def test_pages_larger_than_the_prefix(kv):
    """Nothing of the prefix fills a page: all keys are each row's own."""
    print(f"large pages {kv}", flush=True)
    case = _setup([(1000, [30, 500, 5]), (1023, [1, 2])], 1024, 2, 128, torch.bfloat16, 0, 8, kv, seed=3)
    ref = _reference(case["q"], case["cache"], case["scales"])
    _check(_run(case), *ref, "large pages")
    out = paged_decode_shared_launch(case["q"], case["cache"], case["cu_groups"], case["prefix_lens"], 128 ** -0.5, 1023,
                                     500, scales=case["scales"])
    _check(out, *ref, "large pages, launched")


@pytest.mark.parametrize("mode", ["int8", "float8_e4m3fn"])
def test_samples_of_a_prompt_that_ends_inside_a_page(mode):
    """A prompt, forks of it, and tokens for each through an 8-bit copy."""
    print(f"samples {mode}", flush=True)
    P, hkv, d, prompt, rows = 16, 2, 64, 39, 4
    g = torch.Generator().manual_seed(2)
    k = torch.zeros(20, P, hkv, d, dtype=torch.float16, device=DEV)
    cache = PagedKVCache(k, k.clone(), torch.zeros(rows, 4, dtype=torch.int32, device=DEV), _ints([prompt, 0, 0, 0]), P)
    cache.page_table[0, :3] = _ints([7, 3, 11])
    for page in (7, 3, 11):
        k[page] = torch.randn(P, hkv, d, generator=g).half()
        cache.v_cache[page] = torch.randn(P, hkv, d, generator=g).half()
    copy = quantize_cache(cache, mode=mode)
    fork_sequences(cache, _ints([0] * 3), _ints([1, 2, 3]), _ints([0, 1, 2]), quantized=copy)
    for step in range(4):
        new = torch.randn(2, rows, hkv, d, generator=g) * torch.tensor([1.0, 3.0, 9.0, 0.3]).view(1, rows, 1, 1)
        append_tokens(cache, new[0].half().to(DEV), new[1].half().to(DEV), quantized=copy)
        q = torch.randn(rows, 4, d, generator=g).half().to(DEV)
        scales = {"k": copy[1].k, "v": copy[1].v}
        out = paged_decode_attention_shared(q, copy[0], _ints([0, rows]), _ints([prompt]), scales=scales)
        _check(out, *_reference(q, copy[0], scales), f"{mode} step {step}")
