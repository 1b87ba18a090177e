"""paged_decode_attention_shared against attention in 64 bits over each sequence's
own table (which holds the shared pages too).

Tolerance, per element, from the kernel's roundings (``_reference``): P enters the
second product as fp16 (half a step, 2^-11 of each p; a p in fp16's subnormals is
off by 2^-25 of the largest at most, n keys of them) or, with bf16 queries and 8-bit
caches, as two bf16 (2^-16), so that a weighted mean of v moves by that share of max
|v|; fp32 scores of up to 64 (log2 units, 2^-24 each, and the sums) move p by less
than 2^-16; and the output's own rounding is half a step.  8-bit caches are compared
on code times scale.
"""

from __future__ import annotations

import math

import pytest
import torch

import flashattntile_amd as fat
from flashattntile_amd import PagedKVCache, paged_decode_attention_shared
from flashattntile_amd.kernels.shared import paged_decode_shared_launch
from flashattntile_amd.quant import quantize_kv_pages

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _setup(groups, P, hkv, d, dtype, tokens=1, heads=8, kv="same", seed=0, spare=3, width=None, poison=True,
           scale=1.0):
    """``groups``: a list of (prefix, [keys behind it per sequence]).  Pages are
    scattered; the pages that a prefix fills are shared, one that it ends in is
    each sequence's own with the same first slots.  What no sequence sees is NaN."""
    g = torch.Generator().manual_seed(seed)
    lens = [n + own for n, owns in groups for own in owns]
    per = [math.ceil(n / P) for n in lens]
    pool = sum(per) + spare
    k = torch.randn(pool, P, hkv, d, generator=g) * scale
    v = torch.randn(pool, P, hkv, d, generator=g)
    perm = torch.randperm(pool, generator=g).tolist()
    table = torch.zeros(len(lens), width or max(per), dtype=torch.int32)
    live = torch.zeros(pool, P, dtype=torch.bool)
    b = 0
    for n, owns in groups:
        lead = b
        for own in owns:
            for c in range(per[b]):
                shared = c < n // P and b > lead
                table[b, c] = table[lead, c] if shared else perm.pop()
                page = int(table[b, c])
                if b > lead and c == n // P and n % P:
                    k[page, :n % P] = k[int(table[lead, c]), :n % P]
                    v[page, :n % P] = v[int(table[lead, c]), :n % P]
                live[page, :min(P, lens[b] - c * P)] = True
            b += 1
    scales = None
    if kv != "same":
        # unused slots are zeros here: a page's scale covers all of its slots
        k[~live], v[~live] = 0.0, 0.0
        qk, qv, sk, sv, _ = quantize_kv_pages(k.to(dtype), v.to(dtype), mode={"int8": "int8", "fp8": "float8_e4m3fn"}[kv])
        k, v, scales = qk, qv, {"k": sk, "v": sv}
        if poison:
            dead = ~live.any(dim=1)
            sk[dead], sv[dead] = float("nan"), float("nan")
    else:
        k, v = k.to(dtype), v.to(dtype)
        if poison:
            k[~live], v[~live] = float("nan"), float("nan")
    cache = PagedKVCache(k.to(DEV), v.to(DEV), table.to(DEV), _ints(lens), P)
    shape = (len(lens), heads, d) if tokens == 0 else (len(lens), tokens, heads, d)
    q = (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)
    cu = [0]
    for _, owns in groups:
        cu.append(cu[-1] + len(owns))
    return {"q": q, "cache": cache, "cu_groups": _ints(cu), "prefix_lens": _ints([n for n, _ in groups]),
            "scales": None if scales is None else {n: t.to(DEV) for n, t in scales.items()}}


def _values(cache, scales):
    """K and V pages in 64 bits."""
    pages = {"k": cache.k_cache.double().cpu(), "v": cache.v_cache.double().cpu()}
    return [x if scales is None else x * scales[n].double().cpu()[:, None, :, None] for n, x in pages.items()]


def _reference(q, cache, scales=None, softmax_scale=None):
    """Output and its bound, in 64 bits."""
    k, v = _values(cache, scales)
    q4 = (q if q.dim() == 4 else q[:, None]).double().cpu()
    scale = q.shape[-1] ** -0.5 if softmax_scale is None else softmax_scale
    batch, tokens, heads, d = q4.shape
    group = heads // k.shape[2]
    out, bound = torch.zeros_like(q4), torch.zeros_like(q4)
    table = cache.page_table.cpu().long()
    part = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -16, torch.float32: 2.0 ** -18}[q.dtype]
    part = part if scales is None else 2.0 ** -16
    tiny = 2.0 ** -25 if q.dtype == torch.float16 and scales is None else 0.0
    half = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(cache.seq_lens.tolist()):
        ids = table[b, :math.ceil(n / cache.page_size)]
        kb = k[ids].reshape(-1, *k.shape[2:])[:n].repeat_interleave(group, dim=1)
        vb = v[ids].reshape(-1, *v.shape[2:])[:n].repeat_interleave(group, dim=1)
        for t in range(tokens):
            seen = n - tokens + 1 + t
            s = torch.einsum("hd,jhd->hj", q4[b, t], kb[:seen]) * scale
            out[b, t] = torch.einsum("hj,jhd->hd", torch.softmax(s, dim=1), vb[:seen])
            top = vb[:seen].abs().amax(dim=0)
            bound[b, t] = (part + 2.0 ** -16 + seen * tiny) * top + half * out[b, t].abs() + 2.0 ** -24
    if q.dim() == 3:
        out, bound = out[:, 0], bound[:, 0]
    return out, bound


def _check(out, ref, bound, label=""):
    err = (out.double().cpu() - ref).abs()
    worst = float((err / bound).max())
    print(f"{label} worst error {float(err.max()):.3e}, {worst:.2f} of its bound", flush=True)
    assert bool((err <= bound).all()), label


def _run(case, **more):
    return paged_decode_attention_shared(case["q"], case["cache"], case["cu_groups"], case["prefix_lens"],
                                         scales=case["scales"], **more)


# (prefix, keys behind it): uniform, ragged, ends inside a page, empty, alone, none behind
GROUPS = {
    "one": [(96, [1, 30, 64, 5])],
    "ragged": [(77, [3, 1, 129]), (0, [40, 2]), (33, [8]), (512, [1, 2, 700, 64, 90, 17, 33])],
    "edges": [(1, [4, 4]), (31, [5, 33]), (32, [32, 31]), (33, [64, 4]), (0, [4]), (64, [4] * 9)],
}


@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kv", ["same", "int8", "fp8"])
@pytest.mark.parametrize("d,heads,hkv", [(128, 8, 2), (64, 7, 1), (128, 4, 4), (64, 48, 1)])
def test_against_64_bits(name, dtype, kv, d, heads, hkv):
    for tokens, P in ((0, 16), (1, 64), (3, 16), (4, 1), (0, 12), (2, 32)):
        if any(own < tokens for _, owns in GROUPS[name] for own in owns):
            continue
        if kv != "same" and any(n % P and len(owns) > 1 for n, owns in GROUPS[name]):
            continue  # a page that a prefix ends in has another scale in every sequence
        label = f"{name} {dtype} {kv} D{d} {heads}/{hkv} T{tokens} P{P}"
        print(label, flush=True)
        case = _setup(GROUPS[name], P, hkv, d, DTYPES[dtype], tokens, heads, kv, seed=len(label))
        _check(_run(case), *_reference(case["q"], case["cache"], case["scales"]), label)


@pytest.mark.parametrize("dtype,kv", [("fp16", "same"), ("bf16", "same"), ("fp16", "fp8"), ("bf16", "int8")])
@pytest.mark.parametrize("sequences", [1, 2, 9, 17, 33, 70])
def test_rows_of_a_group_and_splits(dtype, kv, sequences):
    """From one row tile of a group to many, each with several splits."""
    groups = [(640, [1 + 37 * i % 200 for i in range(sequences)])]
    case = _setup(groups, 16, 2, 128, DTYPES[dtype], 0, 8, kv, seed=sequences)
    ref = _reference(case["q"], case["cache"], case["scales"])
    for config in (None, {"prefix_split": 1, "split": 1}, {"prefix_split": 5}, {"prefix_split": 64, "split": 64},
                   {"split": 3}, {"row_blocks": 1}, {"row_blocks": 4},
                   {"row_blocks": 1, "prefix_split": 2}, {"row_blocks": 4, "prefix_split": 3}):
        print(f"sequences {sequences} {dtype} {kv} {config}", flush=True)
        out = _run(case, config=config)
        _check(out, *ref, f"{sequences} {dtype} {kv} {config}")
        assert torch.equal(out, _run(case, config=config))


@pytest.mark.parametrize("row_blocks", [1, 4])
@pytest.mark.parametrize("dtype,kv", [("fp16", "same"), ("bf16", "same"), ("fp16", "fp8"), ("bf16", "fp8"),
                                      ("fp16", "int8"), ("bf16", "int8")])
@pytest.mark.parametrize("d", [64, 128])
def test_every_number_of_rows_of_a_workgroup(row_blocks, dtype, kv, d):
    """Each kernel at few rows and many, masks of several tokens, scores that rise and fall."""
    for name, P, tokens in (("ragged", 16, 0), ("edges", 1, 4), ("edges", 64, 2)):
        if kv != "same" and any(n % P and len(owns) > 1 for n, owns in GROUPS[name]):
            continue
        case = _setup(GROUPS[name], P, 2, d, DTYPES[dtype], tokens, 16, kv, seed=row_blocks)
        label = f"{name} {dtype} {kv} d{d} P{P} T{tokens} row blocks {row_blocks}"
        print(label, flush=True)
        out = _run(case, config={"row_blocks": row_blocks})
        _check(out, *_reference(case["q"], case["cache"], case["scales"]), label)
    case = _setup([(512, [50, 1, 200] * 12)], 16, 1, d, DTYPES[dtype], 0, 8, seed=6, poison=False)
    cache = case["cache"]
    ids = cache.page_table[0, :32].long()
    ramp = torch.cat([torch.linspace(-3, 3, 256), torch.linspace(3, -3, 256)]).to(DEV).view(32, 16, 1, 1)
    cache.k_cache[ids] = (case["q"][0, 0].float() * ramp).to(DTYPES[dtype])
    out = _run(case, softmax_scale=0.3, config={"row_blocks": row_blocks})
    _check(out, *_reference(case["q"], cache, softmax_scale=0.3), f"scores that rise and fall {row_blocks}")


@pytest.mark.parametrize("dtype,kv,P", [("bf16", "same", 16), ("fp16", "int8", 16), ("fp16", "same", 1)])
def test_long_prefixes(dtype, kv, P):
    print(f"long {dtype} {kv} P{P}", flush=True)
    groups = [(20000, [40, 900, 3]), (4096, [1, 2500]), (P * 7, [64] * 20)]
    case = _setup(groups, P, 1, 128, DTYPES[dtype], 0, 8, kv, seed=4)
    _check(_run(case), *_reference(case["q"], case["cache"], case["scales"]), "long")


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0])
def test_softmax_scales(scale):
    case = _setup(GROUPS["ragged"], 16, 2, 64, torch.float16, 0, 8, seed=5, scale=0.5)
    print(f"scale {scale}", flush=True)
    _check(_run(case, softmax_scale=scale), *_reference(case["q"], case["cache"], softmax_scale=scale), f"scale {scale}")


def test_large_scores():
    """Scores that grow along the keys, by more than the lazy maximum allows, and fall."""
    case = _setup([(256, [50, 1, 200])], 16, 1, 64, torch.bfloat16, 0, 4, seed=6, poison=False)
    cache = case["cache"]
    ids = cache.page_table[0, :16].long()
    ramp = torch.linspace(-3, 3, 256, device=DEV).view(16, 16, 1, 1)
    cache.k_cache[ids] = (case["q"][0, 0].float() * ramp).to(torch.bfloat16)
    print("large scores", flush=True)
    _check(_run(case, softmax_scale=0.4), *_reference(case["q"], cache, softmax_scale=0.4), "large scores")


def test_infinite_scores():
    """Keys with scores of -inf count as nothing, a whole prefix of them too; NaN and +inf show."""
    case = _setup([(64, [20, 3]), (64, [33, 9])], 16, 1, 64, torch.float16, 0, 2, seed=7)
    cache, q = case["cache"], case["q"]
    q[:, :, 0] = 1.0
    first = cache.page_table[0, :4].long()
    cache.k_cache[first, :, :, 0] = float("-inf")  # group 0's whole prefix
    some = cache.page_table[2, 1:3].long()
    cache.k_cache[some, :, :, 0] = float("-inf")  # a tile of group 1's
    print("infinite scores", flush=True)
    out = _run(case)
    ref, bound = _reference(q, cache)
    _check(out, ref, bound, "-inf scores")
    last = cache.page_table[3, 4].long()
    cache.v_cache[last, 3, 0, 5] = float("inf")  # seen by sequence 3 alone
    cache.v_cache[last, 4, 0, 6] = float("nan")
    cache.k_cache[cache.page_table[1, 4].long(), 0, 0, 1] = float("nan")  # sequence 1's scores
    out = _run(case).float().cpu()
    assert bool((out[3, :, 5] == float("inf")).all()) and bool(out[3, :, 6].isnan().all())
    assert bool(out[1].isnan().all())
    clean = torch.ones(4, 2, 64, dtype=torch.bool)
    clean[3, :, 5:7], clean[1] = False, False
    assert bool(((out.double() - ref).abs() <= bound)[clean].all())


def test_layouts():
    """Heads before slots, K and V of one tensor, strided table, lengths, groups and queries."""
    base = _setup(GROUPS["ragged"], 16, 2, 64, torch.float16, 0, 8, seed=8)
    want = _run(base)
    c, q = base["cache"], base["q"]
    hnd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.k_cache, c.v_cache)]
    joint = torch.stack([c.k_cache, c.v_cache])
    wide = torch.full((c.batch_size, 2 * c.max_pages_per_seq), -1, dtype=torch.int32, device=DEV)
    wide[:, ::2] = c.page_table
    for k, v in ((c.k_cache, c.v_cache), hnd, (joint[0], joint[1])):
        for table in (c.page_table, wide[:, ::2]):
            two = torch.stack([c.seq_lens, c.seq_lens], dim=1)
            cache = PagedKVCache(k, v, table, two[:, 0], 16)
            pad = torch.zeros(q.shape[0], 9, 64, dtype=q.dtype, device=DEV)
            pad[:, 1:] = q
            cu = torch.stack([base["cu_groups"]] * 2, dim=1)[:, 1]
            assert torch.equal(paged_decode_attention_shared(pad[:, 1:], cache, cu, base["prefix_lens"]), want)


def test_behind_4_gib():
    """Pages whose byte offsets pass 32 bits, in the prefix and behind it."""
    print("behind 4 GiB", flush=True)
    pool = 140000
    k = torch.zeros(pool, 16, 8, 128, dtype=torch.float16, device=DEV)  # 4.6 GB
    table = torch.tensor([[pool - 1, 5, pool - 3, pool - 2], [pool - 1, 5, pool - 3, 7]], dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for page in table.unique().tolist():
        k[page] = torch.randn(16, 8, 128, generator=g, device=DEV).half()
    cache = PagedKVCache(k, k, table, _ints([60, 49]), 16)
    q = torch.randn(2, 8, 128, generator=g, device=DEV).half()
    out = paged_decode_attention_shared(q, cache, _ints([0, 2]), _ints([48]))
    ids = table.unique()
    small = PagedKVCache(k[ids.long()].contiguous(), k[ids.long()].contiguous(),
                         torch.searchsorted(ids, table).to(torch.int32), cache.seq_lens, 16)
    _check(out, *_reference(q, small), "behind 4 GiB")


@pytest.mark.parametrize("dtype,d,kv,heads,tokens", [("fp32", 64, "same", 4, 0), ("fp16", 256, "same", 4, 0),
                                                     ("bf16", 32, "same", 4, 0), ("bf16", 16, "same", 2, 0),
                                                     ("fp16", 256, "int8", 4, 0)])
def test_shapes_that_run_as_ordinary_decode(dtype, d, kv, heads, tokens):
    print(f"ordinary {dtype} D{d} {kv}", flush=True)
    case = _setup(GROUPS["one"], 16, 2, d, DTYPES[dtype], tokens, heads, kv, seed=9)
    out = _run(case)
    ref, bound = _reference(case["q"], case["cache"], case["scales"])
    err = (out.double().cpu() - ref).abs()
    if kv == "same":
        assert bool((err <= bound + 2.0 ** -14).all())
    if case["scales"] is None:
        assert torch.equal(out, fat.paged_decode_attention(case["q"], case["cache"]))
    else:
        assert torch.equal(out, fat.paged_decode_attention_fp8(case["q"], case["cache"], case["scales"]))


def test_refusals():
    case = _setup([(48, [5, 9]), (32, [20])], 16, 2, 64, torch.float16, 0, 8, seed=10)
    q, cache, cu, pre = case["q"], case["cache"], case["cu_groups"], case["prefix_lens"]

    def refused(error, kind=ValueError, q=q, cache=cache, cu=cu, pre=pre, **more):
        with pytest.raises(kind, match=error):
            paged_decode_attention_shared(q, cache, cu, pre, **more)

    refused("cache must be a PagedKVCache", TypeError, cache=None)
    refused("q must be", q=q[0])
    refused("q batch", q=q[:2])
    refused("q head_dim", q=q[..., :32])
    refused("divisible", q=q[:, :7])
    refused("1 to 64 tokens", q=q[:, None].expand(3, 65, 8, 64))
    refused("cu_groups must be a 1-D int32", cu=cu.long())
    refused("prefix_lens must be a 1-D int32", pre=pre.float())
    refused("one entry more", cu=cu[:2])
    refused("one entry more", cu=cu[:1], pre=pre[:0])
    refused("one device", cu=cu.cpu())
    refused("needs scales", scales={"k": q, "v": q})
    refused("must match cache dtype", q=q.float())
    refused("unknown shared decode config", config={"split_k": 2})
    refused("prefix_split must be", config={"prefix_split": 65})
    refused("split must be", config={"split": 0})
    refused("row_blocks must be", config={"row_blocks": 3})
    # what lies on the device
    refused("start at 0", cu=_ints([1, 2, 3]))
    refused("end at the batch size", cu=_ints([0, 1, 2]))
    refused("non-decreasing", cu=_ints([0, 4, 3]))
    refused("non-negative", pre=_ints([48, -1]))
    refused("no longer than", pre=_ints([54, 32]))
    refused("no longer than", q=q[:, None].repeat(1, 7, 1, 1))
    refused("share the pages", cu=_ints([0, 1, 3]))
    refused("hold its 60 new", q=q[:, None].repeat(1, 60, 1, 1), pre=_ints([0, 0]))
    refused("non-negative", AssertionError, cache=PagedKVCache(cache.k_cache, cache.v_cache, cache.page_table,
                                                               _ints([-1, 57, 52]), 16), pre=_ints([0, 0]), cu=_ints([0, 1, 3]))
    refused("capacity", AssertionError, cache=PagedKVCache(cache.k_cache, cache.v_cache, cache.page_table,
                                                           _ints([53, 57, 520]), 16))
    bad = cache.page_table.clone()
    bad[2, 1] = cache.num_pages
    refused("references page", AssertionError, cache=PagedKVCache(cache.k_cache, cache.v_cache, bad, cache.seq_lens, 16))
    bad[2, 1] = -2
    refused("negative page id", AssertionError, cache=PagedKVCache(cache.k_cache, cache.v_cache, bad, cache.seq_lens, 16))
    cpu = PagedKVCache(cache.k_cache.cpu(), cache.v_cache.cpu(), cache.page_table.cpu(), cache.seq_lens.cpu(), 16)
    refused("ROCm", RuntimeError, q=q.cpu(), cache=cpu, cu=cu.cpu(), pre=pre.cpu())
    # and the call still works
    _check(_run(case), *_reference(q, cache), "after refusals")


def test_unused_table_columns_and_bad_ids_behind_the_end():
    """Columns behind a sequence's end hold anything."""
    case = _setup([(40, [5, 60, 8])], 16, 1, 64, torch.float16, 0, 4, seed=11, width=12)
    table = case["cache"].page_table
    for b, n in enumerate(case["cache"].seq_lens.tolist()):
        table[b, math.ceil(n / 16):] = 1 << 30 if b else -7
    print("unused columns", flush=True)
    out = _run(case)
    ok = table.clamp(0, case["cache"].num_pages - 1)
    cache = PagedKVCache(case["cache"].k_cache, case["cache"].v_cache, ok, case["cache"].seq_lens, 16)
    _check(out, *_reference(case["q"], cache), "unused columns")


def test_captured_and_replayed():
    """One graph, replayed while lengths, groups, prefixes and table change, with eager work between."""
    print("capture", flush=True)
    case = _setup([(96, [20, 33, 50]), (64, [70, 8])], 16, 2, 128, torch.bfloat16, 0, 8, seed=12, poison=False)
    cache, q = case["cache"], case["q"]
    cu, pre = case["cu_groups"], case["prefix_lens"]
    out = torch.empty_like(q)
    config = {"prefix_split": 3, "split": 2}
    workspace = torch.empty(4 * 5 * 8 * 5 * 130, dtype=torch.uint8, device=DEV)

    def launch():
        paged_decode_shared_launch(q, cache, cu, pre, 128 ** -0.5, 96, 70, out=out, workspace=workspace, config=config)

    launch()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    start = cache.seq_lens.clone(), cu.clone(), pre.clone()
    for lens, groups, prefixes in ((None, None, None), ([97, 100, 99, 100, 65], [0, 3, 5], [90, 60]),
                                   ([116, 129, 146, 134, 72], [0, 2, 5], [96, 0]), (None, None, None),
                                   ([1, 2, 3, 134, 72], [0, 3, 3], [1, 64])):
        cache.seq_lens.copy_(start[0] if lens is None else _ints(lens))
        cu.copy_(start[1] if groups is None else _ints(groups))
        pre.copy_(start[2] if prefixes is None else _ints(prefixes))
        if groups == [0, 3, 3]:
            cu[2] = 5  # the second group is the last two sequences
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        _check(out, *_reference(q, cache), f"replay {lens} {groups}")
        replayed = out.clone()
        launch()
        assert torch.equal(out, replayed)


def test_on_streams_at_once():
    print("streams", flush=True)
    cases = [_setup([(512, [40, 1, 90, 7]), (64, [300])], 16, 2, 128, torch.float16, 0, 8, seed=s) for s in range(4)]
    want = [_run(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(_run(c))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)
