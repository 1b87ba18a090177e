"""The ways to shared-prefix decode: the custom op, the backend's route, the choice
of splits, the host's refusals (on the CPU), and a run with the operations on
pages (on the GPU)."""

from __future__ import annotations

import pytest
import torch

import flashattntile_amd as fat
from flashattntile_amd import (PagedKVCache, append_tokens, compact_pages, fork_sequences, free_sequences,
                               paged_decode_attention_shared, quantize_cache)
from flashattntile_amd.backend import AttentionMetadata, FlashAttnTileBackend
from flashattntile_amd.kernels.shared import shared_splits


def _cache(dtype=torch.float16, dev="cpu", lens=(20, 24, 9), P=8, hkv=2, d=64, pages=12):
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(pages, P, hkv, d, generator=g).to(dtype).to(dev) for _ in range(2))
    table = torch.tensor([[3, 5, 1, 0], [3, 5, 7, 2], [4, 6, 0, 0]], dtype=torch.int32, device=dev)
    return PagedKVCache(k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev), P)


def _ints(values, dev="cpu"):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def test_op_schema_and_fake_shapes():
    with torch._subclasses.fake_tensor.FakeTensorMode():
        k = torch.empty(12, 16, 2, 64, device="meta")
        pt, sl = torch.empty(3, 3, dtype=torch.int32, device="meta"), torch.empty(3, dtype=torch.int32, device="meta")
        cu, pre = torch.empty(3, dtype=torch.int32, device="meta"), torch.empty(2, dtype=torch.int32, device="meta")
        sc = torch.empty(12, 2, device="meta")
        op = torch.ops.flashattn_tile.paged_decode_shared
        for shape in ((3, 8, 64), (3, 4, 8, 64)):
            q = torch.empty(shape, device="meta")
            assert op(q, k, k, pt, sl, cu, pre, 16, 0.25).shape == shape
            assert op(q, k.to(torch.int8), k.to(torch.int8), pt, sl, cu, pre, 16, 0.25, sc, sc).shape == shape
        with pytest.raises(RuntimeError, match="groups \\+ 1"):
            op(q, k, k, pt, sl, cu, sl, 16, 0.25)
    assert fat.PAGED_DECODE_SHARED_OP == "flashattn_tile::paged_decode_shared"
    assert str(op.default._schema) == (
        "flashattn_tile::paged_decode_shared(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, "
        "Tensor seq_lens, Tensor cu_groups, Tensor prefix_lens, SymInt page_size, float softmax_scale, "
        "Tensor? k_scale=None, Tensor? v_scale=None) -> Tensor")


def test_op_compiles_without_graph_breaks():
    q = torch.empty(2, 4, 64, device="meta", dtype=torch.float16)
    k = torch.empty(4, 16, 2, 64, device="meta", dtype=torch.float16)
    pt, sl = torch.zeros(2, 2, dtype=torch.int32, device="meta"), torch.zeros(2, dtype=torch.int32, device="meta")
    cu, pre = torch.zeros(2, dtype=torch.int32, device="meta"), torch.zeros(1, dtype=torch.int32, device="meta")

    def fn(x):
        return torch.ops.flashattn_tile.paged_decode_shared(x, k, k, pt, sl, cu, pre, 16, 0.35) * 2

    assert torch._dynamo.explain(fn)(q).graph_break_count == 0
    assert torch.compile(fn, fullgraph=True, backend="eager")(q).shape == q.shape


def test_backend_route():
    backend = FlashAttnTileBackend(num_heads=4, num_kv_heads=2, head_dim=64, page_size=8)
    cache, cu, pre = _cache(), _ints([0, 2, 3]), _ints([16, 0])
    meta = AttentionMetadata(cu_groups=cu, prefix_lens=pre)
    for shape in ((3, 4, 64), (3, 1, 4, 64), (3, 2, 4, 64)):
        assert backend.route(torch.zeros(shape), meta) == "decode_shared"
        with pytest.raises(RuntimeError, match="ROCm device"):
            backend.forward(torch.zeros(shape).half(), cache, meta)
    assert "decode_shared" in backend.ROUTES
    assert backend.route(torch.zeros(3, 4, 64), AttentionMetadata()) == "decode"
    assert backend.route(torch.zeros(3, 4, 64), AttentionMetadata(cu_groups=cu, is_prefill=True)) == "prefill"
    with pytest.raises(ValueError, match="prefix_lens"):
        backend.forward(torch.zeros(3, 4, 64).half(), cache, AttentionMetadata(cu_groups=cu))
    with pytest.raises(ValueError, match="heads"):
        backend.forward(torch.zeros(3, 6, 64).half(), cache, meta)
    with pytest.raises(ValueError, match="3-D or 4-D"):
        backend.forward(torch.zeros(4, 64).half(), cache, meta)


def test_host_refusals():
    cache, cu, pre, q = _cache(), _ints([0, 2, 3]), _ints([16, 0]), torch.zeros(3, 4, 64).half()

    def refused(error, kind=ValueError, **more):
        args = dict(q=q, cache=cache, cu_groups=cu, prefix_lens=pre)
        args.update(more)
        with pytest.raises(kind, match=error):
            paged_decode_attention_shared(**args)

    refused("ROCm device", RuntimeError)
    refused("must be a PagedKVCache", TypeError, cache=None)
    refused("q must be", q=torch.zeros(4, 64).half())
    refused("q batch 2", q=torch.zeros(2, 4, 64).half())
    refused("head_dim 32", q=torch.zeros(3, 4, 32).half())
    refused("divisible", q=torch.zeros(3, 5, 64).half())
    refused("1 to 64 tokens", q=torch.zeros(3, 65, 4, 64).half())
    refused("1 to 64 tokens", q=torch.zeros(3, 0, 4, 64).half())
    refused("cu_groups must be a 1-D int32", cu_groups=cu.long())
    refused("prefix_lens must be a 1-D int32", prefix_lens=pre[:, None])
    refused("one entry more", prefix_lens=_ints([16]))
    refused("one entry more", cu_groups=_ints([0]), prefix_lens=_ints([]))
    refused("must match cache dtype", q=torch.zeros(3, 4, 64))
    refused("only such a cache takes them", scales={"k": torch.ones(12, 2), "v": torch.ones(12, 2)})


def _uses(cfg, prefix, own):
    assert cfg["prefix_chunk"] % 32 == 0 and cfg["chunk"] % 32 == 0
    assert 1 <= cfg["prefix_split"] <= 64 and 1 <= cfg["split"] <= 64
    assert cfg["prefix_split"] * cfg["prefix_chunk"] >= prefix and cfg["split"] * cfg["chunk"] >= own


@pytest.mark.parametrize("prefix", [0, 1, 31, 500, 4096, 100000, 2 ** 31 - 5000])
@pytest.mark.parametrize("own", [0, 1, 33, 5000, 2 ** 31 - 5000])
def test_splits_cover_every_length(prefix, own):
    for hkv in (1, 8, 64):
        for rows in (1, 32, 33, 4096):
            for groups in (1.0, 3.7, 500.0):
                for sequences in (1.0, 17.5, 4000.0):
                    _uses(shared_splits(hkv, rows, -(-rows // 32), groups, prefix, sequences, own, 32 * rows), prefix,
                          own)


def test_splits_fill_the_chip_and_no_more():
    # one long prefix of 128 sequences x 4 rows: 8 heads x 4 tiles of 128 rows x 8 = 256 workgroups
    assert shared_splits(8, 512, 1, 1.0, 32768, 128.0, 2000, 4096)["prefix_split"] == 8
    # few rows are worth more partials than many
    few, many = (shared_splits(8, rows, 1, 1.0, 4096, 8.0, 100, 8 * rows)["prefix_split"] for rows in (8, 128))
    assert 8 <= many < few <= 24
    assert shared_splits(8, 8, 1, 1.0, 31, 2.0, 100, 64)["prefix_split"] == 1
    # many sequences need no split of their own keys, few do, in chunks of 256 at least
    assert shared_splits(8, 512, 1, 1.0, 32768, 128.0, 2000, 4096)["split"] == 1
    assert shared_splits(8, 16, 1, 1.0, 512, 2.0, 100000, 64)["split"] == 64
    assert shared_splits(8, 16, 1, 1.0, 512, 2.0, 1000, 64)["split"] == 3


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [0, 1, 3])
@pytest.mark.parametrize("mode", [None, "int8"])
def test_op_and_backend_run_the_function(tokens, mode):
    print(f"op and backend {tokens} {mode}", flush=True)
    cache, cu, pre = _cache(dev="cuda"), _ints([0, 2, 3], "cuda"), _ints([16, 0], "cuda")
    qcache, scales = quantize_cache(cache, mode=mode) if mode else (cache, None)
    sc = () if scales is None else (scales.k, scales.v)
    shape = (3, 4, 64) if tokens == 0 else (3, tokens, 4, 64)
    q = torch.randn(shape, generator=torch.Generator().manual_seed(1)).half().cuda()
    want = paged_decode_attention_shared(q, qcache, cu, pre, softmax_scale=0.11, scales=scales)
    got = torch.ops.flashattn_tile.paged_decode_shared(q, qcache.k_cache, qcache.v_cache, qcache.page_table,
                                                       qcache.seq_lens, cu, pre, 8, 0.11, *sc)
    assert torch.equal(got, want)
    backend = FlashAttnTileBackend(num_heads=4, num_kv_heads=2, head_dim=64, page_size=8)
    meta = AttentionMetadata(softmax_scale=0.11, kv_scales=scales, cu_groups=cu, prefix_lens=pre)
    got = backend.forward(q, qcache, meta)
    assert torch.equal(got, want[:, 0] if tokens == 1 else want)
    compiled = torch.compile(lambda x: torch.ops.flashattn_tile.paged_decode_shared(
        x, qcache.k_cache, qcache.v_cache, qcache.page_table, qcache.seq_lens, cu, pre, 8, 0.11, *sc),
        fullgraph=True, backend="eager")
    assert torch.equal(compiled(q), want)
    with pytest.raises(ValueError, match="given together"):
        torch.ops.flashattn_tile.paged_decode_shared(q, qcache.k_cache, qcache.v_cache, qcache.page_table,
                                                     qcache.seq_lens, cu, pre, 8, 0.11, torch.ones(12, 2, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [None, "float8_e4m3fn"])
def test_a_run_of_samples_of_one_prompt(mode):
    """A prompt, four samples forked from it, tokens for each, decode with the prompt
    read once; two samples end, the pool is packed, and the others decode on: to the
    bit as before the pages moved, and as ordinary decode within both kernels'
    roundings (test_gpu_decode_shared's bound holds for the output; ordinary decode
    is held to 2e-3 elsewhere)."""
    from test_gpu_decode_shared import _check, _reference

    print(f"samples of one prompt {mode}", flush=True)
    P, hkv, d, heads, prompt, rows = 16, 2, 128, 8, 100, 5
    g = torch.Generator().manual_seed(3)
    pages = 40
    cache = PagedKVCache(torch.zeros(pages, P, hkv, d, dtype=torch.float16, device="cuda"),
                         torch.zeros(pages, P, hkv, d, dtype=torch.float16, device="cuda"),
                         torch.zeros(rows, 10, dtype=torch.int32, device="cuda"), _ints([0] * rows, "cuda"), P)
    free = torch.randperm(pages, generator=g).tolist()
    copy = quantize_cache(cache, mode=mode) if mode else None

    def step(live):
        lens = cache.seq_lens.tolist()
        for b in live:
            if lens[b] % P == 0:
                cache.page_table[b, lens[b] // P] = free.pop()
        sub = PagedKVCache(cache.k_cache, cache.v_cache, cache.page_table[live].contiguous(),
                           cache.seq_lens[live].contiguous(), P)
        pair = None
        if mode:
            pair = (PagedKVCache(copy[0].k_cache, copy[0].v_cache, sub.page_table, sub.seq_lens, P), copy[1])
        new = torch.randn(2, len(live), hkv, d, generator=g).half().cuda()
        append_tokens(sub, new[0], new[1], quantized=pair)
        cache.seq_lens[live] = sub.seq_lens

    def decode(q, live, prefix):
        """``live`` rows as one group behind the prompt."""
        source = copy[0] if mode else cache
        sub = PagedKVCache(source.k_cache, source.v_cache, cache.page_table[live].contiguous(),
                           cache.seq_lens[live].contiguous(), P)
        scales = copy[1] if mode else None
        out = paged_decode_attention_shared(q[live], sub, _ints([0, len(live)], "cuda"), _ints([prefix], "cuda"),
                                            scales=scales)
        _check(out, *_reference(q[live], sub, None if scales is None else {"k": scales.k, "v": scales.v}), "samples")
        return out

    for _ in range(prompt):
        step([0])
    take = [free.pop() for _ in range(4)]
    fork_sequences(cache, _ints([0] * 4, "cuda"), _ints([1, 2, 3, 4], "cuda"), _ints(take, "cuda"), quantized=copy)
    # An 8-bit copy's last page has a scale of each row's own tokens: the prefix ends where its pages do.
    prefix = prompt if mode is None else prompt // P * P
    everyone = [0, 1, 2, 3, 4]
    for n in (1, 30):
        for _ in range(n):
            step(everyone)
        decode(torch.randn(rows, heads, d, generator=g).half().cuda(), everyone, prefix)
    left, count = free_sequences(cache, _ints([1, 3], "cuda"))
    assert int(count) == pages - len(set(cache.page_table[[0, 2, 4], :9].flatten().tolist()))
    q = torch.randn(rows, heads, d, generator=g).half().cuda()
    live = [0, 2, 4]
    before = decode(q, live, prefix)
    remap, used = compact_pages(cache, quantized=copy)
    assert int(used) == pages - int(count) and int(remap.max()) == int(used) - 1
    assert torch.equal(decode(q, live, prefix), before)
    free = list(range(pages - 1, int(used) - 1, -1))
    for _ in range(20):
        step(live)
    decode(q, live, prefix)
