"""Host side of shared-prefix decode: buffers that a caller of the launch without
validation brings along, and the partials of a launch (no GPU needed)."""

from __future__ import annotations

import pytest
import torch

from flashattntile_amd import PagedKVCache, _hip
from flashattntile_amd.kernels.shared import paged_decode_shared_launch, shared_splits


def _ints(values):
    return torch.tensor(values, dtype=torch.int32)


def _launch(**more):
    k = torch.zeros(12, 8, 2, 64, dtype=torch.float16)
    cache = PagedKVCache(k, k.clone(), torch.zeros(3, 4, dtype=torch.int32), _ints([20, 24, 9]), 8)
    return paged_decode_shared_launch(torch.zeros(3, 4, 64, dtype=torch.float16), cache, _ints([0, 2, 3]), _ints([16, 0]),
                                      0.125, 16, 9, config={"prefix_split": 1, "split": 1}, **more)


NEED = 4 * 3 * 4 * 2 * 66


@pytest.mark.parametrize("out", [torch.zeros(3, 4, 32, dtype=torch.float16), torch.zeros(2, 4, 64, dtype=torch.float16),
                                 torch.zeros(3, 4, 64), torch.zeros(3, 4, 64, dtype=torch.bfloat16),
                                 torch.zeros(3, 4, 64, dtype=torch.float16, device="meta"),
                                 torch.zeros(3, 4, 128, dtype=torch.float16)[..., ::2]])
def test_launch_refuses_outputs_it_would_write_past(out):
    with pytest.raises(ValueError, match="out must be"):
        _launch(out=out)


def test_launch_refuses_a_workspace_elsewhere_or_with_gaps():
    with pytest.raises(ValueError, match="workspace must"):
        _launch(workspace=torch.zeros(NEED, dtype=torch.uint8, device="meta"))
    with pytest.raises(ValueError, match="workspace must"):
        _launch(workspace=torch.zeros(2 * NEED, dtype=torch.uint8)[::2])


def _partials(batch, tokens, big, small, heads=32, kv_heads=8, prefix=1024, group=None):
    """The splits of one long sequence among short ones, and the bytes of their partials at head_dim 128."""
    own = [big] + [small] * (batch - 1)
    per_seq = tokens * heads // kv_heads
    rows = batch * tokens * heads
    cfg = shared_splits(kv_heads, (group or batch) * per_seq, -(-per_seq // 32), 1.0, prefix, sum(own) / big, big, rows,
                        batch)
    assert cfg["prefix_split"] * cfg["prefix_chunk"] >= prefix and cfg["split"] * cfg["chunk"] >= big
    return cfg, 4 * rows * (cfg["prefix_split"] + cfg["split"]) * 130


def test_one_long_sequence_does_not_cut_every_other_into_64():
    """Every sequence has a slot per chunk: their partials were 145 MB, 1.1 and 2.2 GB."""
    for batch, tokens, big, most, size in ((128, 1, 32768, 16, 48e6), (256, 4, 32768, 16, 250e6), (256, 8, 65536, 16, 512e6)):
        cfg, bytes_ = _partials(batch, tokens, big, 100)
        assert 4 <= cfg["split"] <= most and bytes_ <= size, (batch, tokens, cfg, bytes_)
    # few sequences keep what fills the chip
    assert _partials(2, 1, 100000, 100000, prefix=512)[0]["split"] == 64
    assert _partials(16, 1, 65536, 100)[0]["split"] >= 16


@pytest.mark.parametrize("batch", [1, 7, 300, 4096])
@pytest.mark.parametrize("tokens", [1, 8, 64])
@pytest.mark.parametrize("big", [1, 500, 20000, 1000000])
def test_partials_stay_below_a_ceiling(batch, tokens, big):
    for heads, kv_heads in ((32, 8), (128, 8), (8, 8), (64, 1)):
        for prefix in (0, 100, 100000):
            for small in (1, big):
                cfg, bytes_ = _partials(batch, tokens, big, small, heads, kv_heads, prefix)
                assert bytes_ <= 2 ** 29 or cfg["prefix_split"] == cfg["split"] == 1


@pytest.mark.parametrize("shape", [(3, 4, 64), (3, 5, 4, 64), (1, 2, 64)])
@pytest.mark.parametrize("splits", [(1, 1), (7, 3), (64, 64)])
def test_the_launch_allocates_what_the_library_says(monkeypatch, shape, splits):
    given = []
    monkeypatch.setattr(_hip, "current_stream_handle", lambda device: 0)
    monkeypatch.setattr(_hip, "shared_with_args", lambda a, workspace, stream: given.append(workspace.numel()))
    batch, k = shape[0], torch.zeros(12, 8, 2, 64, dtype=torch.float16)
    cache = PagedKVCache(k, k.clone(), torch.zeros(batch, 4, dtype=torch.int32), _ints([20] * batch), 8)
    paged_decode_shared_launch(torch.zeros(shape, dtype=torch.float16), cache, _ints([0, batch]), _ints([16]), 0.125, 16,
                               9, config={"prefix_split": splits[0], "split": splits[1]})
    rows = batch * (shape[1] if len(shape) == 4 else 1)
    assert given == [_hip.lib().fat_paged_decode_shared_workspace_bytes(rows, shape[-2], 64, sum(splits))]
