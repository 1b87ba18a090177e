"""Host side of shared-prefix decode: buffers that a caller of the launch without
validation brings along, and the partials of a launch (no GPU needed)."""

from __future__ import annotations

import pytest
import torch

from flashattntile_amd import PagedKVCache
from flashattntile_amd.kernels.shared import paged_decode_shared_launch


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
