"""More forks in one call than a grid is high (65535)."""

from __future__ import annotations

import pytest
import torch

from flashattntile_amd import PagedKVCache, fork_sequences

device = pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])


@device
def test_forks_beyond_the_height_of_a_grid(dev):
    print(f"many forks {dev}", flush=True)
    children, P = 65537 + 40, 2
    g = torch.Generator().manual_seed(1)
    pool = children + 2
    k = torch.randn(pool, P, 1, 8, generator=g)
    lens = torch.zeros(children + 1, dtype=torch.int32)
    lens[0] = 3
    table = torch.full((children + 1, 2), -9, dtype=torch.int32)
    table[0] = torch.tensor([5, 1], dtype=torch.int32)
    fresh = torch.tensor([i for i in range(pool) if i not in (1, 5)], dtype=torch.int32)
    cache = PagedKVCache(k.clone().to(dev), (-k).to(dev), table.to(dev), lens.to(dev), P)
    ids = torch.arange(1, children + 1, dtype=torch.int32)
    fork_sequences(cache, torch.zeros(children, dtype=torch.int32).to(dev), ids.to(dev), fresh.to(dev))
    assert bool((cache.seq_lens == 3).all())
    want = torch.stack([torch.full_like(fresh, 5), fresh], dim=1)
    assert torch.equal(cache.page_table[1:].cpu(), want) and cache.page_table[0].tolist() == [5, 1]
    k[fresh.long()] = k[1].clone()
    assert torch.equal(cache.k_cache.cpu(), k) and torch.equal(cache.v_cache.cpu(), -k)
