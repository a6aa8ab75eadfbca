"""GPU: evictions from caches that lie between each other in one buffer, and what the calls refuse."""

from __future__ import annotations

import pytest
import torch

import musa_aiter

pytestmark = pytest.mark.gpu


def make(index=torch.int32):
    gen = torch.Generator(device="cuda").manual_seed(3)
    cache = torch.randn((2, 3, 9, 2, 64, 16), generator=gen, device="cuda").to(torch.bfloat16)  # K and V, layers, blocks
    weights = torch.rand((3, 2, 2, 64), generator=gen, device="cuda")
    tables = torch.tensor([[3, 0, 7, 5], [8, 1, 2, 6]], device="cuda", dtype=index)
    lens, keep = (torch.tensor(x, device="cuda", dtype=index) for x in ([61, 33], [20, 17]))
    return cache, weights, tables, lens, keep


@pytest.mark.parametrize("order", [(0, 1, 2), (1, 0, 2), (1, 2, 0)])
def test_one_buffer(order):
    cache, weights, tables, lens, keep = make()
    plain, moved = weights.clone(), weights.clone()
    k, v = cache[0].clone(), cache[1].clone()
    kept = musa_aiter.kv_evict_paged_tokens(k, v, plain, tables, lens, keep, sinks=2, recent=5)
    back = [order.index(i) for i in range(3)]
    mixed = cache.permute(*order, 3, 4, 5).contiguous().permute(*back, 3, 4, 5)
    got = musa_aiter.kv_evict_paged_tokens(mixed[0], mixed[1], moved, tables, lens, keep, sinks=2, recent=5)
    assert kept.tolist() == got.tolist() == [20, 17] and torch.equal(plain, moved)
    assert torch.equal(mixed[0], k) and torch.equal(mixed[1], v)


@pytest.mark.parametrize("index", [torch.int32, torch.int16])  # the host module's checks, and Python's
def test_caches_that_share_blocks_are_refused(index):
    cache, weights, tables, lens, keep = make(index)
    flat = cache.view(-1, 2, 64, 16)
    before = flat.clone()
    for key, value in ((flat[:9], flat[8:17]), (flat[4:13], flat[:9]), (flat[:18:2], flat[2:20:2])):
        with pytest.raises(ValueError, match="share memory"):
            musa_aiter.kv_evict_paged_tokens(key, value, weights[0], tables, lens, keep)
    assert torch.equal(flat, before)
