"""CPU: caches that kv_evict_paged_tokens refuses because K and V share memory, and some that only lie between each other."""

from __future__ import annotations

import itertools

import pytest
import torch

import musa_aiter
from musa_aiter.ops.kv_paged_attention import _blocks_meet

L, NB, H, D, BS = 3, 5, 2, 4, 8
BLOCK = H * D * BS


def caches(apart, layer, block, layers=L):
    """K at the beginning of a buffer, V `apart` elements behind it."""
    base = torch.zeros(apart + layers * abs(layer) + NB * block + BLOCK)
    shape, strides = (layers, NB, H, D, BS), (layer, block, D * BS, BS, 1)
    return [base.as_strided(shape, strides, at) for at in (0, apart)]


APART = [("one behind the other", L * NB * BLOCK, NB * BLOCK, BLOCK), ("by layer", NB * BLOCK, 2 * NB * BLOCK, BLOCK),
         ("by block", BLOCK, 2 * NB * BLOCK, 2 * BLOCK), ("with gaps", BLOCK + 3, NB * (2 * BLOCK + 7), 2 * BLOCK + 7)]
SHARED = [("a block on", BLOCK, NB * BLOCK, BLOCK), ("an element on", 1, NB * BLOCK, BLOCK),
          ("a layer on", NB * BLOCK, NB * BLOCK, BLOCK), ("half a block on", BLOCK // 2, 2 * NB * BLOCK, 2 * BLOCK),
          ("the last layer's last block", L * NB * BLOCK - BLOCK, NB * BLOCK, BLOCK)]


def evict(key, value):
    layers = key.shape[0] if key.dim() == 5 else None
    return musa_aiter.kv_evict_paged_tokens(
        key, value, torch.zeros(3, H, 32) if layers is None else torch.zeros(layers, 3, H, 32),
        torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("where,shared", [(x, False) for x in APART] + [(x, True) for x in SHARED], ids=lambda x: str(x)[:24])
def test_stacked(where, shared, turned):
    pair = caches(*where[1:])
    if turned:
        pair.reverse()
    # (Nothing else is wrong with these calls but that the tensors are not on a device.)
    with pytest.raises(*((ValueError,) if shared else (RuntimeError,)), match="share memory" if shared else "ROCm"):
        evict(*pair)


def test_single_layer():
    base = torch.zeros(2 * NB, H, D, BS)
    for key, value, shared in ((base[:NB], base[NB:], False), (base[::2], base[1::2], False),
                               (base[:NB], base[NB - 1:-1], True), (base[:1], base[:2][1:], False)):
        with pytest.raises(ValueError if shared else RuntimeError, match="share memory" if shared else "ROCm"):
            evict(key, value)


def test_against_every_pair_of_blocks():
    for apart, layer, block in itertools.product((1, 5, 63, 64, 65, 130, 200, 333, 700, 1500), (64, 320, 500, 700), (64, 70, 128, 200)):
        pair = caches(apart, layer, block)
        starts = [i * layer + j * block for i in range(L) for j in range(NB)]
        want = any(abs(apart + x - y) < BLOCK for x in starts for y in starts)
        assert _blocks_meet(*pair) is want and _blocks_meet(*reversed(pair)) is want, (apart, layer, block)


def test_strides_of_extents_of_one_do_not_count():
    base = torch.zeros(2 * NB * BLOCK + 2 * BLOCK)
    shape = (1, NB, H, D, BS)
    key = base.as_strided(shape, (7, 2 * BLOCK, D * BS, BS, 1), 0)
    value = base.as_strided(shape, (2 * NB * BLOCK, 2 * BLOCK, D * BS, BS, 1), BLOCK)
    assert not _blocks_meet(key, value)
    assert _blocks_meet(key, base.as_strided(shape, (9, 2 * BLOCK, D * BS, BS, 1), 2 * BLOCK))
    one = torch.zeros(1, 2, NB, H, D, BS)
    with pytest.raises(RuntimeError, match="ROCm"):
        evict(one[:, 0, ::2], one[:, 1, ::2])
