"""GPU: the page bookkeeping at lengths near the largest that the state's type holds, and at lengths no row can have."""

from __future__ import annotations

import pytest
import torch

import musa_aiter

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 1 << 20


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_lengths_past_the_states_type(dtype):
    """Rows of 2^31 - 10 tokens: ten more are one too many for int32, and nothing is done."""
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GiB of device memory")
    blocks = 2051
    caches = [torch.empty(blocks, 1, 1, PAGE, dtype=torch.uint8, device=DEV) for _ in range(2)]
    first = (1 << 31) - 10
    lens = torch.tensor([first, 0], dtype=dtype, device=DEV)
    refs = (torch.arange(blocks, device=DEV) < 2048).to(dtype)
    tables = torch.full((2, 2050), -1, dtype=dtype, device=DEV)
    tables[0, :2048] = torch.arange(2048, device=DEV)
    state = (tables, lens, refs)
    before = [t.clone() for t in state]

    def extend(n):
        return musa_aiter.kv_extend_paged_sequences(*caches, *state, torch.tensor([n, 1], device=DEV), n)

    slots, left = extend(10)
    if dtype is torch.int32:
        assert int(left) == -(1 << 62) and (slots == -1).all()
        assert all(torch.equal(a, b) for a, b in zip(state, before))
        slots, left = extend(9)
    n = slots.shape[1]
    assert int(left) == 2 and lens.tolist() == [first + n, 1]
    assert slots[0].tolist() == [first + i for i in range(n)]


@pytest.mark.parametrize("length", [(1 << 63) - 1, (1 << 63) - 17, 1 << 62, (1 << 62) + 3])
def test_lengths_that_no_row_can_have(length):
    """A row whose length was overwritten: extend does nothing, free and fork take it for one that owns its whole row."""
    caches = [torch.zeros(12, 1, 4, 16, dtype=torch.uint8, device=DEV) for _ in range(2)]
    lens = torch.tensor([5, length, 20], dtype=torch.int64, device=DEV)
    tables = torch.tensor([[0, -1, -1], [1, 2, 3], [4, 5, -1]], dtype=torch.int64, device=DEV)
    refs = (torch.arange(12, device=DEV) < 6).to(torch.int64)
    state = (tables, lens, refs)
    before = [t.clone() for t in state]
    for new in ([1, 1, 1], [1, 0, 1]):
        slots, left = musa_aiter.kv_extend_paged_sequences(*caches, *state, torch.tensor(new, device=DEV), 3)
        assert int(left) == -(1 << 62) and (slots == -1).all()
        assert all(torch.equal(a, b) for a, b in zip(state, before))
    musa_aiter.kv_fork_paged_sequences(*state, torch.tensor([0, 1, 1], device=DEV), block_size=16)
    assert refs.tolist() == [1, 2, 2, 2, 0, 0] + [0] * 6 and tables[2].tolist() == [1, 2, 3]
    musa_aiter.kv_free_paged_sequences(*state, torch.tensor([-1, 17, 0], device=DEV), block_size=16)
    assert refs.tolist() == [1, 1, 1] + [0] * 9 and lens.tolist() == [5, 17, 0]
    assert tables.tolist() == [[0, -1, -1], [1, 2, -1], [-1, -1, -1]]
