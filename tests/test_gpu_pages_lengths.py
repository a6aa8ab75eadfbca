"""GPU: kv_extend_paged_sequences at lengths near the largest that the state's type holds."""

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
