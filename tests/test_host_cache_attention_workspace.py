"""CPU: the workspace of the attention over plain paged caches.

Its partial outputs are written 16 bytes at a time, so they have to begin at a multiple of 16 behind the pairs of 8 bytes
that stand in front of them, one for each row of each part of each line (a row tile and a kv head).
"""

from __future__ import annotations

import ctypes
import re

import pytest

from musa_aiter.ops import _hip
from tests.test_host_cache_attention import _header


def workspace(**fields) -> int:
    body = re.search(r"typedef struct musa_aiter_hip_paged_attention_call \{(.*?)\}", _header(), re.S).group(1)
    values = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        for field in decl.split(None, 1)[1].split(","):
            name = re.sub(r"[*\[\]\d]|const|void", "", field).split()[-1]
            size = re.search(r"\[(\d+)\]", field)
            for _ in range(int(size.group(1)) if size else 1):
                values.append(float(fields.get(name, 0)) if decl.startswith("double") else fields.get(name, 0))
    return _hip.fn("musa_aiter_hip_paged_attention_workspace")(_hip._CACHE_ATTENTION_CALL.pack(*values))


@pytest.mark.parametrize("batch", [1, 2, 3])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (4, 1), (7, 1), (6, 2), (3, 3)])
@pytest.mark.parametrize("places,parts", [(1536, 3), (2048, 4), (2560, 5), (3584, 7)])
def test_partial_outputs_begin_at_multiples_of_16(batch, heads, kv_heads, places, parts):
    """Decode rows in parts of 512 positions."""
    block = 64 * kv_heads * 16 * 2
    got = workspace(rows=batch, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=64, block_size=16, num_blocks=999,
                    max_blocks=places // 16, cache_block_stride=block, query_row_stride=heads * 64, query_head_stride=64,
                    table_stride=places // 16, longest=places, softmax_scale=0.125, dtype=2)
    lines = batch * kv_heads
    rows = lines * parts * (heads // kv_heads)
    in_front = got - rows * 64 * 4 - lines * 16  # behind the outputs 16 bytes a line
    assert 8 * rows <= in_front < 8 * rows + 16 and in_front % 16 == 0
