"""GPU: kv_accumulate_attention_weights with many more rows than the window.

The values against a 64-bit implementation (tolerance as in test_gpu_attention_weights.py), and that the work goes by the
window: rows that do not see a position are not gone through for it.
"""

from __future__ import annotations

import pytest
import torch

import musa_aiter
from tests.test_gpu_attention_weights import check, go, prepared
from tests.test_gpu_cache_attention import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hd,heads,kv_heads", [("bf16", 64, 8, 2), ("fp16", 128, 4, 4), ("bf16", 256, 2, 1),
                                                     ("fp32", 64, 2, 1), ("bf16", 40, 3, 3)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (16, 0), (64, 1), (128, 130), (127, 200), (700, 4)])
def test_values(dtype, hd, heads, kv_heads, window, sinks):
    case = Case(lens=[800, 300, 515], rows=[700, 300, 2], heads=heads, kv_heads=kv_heads, hd=hd, dtype=dtype,
                window=window, sinks=sinks, seed=window + hd)
    weights, lse = prepared(case)
    check(case, go(case, weights, lse), weights, lse)


def test_rows_before_the_sequence_and_lengths_past_the_table():
    case = Case(lens=[200, 40, 0], rows=[300, 60, 5], heads=8, hd=128, window=20, sinks=2, seed=3)
    weights, lse = prepared(case)
    check(case, go(case, weights, lse), weights, lse)
    case = Case(lens=[64, 64], rows=[40, 3], hd=64, extra=0, index=torch.int64, window=10, sinks=3, seed=7)
    weights, lse = prepared(case)
    for far in (2 ** 31, 2 ** 40, 2 ** 62):
        case.lens[1] = far
        given = lse.copy()
        given[40:] = 0.0
        out = go(case, weights, given)
        assert torch.isfinite(out).all()
        assert torch.equal(out[1, :, 3:].cpu(), torch.from_numpy(weights)[1, :, 3:])  # the first tokens alone


@pytest.mark.parametrize("dtype,rows,heads,hd", [("bf16", 4096, 32, 128), ("fp32", 768, 8, 64)])
def test_the_work_goes_by_the_window(dtype, rows, heads, hd):
    """A 64th of the scores (a 12th): less than half of the time of the call that sees everything."""
    case = Case(lens=[rows], rows=[rows], heads=heads, kv_heads=heads // 4, hd=hd, dtype=dtype, seed=9)
    query, key, _, tables, lens = case.args()
    weights = torch.zeros((1, heads // 4, rows), device=DEV)
    lse = torch.full((rows, heads), 20.0, device=DEV)
    starts = case.index_of(case.starts)

    def fastest(window):
        times = []
        for _ in range(8):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            musa_aiter.kv_accumulate_attention_weights(weights, query, key, tables, lens, lse, window=window,
                                                       query_starts=starts)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    assert fastest(64) < 0.5 * fastest(None)
