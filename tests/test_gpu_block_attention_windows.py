"""GPU: kv_paged_attention_fp8 with a window reads nothing into its result from pages that lie in front of it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests.test_gpu_block_attention import Case, _go

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -1.0, 3e38])
@pytest.mark.parametrize("form", [
    dict(lens=[200, 130, 61], hd=64),
    dict(lens=[200, 130, 61], hd=128, fmt="e5m2"),
    dict(lens=[200, 130, 61], hd=40, dtype="fp16"),
    dict(lens=[200, 130, 61], hd=256),
    dict(lens=[200, 130, 61], hd=64, dtype="fp32"),
    dict(lens=[200, 130, 61], rows=[3, 1, 4], heads=16, hd=128),
    dict(lens=[250, 190], rows=[70, 66], hd=64),
    dict(lens=[250, 190], rows=[70, 66], hd=128, dtype="fp16", fmt="e5m2"),
    dict(lens=[250, 190], rows=[70, 66], hd=96),
    dict(lens=[5000, 900], hd=64, bs=32),
    dict(lens=[2000, 900], rows=[2, 3], hd=64),
])
@pytest.mark.parametrize("window", [1, 37])
def test_scales_of_pages_in_front_of_the_window(form, window, odd):
    """Such pages may belong to others or to nobody by then: whatever their scales are, the rows do not see them."""
    case = Case(window=window, seed=5, **form)
    bs = case.cache[0].shape[-1]
    calls = [{}, {"max_seq_len": 1 << 20}]
    clean = [_go(case, **more) for more in calls]
    case.check(*clean[0])
    count = case.rows if case.rows is not None else np.ones(len(case.lens), dtype=np.int64)
    begin = np.maximum(case.lens - count - window + 1, 0)  # the first position that any row of a sequence sees
    hidden = 0
    for b, first in enumerate(begin):
        for s in case.scales:
            s[case.tables[b, :first // bs]] = odd
        hidden += int(first // bs)
    assert hidden > 0
    for more, (want, want_lse) in zip(calls, clean):
        out, lse = _go(case, **more)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
