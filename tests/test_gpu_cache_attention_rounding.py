"""GPU: how many bits the forms of the plain-cache operators hold, at values and scores where too few would show.

Queries have one dim that is not zero, and it is a small power of two or a small integer, as the keys' are: every score is
exact in float32 (one product), so that `spread` of test_gpu_cache_attention.py is the score itself and its error comes
from the product with the scale, the difference to the maximum and the power of two: 2^-22 * (4 + |score|) is past the
sum of these (three roundings of 2^-24 relative to the score or its maximum, in both of which |score| is the largest of
the row, and 2^-22 of the power).

A weight that is held as two summands of a 16-bit type is off by half a step squared: 2^-16 (bf16), 2^-22 (fp16).  What
lies below float16's smallest normal value may be lost in either summand: 2 * 2^-28 of the row's largest weight (`faint`).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.test_gpu_cache_attention import Case, call
from tests.test_gpu_cache_attention_forms import at_once

pytestmark = pytest.mark.gpu


def one_product(case, top=16):
    """Scores of one product: integers in [0, top) over 8."""
    query, key = torch.zeros_like(case.query), torch.zeros_like(case.cache[0])
    query[:, :, 3] = 1.0
    nb, nh, _, bs = key.shape
    key[:, :, 3] = torch.from_numpy(case.rng.integers(0, top, size=(nb, nh, bs)) / 8.0).to(case.dtype)
    case.query, case.cache[0] = query, key
    return case


def check_two_summands(case, out):
    want, want_lse, weight, _, faint = case.expect(1.0)
    got = out.double().cpu().numpy()
    mine = np.isfinite(want_lse)
    step, largest = torch.finfo(case.dtype).eps / 2, 2.0
    tokens = np.concatenate([n - k + 1 + np.arange(k) for n, k in zip(case.lens, case.rows)])[:, None, None]  # at most
    noise = 2.0 ** -22 * (4 + largest)
    bound = step * np.abs(want) + weight * (step * step + np.expm1(2 * noise) + (tokens + 8) * 2.0 ** -24) * (1 + step)
    if case.dtype is torch.float16:
        bound += 2 * 2.0 ** -28 * (1 + 2.0 ** -8) * faint + 2.0 ** -25
    off = np.abs(got - want)[mine] - bound[mine]
    assert off.max() <= 0, f"{off.max()} past the bound, worst {np.abs(got - want)[mine].max()}"


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("tree", [0, 1])
def test_a_row_keeps_its_bits_whatever_its_neighbours(dtype, hd, tree):
    """The same rows in a call of many rows, and of few: a weight is held as two summands in both."""
    def make(rows, lens):
        return one_product(Case(lens=lens, rows=rows, heads=12, kv_heads=3, hd=hd, dtype=dtype, tree=3 * tree, extra=60,
                                seed=31))

    many, few = make([150, 64, 129, 130], [1300, 64, 135, 130]), make([5, 4, 3, 3], [5, 64, 4, 3])
    assert not at_once(many)
    for case in (many, few):
        check_two_summands(case, call(case, softmax_scale=1.0)[0])
