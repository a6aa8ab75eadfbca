"""GPU: kv_accumulate_attention_weights at scores and logarithms of every size, to the bits that float32 holds."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import cache_attention_ref as ref
from tests.test_gpu_cache_attention import DEV, Case

pytestmark = pytest.mark.gpu


def gather(case, lse, scale):
    query, key, _, tables, lens = case.args()
    out = torch.zeros((len(case.lens), key.shape[1], int(case.lens.max())), device=DEV)
    musa_aiter.kv_accumulate_attention_weights(out, query, key, tables, lens, torch.from_numpy(lse).to(DEV),
                                               softmax_scale=scale, **case.sight())
    return out.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [[1, 3, 2], [40, 9, 70]])
@pytest.mark.parametrize("scale", [0.125, -0.125, 128 ** -0.5])
@pytest.mark.parametrize("size", [1, 64, 4096])
def test_gathered_weights_of_large_scores(dtype, rows, scale, size):
    """weights[j] = sum of e^(s_j - lse) with scores of up to 2048 * size / 4, and logarithms given as float32.

    Dots are exact (two products of small integers).  The difference s - lse, d in size, is made with two roundings of it
    at most, its product with log2(e), itself a rounded number, with one: 4 * 2^-24 d is past their sum.  The power of two
    and one of the logarithm's rest give 2^-22 each, n terms add (n + 1) * 2^-24.
    """
    case = Case(lens=[50, 301, 129], rows=rows, heads=8, kv_heads=2, hd=64, dtype=dtype, seed=36)
    query, key = torch.zeros_like(case.query), torch.zeros_like(case.cache[0])
    query[:, :, 3], query[:, :, 40] = 64.0, 1.0
    key[:, :, 3] = float(size)
    nb, nh, _, bs = key.shape
    key[:, :, 40] = torch.from_numpy(case.rng.integers(-60, 60, size=(nb, nh, bs)).astype(np.float32)).to(case.dtype)
    case.query, case.cache[0] = query, key
    lse = case.expect(scale)[1].astype(np.float32)
    got = gather(case, lse, scale)
    want, most = np.zeros_like(got), np.zeros_like(got)
    terms = np.zeros_like(got)
    for t, g, h, b, at, s, _, _ in ref.Rows(query.double().numpy(), key.double().numpy(), key.double().numpy(), case.tables,
                                            case.lens, starts=case.starts, scale=scale).each():
        d = s - float(lse[t, g])
        want[b, h, at] += np.exp(d)
        most[b, h, at] += np.exp(d) * np.expm1(2.0 ** -22 * np.abs(d) + 2.0 ** -21)
        terms[b, h, at] += 1
    assert (np.abs(got - want) <= most + (terms + 1) * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("lse", [float("inf"), float("-inf"), float("nan"), 3.0e38])
@pytest.mark.parametrize("rows", [[1, 3, 2], [40, 9, 70]])
def test_gathered_weights_of_logarithms_that_are_none(lse, rows):
    case = Case(lens=[50, 301, 129], rows=rows, heads=8, kv_heads=2, hd=64, seed=37)
    given = np.zeros((int(sum(rows)), 8), dtype=np.float32)
    given[:] = case.expect()[1]
    want = gather(case, given, None)
    given[0] = lse  # of the first sequence
    got = gather(case, given, None)
    assert np.array_equal(got[1:], want[1:])
    assert np.isnan(got[0, :, 0]).all() if np.isnan(lse) else np.isfinite(got).all() and (got[0] <= want[0]).all()


@pytest.mark.parametrize("dtype,hd", [("fp32", 64), ("bf16", 40), ("bf16", 64), ("fp16", 128)])
@pytest.mark.parametrize("scale", [0.125, 40 ** -0.5, -0.3])
@pytest.mark.parametrize("rows", [[1, 3, 2], [40, 9, 70]])
def test_gathered_weights_of_infinite_scores(dtype, hd, scale, rows):
    """Keys that make a score -inf gather nothing; one of +inf makes its position's sum infinite, and no other."""
    case = Case(lens=[50, 301, 129], rows=rows, heads=8, kv_heads=2, hd=hd, dtype=dtype, seed=38)
    case.query[:, :, 3] = 1.0
    lse = case.expect(scale)[1].astype(np.float32)
    want = gather(case, lse, scale)
    sign = 1.0 if scale > 0 else -1.0
    for at, value in ((7, -np.inf), (40, np.inf)):
        case.cache[0][case.tables[0, at // 16], 1, 3, at % 16] = sign * value
    got = gather(case, lse, scale)
    assert got[0, 1, 7] == 0.0 and np.isposinf(got[0, 1, 40])
    same = np.ones(want.shape, dtype=bool)
    same[0, 1, [7, 40]] = False
    assert np.array_equal(got[same], want[same])
