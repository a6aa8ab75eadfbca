"""GPU: kv_accumulate_attention_weights against a 64-bit implementation.

Tolerance of weights[b, h, j] = old + sum of e^(s - lse).  A score's error is at most (head_dim + 8) * 2^-24 times the
sum of its products' sizes, the difference to lse and its product with log2(e) are rounded once each, relative to at
most |s| + |lse|, and the power of two adds 2^-22: with `spread` the largest of those sizes plus |lse|, every term's
relative error is below d = expm1((head_dim + 12) * 2^-24 * spread + 2^-22).  n terms are added in float32 in some
order: (n + 1) * 2^-24 of the sum of them and the old value.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import cache_attention_ref as ref
from tests.test_gpu_cache_attention import DEV, ODD, SHAPES, Case

pytestmark = pytest.mark.gpu


def go(case, weights, lse, **more):
    query, key, _, tables, lens = case.args()
    out = torch.from_numpy(weights).to(DEV)
    musa_aiter.kv_accumulate_attention_weights(out, query, key, tables, lens, torch.from_numpy(lse).to(DEV),
                                               **case.sight(), **more)
    return out


def prepared(case, tokens=None):
    """Old weights and the logarithms of the attention."""
    kv_heads = case.cache[0].shape[1]
    tokens = max(int(case.lens.max()), 1) if tokens is None else tokens
    weights = (case.rng.random((len(case.lens), kv_heads, tokens)) ** 4).astype(np.float32)
    lse = case.expect()[1].astype(np.float32)
    return weights, np.where(np.isnan(lse), -np.inf, lse).astype(np.float32)


def check(case, out, weights, lse, scale=None):
    hd = case.query.shape[2]
    want, spread, terms = ref.gathered(weights, case.query.double().numpy(), case.cache[0].double().numpy(),
                                       case.tables, case.lens, lse, starts=case.starts, window=case.window,
                                       sinks=case.sinks, scale=scale)
    got = out.double().cpu().numpy()
    gained = want - weights
    bound = gained * np.expm1((hd + 12) * 2.0 ** -24 * spread + 2.0 ** -22) + (terms + 1) * 2.0 ** -24 * want
    off = np.abs(got - want) - bound * (1 + 2.0 ** -10)
    assert off.max() <= 0, f"{off.max()} past the bound"
    same = terms == 0
    assert np.array_equal(got[same], weights[same].astype(np.float64))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd,bs", SHAPES + ODD)
def test_decode_and_draft_rows(dtype, hd, bs):
    case = Case(lens=[1, 0, 2, 15, 17, 127, 129, 513], hd=hd, bs=bs, heads=8, dtype=dtype, seed=hd)
    weights, lse = prepared(case)
    check(case, go(case, weights, lse), weights, lse)
    case = Case(lens=[40, 0, 300], rows=[3, 0, 9], pad=2, hd=hd, bs=bs, heads=6, window=33, sinks=4, dtype=dtype, seed=hd)
    weights, lse = prepared(case)
    check(case, go(case, weights, lse), weights, lse)


@pytest.mark.parametrize("heads,kv_heads,hd,bs", [(8, 2, 128, 16), (32, 4, 64, 32), (5, 1, 96, 16), (4, 4, 256, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 6)])
def test_prompt_rows(heads, kv_heads, hd, bs, window, sinks):
    case = Case(lens=[400, 70, 900], rows=[130, 70, 33], heads=heads, kv_heads=kv_heads, hd=hd, bs=bs, window=window,
                sinks=sinks, seed=hd)
    weights, lse = prepared(case)
    out = go(case, weights, lse)
    check(case, out, weights, lse)
    assert torch.equal(out, go(case, weights, lse))
    # All that the rows gave: one each, in every head.
    total = (out.double().cpu().numpy() - weights).sum(axis=2)
    assert np.allclose(total, np.asarray([130, 70, 33])[:, None] * heads // kv_heads, rtol=1e-4)


def test_rows_that_give_nothing_and_positions_past_the_weights():
    case = Case(lens=[60, 300], rows=[4, 5], heads=8, hd=128, seed=5)
    for tokens in (0, 1, 37, 299, 500):
        weights, lse = prepared(case, tokens)
        lse[1], lse[6, 3] = -np.inf, -np.inf
        out = go(case, weights, lse)
        if tokens:
            check(case, out, weights, lse)


def test_missing_pages_and_values_that_are_not_seen():
    case = Case(lens=[60, 300], rows=[4, 5], heads=8, hd=128, window=50, sinks=2, seed=5)
    weights, lse = prepared(case)
    case.tables[1, 17] = -1
    case.cache[0][case.tables[1, 5]] = float("nan")     # in the gap
    case.cache[0][case.tables[0, 3], :, :, 12:] = float("inf")  # behind the first sequence
    check_case = go(case, weights, lse)
    case.cache[0] = torch.nan_to_num(case.cache[0], 0.0, 0.0, 0.0)
    check(case, check_case, weights, lse)


@pytest.mark.parametrize("longest", [1, 100, 100000])
def test_max_seq_len_only_cuts(longest):
    case = Case(lens=[2000, 40], rows=[3, 2], heads=8, hd=128, seed=15)
    weights, lse = prepared(case)
    check(case, go(case, weights, lse, max_seq_len=longest), weights, lse)


def test_layouts_and_scale():
    case = Case(lens=[60, 300], rows=[4, 5], heads=8, hd=128, seed=16)
    weights, lse = prepared(case)
    query, key, _, tables, lens = case.args()
    base = torch.full((2, 4, 700), 9.0, device=DEV)
    given = base[:, ::2, 1::2][..., :300]
    given.copy_(torch.from_numpy(weights))
    musa_aiter.kv_accumulate_attention_weights(given, query, key.transpose(2, 3).contiguous().transpose(2, 3), tables, lens,
                                               torch.from_numpy(lse).to(DEV).t().contiguous().t(), **case.sight())
    check(case, given, weights, lse)
    assert (base[:, 1::2] == 9).all() and (base[:, :, ::2] == 9).all()
    lse = lse * 0 + 3.0
    check(case, go(case, weights, lse, softmax_scale=-0.11), weights, lse, scale=-0.11)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,rows", [(64, 30), (128, 30), (128, 5)])
def test_many_positions(dtype, hd, rows):
    """More than 256 workgroups: four waves share positions where there are many rows, or take different ones."""
    case = Case(lens=[900, 870, 1001, 1024, 600, 77], rows=[rows] * 6, heads=16, kv_heads=8, hd=hd, dtype=dtype, seed=hd)
    weights, lse = prepared(case)
    check(case, go(case, weights, lse), weights, lse)
