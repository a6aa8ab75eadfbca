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


SIZES = {"any": dict(lens=[40, 3000, 7], rows=[2, 3, 1], heads=2, kv_heads=1, hd=40),
         "few": dict(lens=[40, 3000, 7], rows=[2, 3, 1], heads=8, hd=64),
         "many": dict(lens=[1300, 640, 700], rows=[200, 64, 129], heads=12, kv_heads=3, hd=64, extra=60)}


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -122, 2.0 ** -110, 2.0 ** -98, 2.0 ** 120, 1.5 * 2.0 ** 127])
@pytest.mark.parametrize("form", ["any", "few", "many"])
def test_values_of_every_size(dtype, size, form):
    """One value everywhere: every row's output is that value, be it the smallest normal one or next to the largest.

    What is off: the output's rounding, the sums of weights and of products (tokens + 8) * 2^-24 each, a weight as two
    summands 2^-16, and of a product below float32's smallest normal value 2^-126 what lies under its last place, 2^-149:
    times the tokens, over a sum of weights of at least one.
    """
    case = one_product(Case(**SIZES[form], dtype=dtype, seed=33))
    case.cache[1] = torch.full_like(case.cache[1], size)
    if form == "many":
        assert not at_once(case)
    out, lse = call(case, softmax_scale=1.0)
    _, want_lse, *_ = case.expect(1.0)
    tokens = int(case.lens.max())
    step = torch.finfo(case.dtype).eps / 2
    bound = size * (step + 2.0 ** -16 + 2 * (tokens + 8) * 2.0 ** -24) + tokens * 2.0 ** -149
    off = np.abs(out.double().cpu().numpy() - size)
    assert off.max() <= bound, f"{off.max() / size} of {size}, bound {bound / size}"
    assert np.abs(lse.double().cpu().numpy() - want_lse).max() <= 2.0 ** -19 + (tokens + 8) * 2.0 ** -24


@pytest.mark.parametrize("form", ["any", "few", "many"])
def test_small_and_large_values_side_by_side(form):
    """A dim next to float32's largest values does not cost another its small ones."""
    case = one_product(Case(**SIZES[form], dtype="fp32" if form == "any" else "bf16", seed=34))
    case.cache[1] = torch.full_like(case.cache[1], 2.0 ** -110)
    case.cache[1][:, :, 5] = 1.5 * 2.0 ** 127
    out, _ = call(case, softmax_scale=1.0)
    want = torch.full_like(out, 2.0 ** -110)
    want[:, :, 5] = 1.5 * 2.0 ** 127
    step, tokens = torch.finfo(case.dtype).eps / 2, int(case.lens.max())
    assert ((out.double() / want.double() - 1).abs() <= step + 2.0 ** -16 + 2 * (tokens + 8) * 2.0 ** -24 + tokens * 2.0 ** -39).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("form", ["few", "many"])
@pytest.mark.parametrize("power", [22, 24, 26])
def test_scores_with_coarse_steps(dtype, form, power):
    """Scores of 2^power, where float32 has steps of up to 8 in base 2, all of a row the same: outputs are the means of
    the values, and a logarithm is off by its own rounding and those of the product with the scale and of its ways between
    the bases: 4 * 2^-24."""
    case = Case(**SIZES[form], dtype=dtype, seed=35)
    query, key = torch.zeros_like(case.query), torch.zeros_like(case.cache[0])
    query[:, :, 3] = 64.0
    key[:, :, 3] = 64.0
    case.query, case.cache[0] = query, key
    scale = 2.0 ** (power - 12)
    out, lse = call(case, softmax_scale=scale)
    want, want_lse, weight, *_ = case.expect(scale)
    step, tokens = torch.finfo(case.dtype).eps / 2, int(case.lens.max())
    off = np.abs(out.double().cpu().numpy() - want)
    assert (off <= step * np.abs(want) + weight * (step * step + 2.0 ** -20 + (tokens + 8) * 2.0 ** -23)
            + (2.0 ** -25 if case.dtype is torch.float16 else 0)).all()
    assert (np.abs(lse.double().cpu().numpy() - want_lse) <= 2.0 ** -22 * np.abs(want_lse)).all()
