"""GPU: kv_paged_attention_fp8 with scores of every size, and queries of up to 2^100.

All keys of a sequence are equal but one's, which is twice as large: a row's scores s are equal and differ from that
one's by as much as themselves.  So the weights are those of the same rows with queries scaled down to scores of some
thousand (one token's alone, or those of all others alike), and what is rounded beyond them is known: the weights, to at
worst 11 bits, the sums over the tokens, the output.  Equal scores stay equal but for one rounding of their product with
the scales, 2^-24 |s|, which the kernels may leave out, and one of the difference to the running maximum, which is
another 2^-24 |s| at most; two scores then differ by 2^-22 |s| in all, and weights, which are divided by their sum, by a
factor of e^(2^-21 |s|).  Past 2^23 (in base 2) every product is rounded, so equal scores are equal."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import serving_ref as ref
from tests.test_gpu_block_attention import Case

pytestmark = pytest.mark.gpu
FORMS = [dict(lens=[40, 130, 700], hd=64), dict(lens=[5000, 130], hd=128), dict(lens=[40, 130], rows=[3, 5], hd=72),
         dict(lens=[150, 130], rows=[100, 90], hd=64), dict(lens=[150, 130], rows=[100, 90], hd=128),
         dict(lens=[150, 90], rows=[100, 90], hd=72, dtype="fp16"), dict(lens=[40, 130], hd=256),
         dict(lens=[40, 130], rows=[2, 9], hd=64, dtype="fp32")]


def _check(fmt, form, up, key_scale, value_scale=0.01, below=None):
    """Query values of 2^up and a half of it; rows that have scores (in base 2) of `below` and more get smaller ones."""
    case = Case(heads=4, kv_heads=2, seed=30, fmt=fmt, **form)
    rng = np.random.default_rng(2)
    hd = case.query.shape[2]
    signs = torch.from_numpy(rng.choice([-1.0, 0.5, 1.0], size=case.query.shape))
    one = {"e4m3": 7 << 3, "e5m2": 15 << 2}[fmt]  # the code of 1.0, and one exponent
    step = {"e4m3": 1 << 3, "e5m2": 1 << 2}[fmt]
    key = (one + rng.integers(0, step, size=(1, 2, hd, 1))).astype(np.uint8)
    case.cache[0][:] = key
    for b, n in enumerate(case.lens):
        pos = int(n) // 3
        case.cache[0][case.tables[b, pos // 16], :, :, pos % 16] = key[0, :, :, 0] + step
    case.scales[0][:] = key_scale
    case.scales[1] *= value_scale / 0.01
    table = ref.decode_table(fmt)
    score = np.einsum("thd,hd->th", signs.numpy(), np.repeat(table[key[0, :, :, 0]], 2, axis=0))
    if below is not None:
        past = 2 * np.abs(score) * 2.0 ** up * key_scale * hd ** -0.5 * np.log2(np.e) >= below
        signs, score = signs / np.where(past, 16.0, 1.0)[..., None], score / np.where(past, 16.0, 1.0)
    clear = np.abs(score) >= 0.5  # the others' scores nearly cancel
    case.query = (signs * 2.0 ** up).to(case.dtype)
    assert torch.isfinite(case.query).all()
    args, kw = case.args()
    out, lse = musa_aiter.kv_paged_attention_fp8(*args, **kw, return_lse=True)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(got).all()
    exact = case.query.double().numpy()
    case.query = torch.from_numpy(exact * 2.0 ** (16 - up) / key_scale)
    want, want_lse, weight, _, faint = case.expect()
    tokens = int(case.lens.max())
    eps = torch.finfo(case.dtype).eps / 2
    bound = (eps * np.abs(want) + weight * (2.0 ** -11 * (1 + 2.0 ** -8) + (tokens + 8) * 2.0 ** -24)
             + 2.0 ** -28 * (1 + 2.0 ** -8) * faint + 2.0 ** -40 + (2.0 ** -25 if case.dtype is torch.float16 else 0))
    logit = np.abs(score) * 2.0 ** up * key_scale * hd ** -0.5
    bound += weight * np.expm1(np.where(logit * np.log2(np.e) > 2.0 ** 23, 0.0, logit * 2.0 ** -21))[..., None]
    assert (np.abs(got - want) <= bound)[clear].all()
    full = clear & np.isfinite(want_lse)
    with np.errstate(over="ignore"):  # scores past float32 are not asked for
        size = np.abs(exact).sum(axis=2) * 4 * key_scale * hd ** -0.5
    back = 2.0 ** (up - 16) * key_scale
    assert (np.abs(got_lse / back - want_lse)[full] <= ((hd + 16) * 2.0 ** -24 * size / back + np.log(tokens) * (1 + 1 / back))[full]).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("up", [12, 16, 18, 20, 21, 22, 23, 24, 25, 26, 27, 28, 29, 30, 31, 33, 40])
def test_scores_of_every_size(fmt, form, up):
    if form.get("dtype") == "fp16":
        _check(fmt, form, 12, 2.0 ** (up - 12))
    else:
        _check(fmt, form, up, 1.0)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("form", [f for f in FORMS if f.get("dtype") != "fp16"])
@pytest.mark.parametrize("up", [80, 90, 100])
def test_queries_of_the_largest_values(fmt, form, up):
    _check(fmt, form, up, 2.0 ** -60)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("form", FORMS[:5])
@pytest.mark.parametrize("value_scale", [2.0 ** -20, 2.0 ** -8, 0.25])
def test_scores_of_millions_and_value_scales(fmt, form, value_scale):
    for up in (20, 23, 25, 27, 31):
        _check(fmt, form, up, 1.0, value_scale)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("form", [f for f in FORMS if f.get("dtype") != "fp16"])
def test_large_queries_over_blocks_of_zeros(fmt, form):
    """Scores of zero times whatever the queries are."""
    case = Case(heads=4, kv_heads=2, seed=31, fmt=fmt, **form)
    case.query = (case.query.sign() * 2.0 ** 100).to(case.dtype)
    case.scales[0][:] = 0
    args, kw = case.args()
    out, lse = musa_aiter.kv_paged_attention_fp8(*args, **kw, return_lse=True)
    case.check(out, lse)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("form", FORMS[:5])
@pytest.mark.parametrize("value_scale", [64.0, 2.0 ** 30])
def test_large_value_scales_below_the_coarse_scores(fmt, form, value_scale):
    """Scores (in base 2) of up to 2^25 next to value scales of any size."""
    for up in (16, 18, 20, 21, 22):
        _check(fmt, form, up, 1.0, value_scale, below=2.0 ** 25)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("form", [dict(lens=[900, 300], rows=None), dict(lens=[200, 150], rows=[4, 3]),
                                  dict(lens=[900, 300], rows=[100, 90])])
@pytest.mark.parametrize("up", [20, 22, 23, 24, 25, 26])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_differ_by_a_step(fmt, form, up, rising):
    """Scores of 2^up + 0, 2, 4, ...: neighbours in float32, whose differences decide.  Products and sums may be rounded to
    a step, so what is asked of the output is that it lies among the values: a mean of them in 64 bits has no larger size,
    and the rounding adds 2^-7 of it at most (the weights' 2^-11 and the output's 2^-8)."""
    case = Case(heads=2, kv_heads=2, hd=64, seed=33, fmt=fmt, **form)
    one, step = {"e4m3": (7 << 3, 1 << 3), "e5m2": (15 << 2, 1 << 2)}[fmt]
    case.cache[0][:] = 0
    case.cache[0][:, :, 0, :] = one
    for b, n in enumerate(case.lens):
        for pos in range(int(n)):  # 2, 4, 8, 16, ... in this order, or the other way round
            j = pos * 7 // int(n) if rising else 6 - pos * 7 // int(n)
            case.cache[0][case.tables[b, pos // 16], :, 1, pos % 16] = one + (j + 1) * step
    case.query[:] = 0
    case.query[..., 0], case.query[..., 1] = 2.0 ** up, 1.0
    case.scales[0][:] = 1.0
    case.scales[1][:] = 3.5
    args, kw = case.args()
    out, lse = musa_aiter.kv_paged_attention_fp8(*args, **kw, softmax_scale=float(np.log(2.0)), return_lse=True)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all() and torch.isfinite(lse).all()
    assert np.abs(got).max() <= 3.5 * np.abs(ref.decode_table(fmt)).max() * (1 + 2.0 ** -7)
    assert (np.abs(lse.double().cpu().numpy() / np.log(2.0) - 2.0 ** up) <= 300 + 2.0 ** (up - 21)).all()
