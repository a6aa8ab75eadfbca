"""GPU: what kv_paged_attention_fp8 leaves for rows that belong to no sequence: `out` as it was where the caller gives one,
and in every case -inf for their logarithms."""

from __future__ import annotations

import pytest
import torch

import musa_aiter
from tests.test_gpu_block_attention import DEV, Case

pytestmark = pytest.mark.gpu

# One call for each form: 16 and 32 rows a wave, parts, prompt chunks (whole, by elements, in parts), any shape.
FORMS = [
    dict(lens=[70, 0, 40], rows=[1, 0, 1], hd=64),
    dict(lens=[70, 0, 40], rows=[5, 0, 3], heads=16, hd=128),
    dict(lens=[3000, 900], rows=[2, 2], hd=64),
    dict(lens=[200, 90], rows=[80, 70], hd=128),
    dict(lens=[200, 90], rows=[80, 70], hd=72),
    dict(lens=[4000, 777], rows=[70, 40], heads=8, hd=64),
    dict(lens=[60, 33], rows=[2, 4], hd=64, dtype="fp32"),
    dict(lens=[2000, 33], rows=[2, 4], hd=33, dtype="fp32", bs=5),
    dict(lens=[60, 33], rows=[0, 0], hd=64),
]


def _poison(rows: int, heads: int) -> None:
    """Leaves NaN in the memory that the next tensors of [rows, heads] floats are likely to get."""
    held = [torch.full((rows, heads), float("nan"), device=DEV) for _ in range(16)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("layout", ["new", "given", "transposed"])
def test_logarithms_of_rows_of_no_sequence(form, layout):
    case = Case(pad=5, seed=3, **form)
    args, kw = case.args()
    kw["query_starts"] = kw["query_starts"] + 2  # two rows in front of the sequences, three behind them
    rows, heads, hd = args[0].shape
    loose = torch.ones(rows, dtype=torch.bool, device=DEV)
    loose[2:2 + int(case.rows.sum())] = False
    out = None
    if layout == "given":
        out = torch.full_like(args[0], 7.0)
    elif layout == "transposed":
        out = torch.full((rows, hd, heads), 7.0, dtype=case.dtype, device=DEV).transpose(1, 2)
    _poison(rows, heads)
    got, lse = musa_aiter.kv_paged_attention_fp8(*args, **kw, out=out, return_lse=True)
    torch.cuda.synchronize()
    assert torch.isneginf(lse[loose]).all()
    assert (got[loose] == (0 if out is None else 7)).all()
    assert not torch.isnan(lse).any() and torch.isfinite(got[~loose].float()).all()
    case.starts = case.starts + 2
    case.check(got, lse)


def test_no_sequences_with_a_given_output():
    case = Case(lens=[5], seed=1)
    args, _ = case.args()
    starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(args[0], 7.0)
    _poison(*args[0].shape[:2])
    got, lse = musa_aiter.kv_paged_attention_fp8(args[0], *args[1:3], args[3][:0], args[4][:0], *args[5:],
                                                 query_starts=starts, out=out, return_lse=True)
    assert got is out and (out == 7).all() and torch.isneginf(lse).all()
