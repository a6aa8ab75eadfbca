"""GPU: attention over plain paged caches in an odd number of parts of odd numbers of rows.  Tolerances as in
test_gpu_cache_attention.py."""

from __future__ import annotations

import pytest

from tests.test_gpu_cache_attention import Case, call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (7, 1), (9, 3)])
@pytest.mark.parametrize("length", [1025, 1536, 2300, 3500])
def test_decode_rows(hd, heads, kv_heads, length):
    for batch in (1, 3):
        case = Case(lens=[length, 700, 1300][:batch], heads=heads, kv_heads=kv_heads, hd=hd, seed=length, extra=0)
        case.check(*call(case))


@pytest.mark.parametrize("rows", [1, 3])
def test_any_shape(rows):
    case = Case(lens=[2500], rows=[rows], heads=5, kv_heads=1, hd=40, dtype="fp32", seed=rows)
    case.check(*call(case))
