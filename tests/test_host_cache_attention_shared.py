"""CPU: which tensors share memory, as the operators on plain paged caches ask it."""

from __future__ import annotations

import pytest
import torch

from musa_aiter.ops.kv_block_cache import _spans_meet, _Written


@pytest.mark.parametrize("a,b,meet", [
    ((0, 4), (4, 8), False), ((0, 4), (3, 8), True), ((3, 8), (0, 4), True), ((0, 8), (2, 3), True), ((4, 4), (0, 8), False)])
def test_spans(a, b, meet):
    base = torch.zeros(8, 2, 3)
    assert _spans_meet(base[slice(*a)], base[slice(*b)]) is meet


def test_spans_of_strided_views():
    base = torch.zeros(6, 2, 4, 3)
    assert _spans_meet(base[:, 0], base[:, 1])          # between each other's rows: taken for shared
    assert not _spans_meet(base[0, 0], base[0, 1])
    assert _spans_meet(base[:, 1, :, 2], base[-1, 1, -1, 2:])
    assert not _spans_meet(base, torch.zeros(6))


def test_a_copy_goes_back():
    t = torch.arange(6.0).view(2, 3)
    for fits in (True, False):
        target = _Written(t, fits)
        assert (target.t is t) is fits and torch.equal(target.t, t) and target.t.is_contiguous()
        target.t[1] = 9.0 + fits
        target.finish()
        assert t[1].tolist() == [9.0 + fits] * 3 and t[0].tolist() == [0.0, 1.0, 2.0]
