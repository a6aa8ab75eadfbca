"""CPU: how many parts an attention call is cut into (0: evenly over the chip), from its sizes alone."""

from __future__ import annotations

import pytest

from musa_aiter.ops import _hip

TURN, TILE = 256, 64  # tokens of a workgroup's turn; parts begin at multiples of a tile


def _splits(*, rows, batch, heads=16, kv_heads=2, hd=64, bs=16, longest, window=0, table=1 << 20, starts=False, dtype=2):
    call = _hip._ATTENTION_CALL.pack(
        16, 16, 0, 16, 16, 16, 16, 16, 16, 16 if starts else 0, 0, 0, rows, batch, heads, kv_heads, hd, bs, 1 << 16,
        table // bs, heads * hd, hd, kv_heads * hd * bs, kv_heads * hd * bs, kv_heads, kv_heads, 1, 1, table // bs, window,
        1, hd ** -0.5, dtype, 1, 0, 0, 0, 1)
    return _hip.fn("musa_aiter_hip_attention_splits")(call, longest)


@pytest.mark.parametrize("window", [1, 64, 1000, 3900])
@pytest.mark.parametrize("batch", [1, 8, 64])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_decode_steps_with_a_window(window, batch, dtype):
    """No row sees more than its window, so all lines are about equally long: parts, and no more than have work."""
    for longest in (8192, 1 << 17, 1 << 29):
        got = _splits(rows=batch, batch=batch, longest=longest, window=window, dtype=dtype)
        assert 1 <= got <= -(-(window + TILE) // TURN)
    assert window != 1 or got == 1


@pytest.mark.parametrize("heads,kv_heads,hd,rows,batch", [(16, 2, 64, 64, 8), (32, 8, 128, 20, 4), (8, 8, 256, 12, 3),
                                                          (32, 8, 128, 600, 2), (4, 4, 64, 700, 1)])
@pytest.mark.parametrize("window", [1, 256, 2000])
def test_rows_with_a_window(heads, kv_heads, hd, rows, batch, window):
    group = heads // kv_heads
    many = -(-rows // batch) * group > 64 and hd <= 128
    size = 128 if many else 32 if hd <= 128 else 16  # rows of a tile, at most
    positions = -(-size // group) + 1
    for longest in (4096, 1 << 16):
        got = _splits(rows=rows, batch=batch, heads=heads, kv_heads=kv_heads, hd=hd, longest=longest, window=window,
                      starts=True)
        assert 1 <= got <= -(-(window + positions + TILE) // TURN)


@pytest.mark.parametrize("starts", [False, True])
@pytest.mark.parametrize("longest", [1, 500, 2000, 9000, 100_000])
def test_windows_that_hide_nothing_change_nothing(starts, longest):
    sizes = dict(rows=24, batch=24, longest=longest, starts=starts)
    plain = _splits(**sizes)
    for window in (longest, longest + 1, 1 << 40, (1 << 63) - 1):
        assert _splits(**sizes, window=window) == plain
    if not starts:
        assert (plain == 0) == (longest > 4096)


def test_long_windows_are_cut_as_sequences_of_their_length():
    sizes = dict(rows=16, batch=16, heads=32, kv_heads=8, hd=128)
    assert _splits(**sizes, longest=1 << 17, window=8192) == 0
    assert _splits(**sizes, longest=1 << 17, window=2000) == _splits(**sizes, longest=2000 + TILE)
