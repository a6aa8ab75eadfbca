"""GPU: kv_paged_attention_fp8 at the borders of its forms: prompt chunks' 128-row tiles, the decode step's even cut,
and calls that the host module hands to the Python checks.  Tolerances: see test_gpu_block_attention."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from musa_aiter.ops import _hip
from tests.test_gpu_block_attention import DEV, Case, _go

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,dtype", [("e4m3", "bf16"), ("e4m3", "fp16"), ("e5m2", "bf16"), ("e5m2", "fp16")])
@pytest.mark.parametrize("hd", [8, 64, 72, 96, 128])
@pytest.mark.parametrize("rows", [65, 127, 128, 129, 260])
def test_rows_around_a_tile(rows, hd, fmt, dtype):
    case = Case(lens=[rows + 3], rows=[rows], heads=1, kv_heads=1, hd=hd, fmt=fmt, dtype=dtype, seed=rows + hd)
    case.check(*_go(case))


@pytest.mark.parametrize("group", [1, 3, 40, 130])
@pytest.mark.parametrize("window", [None, 1, 50, 1000])
def test_groups_and_windows_of_chunks(group, window):
    case = Case(lens=[200, 64, 0, 1, 63, 130], rows=[100, 64, 0, 1, 65, 130], heads=2 * group, kv_heads=2, hd=64,
                bs=32, window=window, pad=5, seed=group, index=torch.int64)
    out, lse = _go(case)
    case.check(out, lse)
    assert (out[-5:] == 0).all() and torch.isneginf(lse[-5:]).all()


@pytest.mark.parametrize("hd,fmt", [(64, "e4m3"), (128, "e4m3"), (128, "e5m2")])
@pytest.mark.parametrize("bs", [16, 48, 64])
def test_chunks_of_long_sequences_in_parts(hd, fmt, bs):
    case = Case(lens=[4000, 777, 2049], rows=[40, 40, 33], heads=8, kv_heads=2, hd=hd, fmt=fmt, bs=bs, seed=hd, extra=7)
    out, lse = _go(case)
    case.check(out, lse)
    for longest in (1, 1000, 1 << 40):
        case.check(*_go(case, max_seq_len=longest))
    windowed = Case(lens=[4000, 777, 2049], rows=[40, 40, 33], heads=8, kv_heads=2, hd=hd, fmt=fmt, bs=bs, window=300,
                    seed=hd)
    windowed.check(*_go(windowed))


def test_chunks_with_blocks_outside_the_cache():
    for index in (torch.int32, torch.int64):
        case = Case(lens=[300, 128], rows=[120, 90], heads=4, kv_heads=2, hd=128, seed=3, index=index)
        nb = case.cache[0].shape[0]
        case.tables[0, 2:5], case.tables[1, :] = -1, nb
        if index is torch.int64:
            case.tables[0, 7] = (1 << 32) + 1  # its low half is a block
        out, lse = _go(case)
        case.check(out, lse)
        assert (out[120:] == 0).all() and torch.isneginf(lse[120:]).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_chunks_with_scales_of_every_size(fmt):
    case = Case(lens=[300, 160], rows=[100, 160], heads=4, kv_heads=2, hd=128, seed=10, fmt=fmt)
    rng = np.random.default_rng(1)
    shape = case.scales[1].shape
    case.scales[1][:] = (2.0 ** rng.integers(-58, 40, size=shape)).astype(np.float32)
    case.scales[1][rng.random(shape) < 0.2] = 0
    case.scales[0][rng.random(shape) < 0.2] = 0
    case.check(*_go(case))


@pytest.mark.parametrize("size,scale", [(1e4, 1e-4), (3.0, 0.0), (1.0, -0.2), (1e-6, 1e5), (30.0, 1.0)])
def test_chunks_with_large_and_small_scores(size, scale):
    case = Case(lens=[230, 130], rows=[100, 70], heads=4, kv_heads=2, hd=64, seed=12)
    case.query = (case.query.float() * size).to(case.dtype)
    args, kw = case.args()
    out, lse = musa_aiter.kv_paged_attention_fp8(*args, **kw, softmax_scale=scale, return_lse=True)
    case.check(out, lse, scale=scale)


def test_a_maximum_that_grows_with_every_tile():
    """Scores that rise over the sequence: the weights' reference follows them by steps."""
    case = Case(lens=[900], rows=[70], heads=2, kv_heads=2, hd=64, seed=5, codes="kept")
    case.query = case.query.abs()
    for block in range(case.tables.shape[1] - 1):
        at = case.tables[0, block]
        case.cache[0][at] &= 0x7F
        case.scales[0][at] = 1e-4 * (block + 1)
    case.check(*_go(case))


def test_nan_and_infinite_queries_of_chunks_stay_in_their_rows():
    case = Case(lens=[150, 160], rows=[100, 90], heads=4, kv_heads=2, seed=13)
    clean, _ = _go(case)
    case.query[2, 3, 5] = float("nan")
    case.query[120, 1, 0] = float("inf")
    out, _ = _go(case)
    assert torch.isnan(out[2, 3]).all() and torch.isnan(out[120, 1]).any()
    keep = torch.ones(190, 4, dtype=torch.bool, device=DEV)
    keep[2, 3] = keep[120, 1] = False
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("offset", [1, 4, 8])
def test_chunks_of_queries_at_other_addresses(offset):
    case = Case(lens=[150, 160], rows=[100, 90], heads=4, kv_heads=2, hd=128, seed=14)
    want, _ = _go(case)
    args, kw = case.args()
    loose = torch.zeros(args[0].numel() + 16, dtype=args[0].dtype, device=DEV)
    at = loose[offset:offset + args[0].numel()].view(args[0].shape)
    at.copy_(args[0])
    out = torch.zeros_like(loose)[offset:offset + want.numel()].view(want.shape)
    got = musa_aiter.kv_paged_attention_fp8(at, *args[1:], **kw, out=out)
    assert got is out and torch.equal(out, want)


@pytest.mark.parametrize("lens,rows", [([700, 90, 1300], None), ([60, 20], None), ([900, 700], [3, 5]), ([300, 300], [90, 80])])
def test_output_in_place_of_the_query(lens, rows):
    case = Case(lens=lens, rows=rows, heads=8, kv_heads=2, hd=128, seed=15)
    want, _ = _go(case)
    args, kw = case.args()
    got = musa_aiter.kv_paged_attention_fp8(*args, **kw, out=args[0])
    assert got is args[0] and torch.equal(got, want)


def test_chunks_captured_and_replayed():
    case = Case(lens=[1500, 1200], rows=[150, 40], heads=8, kv_heads=2, hd=128, seed=16)
    args, kw = case.args()
    musa_aiter.kv_paged_attention_fp8(*args, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = musa_aiter.kv_paged_attention_fp8(*args, **kw, return_lse=True)
    for rep in range(3):
        args[0].copy_(torch.randn(args[0].shape))
        args[4].sub_(rep * 31)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = musa_aiter.kv_paged_attention_fp8(*args, **kw, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), rep


@pytest.mark.parametrize("hd,fmt,dtype", [(40, "e4m3", "bf16"), (64, "e5m2", "bf16"), (96, "e4m3", "fp16"),
                                          (100, "e5m2", "fp16"), (128, "e5m2", "fp16"), (256, "e4m3", "bf16")])
@pytest.mark.parametrize("window", [None, 1, 400])
@pytest.mark.parametrize("heads", [3, 40])
def test_even_cut(hd, fmt, dtype, window, heads):
    lens = [0, 1, 2500, 64, 0, 513, 0]
    case = Case(lens=lens, heads=heads, kv_heads=1, hd=hd, fmt=fmt, dtype=dtype, window=window, seed=hd, index=torch.int64)
    case.check(*_go(case, max_seq_len=1 << 20))  # a hint: decode steps of long sequences are cut evenly
    case.check(*_go(case, max_seq_len=2500))


@pytest.mark.parametrize("batch,longest", [(1, 9000), (70, 700), (200, 530)])
def test_even_cut_of_few_and_many_sequences(batch, longest):
    rng = np.random.default_rng(batch)
    lens = rng.integers(0, longest, size=batch)
    lens[-1] = longest
    case = Case(lens=lens, heads=8, kv_heads=4, hd=64, seed=batch)
    case.check(*_go(case, max_seq_len=1 << 20))
    case.check(*_go(case))


@pytest.mark.parametrize("lens,rows", [([700, 90], None), ([60, 20], None), ([300, 300], [90, 80])])
def test_python_checks_give_the_same(monkeypatch, lens, rows):
    case = Case(lens=lens, rows=rows, heads=8, kv_heads=2, hd=128, seed=17)
    want = _go(case)
    monkeypatch.setattr(_hip, "attention_native", lambda *a: None)
    got = _go(case)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_places_past_32_bits():
    """A cache of more than 2^32 bytes whose last blocks are read: decode, drafts and a chunk."""
    nb, kv_heads, hd, bs = 70_000, 8, 128, 64
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GiB of device memory")
    for rows in ([1, 1], [4, 5], [70, 40]):
        case = Case(lens=[300, 700], rows=rows, heads=16, kv_heads=kv_heads, hd=hd, bs=bs, seed=18)
        want, _ = _go(case)
        args, kw = case.args()
        shift = nb - case.cache[0].shape[0]
        big = []
        for i in (1, 2):
            c = torch.empty(nb, kv_heads, hd, bs, dtype=torch.uint8, device=DEV)
            c[shift:] = args[i]
            big.append(c)
        scales = []
        for i in (5, 6):
            s = torch.zeros(nb, kv_heads, device=DEV)
            s[shift:] = args[i]
            scales.append(s)
        tables = torch.where(args[3] >= 0, args[3] + shift, -1)
        got = musa_aiter.kv_paged_attention_fp8(args[0], *big, tables, args[4], *scales, **kw)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del big, c


def test_even_cut_captured_and_replayed_on_two_streams():
    case = Case(lens=[700, 1300, 20, 0, 5000], heads=8, kv_heads=2, hd=128, seed=19)
    args, kw = case.args()
    musa_aiter.kv_paged_attention_fp8(*args, **kw)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(musa_aiter.kv_paged_attention_fp8(*args, **kw, return_lse=True))
        graphs.append(graph)
    for rep in range(3):
        args[0].copy_(torch.randn(args[0].shape))
        args[4].copy_(torch.from_numpy(np.maximum(case.lens - 31 * rep, 0)))
        torch.cuda.synchronize()
        for graph in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.replay()
        torch.cuda.synchronize()
        want = musa_aiter.kv_paged_attention_fp8(*args, **kw, return_lse=True)
        for got in outs:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), rep
