"""GPU: the forms of kv_paged_attention that calls of a certain size take, and their borders.

Calls whose tiles of 16 rows all run at once (512 workgroups of 512 positions) take these; the cases here are larger, and
take tiles of 32 rows (17 to 32 rows a sequence) or of 128 (more), in one part or several.  Tolerances as in
test_gpu_cache_attention.py.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests.test_gpu_cache_attention import DEV, Case, call

pytestmark = pytest.mark.gpu


def at_once(case, longest=None) -> bool:
    """The rule by which a call stays with tiles of 16 rows."""
    kv_heads, group = case.cache[0].shape[1], case.query.shape[1] // case.cache[0].shape[1]
    places = case.tables.shape[1] * case.cache[0].shape[3] if longest is None else longest
    if case.window:
        places = min(places, case.window + -(-16 // group) + 15 + -(-case.sinks // 16) * 16)
    return (case.query.shape[0] * group // 16 + len(case.lens)) * kv_heads * -(-places // 512) <= 512


WIDE = dict(lens=[1300, 64, 700, 0, 130, 950], rows=[200, 64, 129, 0, 1, 100], pad=3, heads=12, kv_heads=3, extra=60)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,bs", [(64, 16), (96, 16), (128, 16), (128, 64), (64, 8), (96, 24), (128, 32)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 9)])
def test_many_rows(dtype, hd, bs, window, sinks):
    case = Case(**WIDE, hd=hd, bs=bs, dtype=dtype, window=window, sinks=sinks, seed=hd + bs)
    assert not at_once(case)
    out, lse = call(case)
    case.check(out, lse)
    assert (out[-3:] == 0).all()
    again = call(case)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd,bs", [(64, 16), (96, 32), (128, 16)])
@pytest.mark.parametrize("group", [1, 3, 4, 8])
def test_many_rows_of_trees(dtype, hd, bs, group):
    case = Case(lens=[1300, 64, 700, 0, 130, 950], rows=[130, 64, 129, 0, 1, 100], pad=3, heads=4 * group, kv_heads=4,
                hd=hd, bs=bs, dtype=dtype, tree=3, extra=200, seed=hd + group)
    assert not at_once(case)
    case.check(*call(case))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tree", [0, 1])
def test_seventeen_to_thirty_two_rows(dtype, hd, tree):
    rng = np.random.default_rng(hd)
    case = Case(lens=rng.integers(9, 200, size=72), rows=rng.integers(4, 9, size=72), heads=32, kv_heads=8, hd=hd,
                dtype=dtype, tree=tree, seed=hd)
    assert not at_once(case)
    case.check(*call(case))


@pytest.mark.parametrize("extra", [40, 200])
@pytest.mark.parametrize("heads,kv_heads", [(64, 1), (40, 2), (130, 1)])
def test_decode_steps_of_wide_groups(heads, kv_heads, extra):
    rng = np.random.default_rng(heads)
    case = Case(lens=rng.integers(0, 300, size=72), heads=heads, kv_heads=kv_heads, hd=64, extra=extra, seed=heads)
    assert not at_once(case)
    case.check(*call(case))


@pytest.mark.parametrize("tree", [0, 2])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_many_rows_and_what_they_do_not_see(tree, dtype):
    def make():
        rows = [128, 64, 100] if tree else [300, 64, 429]
        return Case(lens=[900, 64, 700], rows=rows, heads=12, kv_heads=3, hd=128, extra=100, tree=tree,
                    window=None if tree else 300, sinks=5, dtype=dtype, seed=8)

    clean = make()
    assert not at_once(clean)
    want, want_lse = call(clean)
    clean.check(want, want_lse)
    for bad in (float("nan"), float("inf")):
        case = make()
        used = np.zeros(case.cache[0].shape[0] * 16, dtype=bool)
        for b, n in enumerate(case.lens):
            j = np.arange(n)
            used[case.tables[b, j // 16] * 16 + j % 16] = True
        free = torch.from_numpy(~used.reshape(-1, 16))[:, None, None]
        for cache in case.cache:
            cache.masked_fill_(free, bad)
        out, lse = call(case)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        # A value of the last token, which the last row sees, and in a tree some others.
        case.cache[1][case.tables[0, 899 // 16], 1, 7, 899 % 16] = bad
        out, lse = call(case)
        last = int(case.rows[0]) - 1
        sees = [last] if not tree else [t for t in range(last + 1) if case.masks[t, last // 64] >> (last % 64) & 1]
        assert not torch.isfinite(out[sees][:, 4:8, 7]).any()
        keep = torch.ones(out.shape, dtype=torch.bool, device=DEV)
        for t in sees:
            keep[t, 4:8, 7] = False
        got = torch.where(keep, out, want)
        clean.check(got)
        assert torch.equal(lse, want_lse) or (lse - want_lse)[torch.isfinite(want_lse)].abs().max() < 1e-4


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-40, 0.09])
def test_many_rows_and_scales(scale):
    case = Case(**WIDE, hd=64, seed=3)
    case.check(*call(case, softmax_scale=scale), scale=scale)


@pytest.mark.parametrize("longest", [1, 700, 1300, 10 ** 9])
def test_many_rows_in_parts(longest):
    case = Case(lens=[1300, 64, 700], rows=[200, 64, 129], heads=12, kv_heads=3, hd=64, extra=4000, seed=4)
    case.check(*call(case, max_seq_len=longest))


def test_few_rows_in_many_parts():
    for extra in (10, 3000):
        case = Case(lens=[9000, 700, 1, 5200], rows=[2, 1, 1, 3], heads=8, hd=64, extra=extra, seed=5)
        case.check(*call(case))


def test_rising_scores_move_the_maximum():
    """Keys that grow along the sequence: every tile has a new maximum, in small steps and in large ones."""
    for dtype in ("bf16", "fp16"):
        for rise in (0.002, 0.1):
            case = Case(**WIDE, hd=64, dtype=dtype, seed=6)
            query = torch.ones_like(case.query)
            key = torch.zeros_like(case.cache[0])
            for b, n in enumerate(case.lens):
                j = np.arange(n)
                key[case.tables[b, j // 16], :, 0, j % 16] = (torch.from_numpy(j * rise * 8).to(case.dtype)[:, None])
            case.query, case.cache[0] = query, key
            case.check(*call(case))


def test_sequences_in_blocks_past_32_bits():
    """16-bit caches of more than 2^32 bytes, the last blocks in use."""
    nh, hd, bs = 8, 128, 16
    nb = (1 << 32) // (nh * hd * bs * 2) + 600
    case = Case(lens=[300, 200, 777], rows=[70, 1, 40], heads=32, kv_heads=nh, hd=hd, seed=7, extra=30)
    assert not at_once(case)
    far = torch.arange(nb - case.cache[0].shape[0], nb)
    big = []
    for cache in case.cache:
        t = torch.empty((nb, nh, hd, bs), dtype=case.dtype, device=DEV)
        t[far] = cache.to(DEV)
        big.append(t)
    tables = np.where(case.tables >= 0, case.tables + int(far[0]), -1)
    for more in (dict(query_starts=case.index_of(case.starts)), dict(query_starts=case.index_of(case.starts), window=100)):
        out, lse = musa_aiter.kv_paged_attention(case.query.to(DEV), *big, case.index_of(tables), case.index_of(case.lens),
                                                 return_lse=True, **more)
        case.window = more.get("window")
        case.check(out, lse)
    case.window = None
    weights = torch.zeros((3, nh, 777), device=DEV)
    out, lse = musa_aiter.kv_paged_attention(case.query.to(DEV), *big, case.index_of(tables), case.index_of(case.lens),
                                             return_lse=True, query_starts=case.index_of(case.starts))
    musa_aiter.kv_accumulate_attention_weights(weights, case.query.to(DEV), big[0], case.index_of(tables),
                                               case.index_of(case.lens), lse, query_starts=case.index_of(case.starts))
    assert torch.allclose(weights.sum(2), torch.tensor([70., 1., 40.], device=DEV)[:, None] * 4, rtol=1e-4)
    kept = musa_aiter.kv_evict_paged_tokens(*big, weights, case.index_of(tables), case.index_of(case.lens),
                                            case.index_of([100, 100, 200]), recent=10)
    assert kept.tolist() == [100, 100, 200]
    # The last ten tokens of the first sequence now end at position 99.
    pages = torch.from_numpy(tables[0]).to(DEV)
    j = torch.arange(10, device=DEV)
    new, old = 90 + j, 290 + j
    got = big[1][pages[new // bs], :, :, new % bs]
    want = case.cache[1].to(DEV)[torch.from_numpy(case.tables[0]).to(DEV)[old // bs], :, :, old % bs]
    assert torch.equal(got, want)
