"""GPU: kv_paged_attention and kv_paged_attention_tree against a 64-bit implementation.

Tolerance of an output o_d = sum_j p_j v_jd.  Queries, keys and values enter as they are; what is rounded: the output
once (half a step of its type relative to it), every weight p_j once to the caches' type (half a step of it each, in
all that times sum_j p_j |v_jd|), and the scores in float32.  A score is a sum of head_dim products: its error is at
most (head_dim + 8) * 2^-24 times the sum of their sizes (`spread`), it is taken times log2(e) and to the power of two
in float32 (2^-22 more, relative), and an error d of all scores changes p_j by at most e^(2 d) - 1.  The accumulations
over the tokens add (tokens + 8) * 2^-24 * sum_j p_j |v_jd|.  float16 weights are scaled so that the largest is 2^14: one
below float16's smallest normal value, 2^-14, may be lost, which adds 2^-28 * max_j(p_j) * |v_jd| for every token
(`faint`).  Half a step of float16's smallest values, 2^-25, is the least that its output is off by.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import cache_attention_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def tree_masks(rng, rows, words=1, deep=4):
    """int64 [sum(rows), words]: the bits of each row's ancestors and itself."""
    out = []
    for n in rows:
        seen: list[int] = []
        for i in range(int(n)):
            parent = int(rng.integers(max(-1, i - deep), i)) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        out += [[s >> 64 * w & (1 << 64) - 1 for w in range(words)] for s in seen]
    return np.asarray(out, dtype=np.uint64).reshape(-1, words).view(np.int64)


class Case:
    """Sequences over a shuffled pool; `rows` None is a decode step, `tree` words of masks make the rows a tree."""

    def __init__(self, *, lens, rows=None, heads=4, kv_heads=2, hd=64, bs=16, dtype="bf16", window=None, sinks=0,
                 pad=0, tree=0, seed=0, spare=3, extra=1, index=torch.int32, size=1.0):
        rng = np.random.default_rng(seed)
        self.dtype, self.window, self.sinks, self.index, self.rng = DTYPES[dtype], window, sinks, index, rng
        self.lens = np.asarray(lens, dtype=np.int64)
        pages = -(-np.maximum(self.lens, 0) // bs)
        nb = int(pages.sum()) + spare
        order, used = rng.permutation(nb), 0
        self.tables = np.full((len(lens), int(pages.max(initial=0)) + extra), -1, dtype=np.int64)
        for b, k in enumerate(pages):
            self.tables[b, :k] = order[used:used + k]
            used += int(k)
        channel = np.exp(0.3 * rng.normal(size=(hd, 1)))
        self.cache = [torch.from_numpy((rng.normal(size=(nb, kv_heads, hd, bs)) * channel * size).astype(np.float32))
                      .to(self.dtype) for _ in range(2)]
        self.rows = None if rows is None else np.asarray(rows, dtype=np.int64)
        self.starts = None if rows is None else np.concatenate([[0], np.cumsum(self.rows)])
        total = len(lens) if rows is None else int(self.rows.sum()) + pad
        self.query = torch.from_numpy((1.5 * rng.normal(size=(total, heads, hd))).astype(np.float32)).to(self.dtype)
        self.masks = None
        if tree:
            counts = np.ones(len(lens), dtype=np.int64) if rows is None else self.rows
            masks = tree_masks(rng, counts, tree)
            self.masks = np.concatenate([masks, np.zeros((total - len(masks), tree), dtype=np.int64)])

    def index_of(self, x):
        return torch.from_numpy(np.asarray(x)).to(device=DEV, dtype=self.index)

    def sight(self):
        more = {} if self.starts is None else {"query_starts": self.index_of(self.starts)}
        return more if self.masks is not None else {**more, "window": self.window, "sinks": self.sinks}

    def args(self):
        return [self.query.to(DEV), *(c.to(DEV) for c in self.cache), self.index_of(self.tables),
                self.index_of(self.lens)]

    def expect(self, scale=None):
        return ref.attention(self.query.double().numpy(), *(c.double().numpy() for c in self.cache), self.tables,
                             self.lens, starts=self.starts, scale=scale, window=self.window, sinks=self.sinks,
                             masks=self.masks)

    def check(self, out, lse=None, scale=None):
        want, want_lse, weight, spread, faint = self.expect(scale)
        got = out.double().cpu().numpy()
        hd, tokens = want.shape[2], int(self.lens.max(initial=1))
        mine = ~np.isnan(want_lse)
        step = torch.finfo(self.dtype).eps / 2
        noise = (hd + 8) * 2.0 ** -24 * spread + 2.0 ** -22 * (1 + np.where(np.isfinite(want_lse), np.abs(want_lse), 0))
        bound = step * np.abs(want) + weight * (step * (1 + 2.0 ** -8) + np.expm1(2 * noise) + (tokens + 8) * 2.0 ** -24
                                                )[..., None] * (1 + step) + 2.0 ** -60
        if self.dtype is torch.float16:
            bound += 2.0 ** -28 * (1 + 2.0 ** -8) * faint + 2.0 ** -25
        assert np.isfinite(got[mine]).all()
        off = np.abs(got - want)[mine] - bound[mine]
        assert off.size == 0 or off.max() <= 0, f"{off.max()} past the bound, worst {np.abs(got - want)[mine].max()}"
        if lse is not None:
            g = lse.double().cpu().numpy()
            assert np.isneginf(g[np.isneginf(want_lse) | ~mine]).all()
            full = mine & ~np.isneginf(want_lse)
            assert (np.abs(g[full] - want_lse[full]) <= (noise + (tokens + 8) * 2.0 ** -24 + 2.0 ** -20)[full]).all()
        return got


def call(case, **more):
    args = case.args()
    if case.masks is not None:
        return musa_aiter.kv_paged_attention_tree(*args, torch.from_numpy(case.masks).to(DEV), **case.sight(),
                                                  return_lse=True, **more)
    return musa_aiter.kv_paged_attention(*args, **case.sight(), return_lse=True, **more)


SHAPES = [(64, 16), (128, 16), (128, 64), (96, 32), (256, 16), (128, 8), (128, 24), (192, 16)]
ODD = [(1, 16), (33, 16), (72, 8), (80, 16), (512, 16), (64, 1), (64, 5), (128, 4), (40, 24)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd,bs", SHAPES)
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (4, 4), (5, 1), (40, 2)])
def test_decode_lengths(dtype, hd, bs, heads, kv_heads):
    case = Case(lens=[1, 0, 2, 15, 16, 17, 127, 128, 129, 200, 513], hd=hd, bs=bs, heads=heads, kv_heads=kv_heads,
                dtype=dtype, seed=hd + bs)
    case.check(*call(case))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("hd,bs", ODD)
def test_any_shape(dtype, hd, bs):
    case = Case(lens=[1, 7, 40, 129], rows=[1, 3, 1, 4], hd=hd, bs=bs, dtype=dtype, seed=hd * bs, window=30, sinks=3)
    case.check(*call(case))
    case = Case(lens=[1, 7, 40, 129], rows=[1, 3, 9, 4], hd=hd, bs=bs, dtype=dtype, seed=hd * bs, tree=1)
    case.check(*call(case))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,hd,bs", [(8, 2, 64, 16), (32, 4, 128, 16), (6, 3, 96, 32), (16, 1, 128, 64),
                                                  (2, 2, 256, 16), (40, 2, 64, 16), (4, 2, 128, 8)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (37, 1), (64, 4), (20, 100), (128, 16)])
def test_ragged_rows(dtype, heads, kv_heads, hd, bs, window, sinks):
    case = Case(lens=[5, 260, 33, 0, 700, 64], rows=[5, 17, 1, 0, 40, 2], pad=3, heads=heads, kv_heads=kv_heads, hd=hd,
                bs=bs, dtype=dtype, window=window, sinks=sinks, seed=heads + hd)
    out, lse = call(case)
    case.check(out, lse)
    assert (out[-3:] == 0).all()


@pytest.mark.parametrize("hd,bs", [(128, 16), (64, 64), (96, 16)])
@pytest.mark.parametrize("window,sinks", [(1, 1), (100, 5), (128, 33), (1000, 64), (17, 600)])
def test_decode_windows_and_first_tokens(hd, bs, window, sinks):
    case = Case(lens=[1, 90, 128, 137, 145, 700, 2300], hd=hd, bs=bs, window=window, sinks=sinks, heads=8, seed=window)
    case.check(*call(case))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,hd,bs", [(8, 2, 128, 16), (4, 4, 64, 32), (32, 4, 128, 16), (5, 1, 96, 8)])
def test_trees(dtype, heads, kv_heads, hd, bs):
    case = Case(lens=[70, 20, 130, 700, 1, 33], rows=[64, 20, 1, 65, 1, 9], tree=2, pad=2, heads=heads,
                kv_heads=kv_heads, hd=hd, bs=bs, dtype=dtype, seed=hd)
    case.check(*call(case))
    narrow = Case(lens=[70, 140, 130], rows=[64, 100, 7], tree=1, heads=heads, kv_heads=kv_heads, hd=hd, bs=bs,
                  dtype=dtype, seed=hd + 1)  # drafts past the one word are not seen
    narrow.check(*call(narrow))


def test_any_masks_rows_that_see_nothing_and_rows_before_the_sequence():
    case = Case(lens=[6, 3, 200], rows=[6, 5, 70], tree=2, heads=8, seed=4)  # the second has more rows than tokens
    case.masks = case.rng.integers(-2 ** 63, 2 ** 63, size=case.masks.shape, dtype=np.int64)
    case.masks[2] = 0
    out, lse = call(case)
    case.check(out, lse)
    assert (out[2] == 0).all() and torch.isneginf(lse[2]).all()
    case = Case(lens=[3, 0, -4], rows=[5, 2, 2], heads=8, seed=5)
    case.check(*call(case))


@pytest.mark.parametrize("tree", [0, 1])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_what_is_not_seen_does_not_reach_a_row(tree, dtype):
    """NaN and infinities behind the sequences, in the gap and at positions that only some rows see."""
    clean = Case(lens=[50, 301, 129], rows=[7, 40, 3], heads=8, hd=128, window=None if tree else 70, sinks=5, tree=tree,
                 dtype=dtype, seed=8)
    want, want_lse = call(clean)
    for bad in (float("nan"), float("inf"), float("-inf")):
        case = Case(lens=[50, 301, 129], rows=[7, 40, 3], heads=8, hd=128, window=None if tree else 70, sinks=5,
                    tree=tree, dtype=dtype, seed=8)
        used = np.zeros(case.cache[0].shape[0] * 16, dtype=bool)
        for b, n in enumerate(case.lens):
            j = np.arange(n)
            used[case.tables[b, j // 16] * 16 + j % 16] = True
        free = torch.from_numpy(~used.reshape(-1, 16))[:, None, None]
        for cache in case.cache:
            cache.masked_fill_(free, bad)
        out, lse = call(case)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        # The last token of the second sequence: its last row alone may see it.
        last = 300
        for cache in case.cache:
            cache[case.tables[1, last // 16], :, :, last % 16] = bad
        out, lse = call(case)
        rows = torch.ones(50, dtype=torch.bool)
        sees = [46] if not tree else [t for t in range(7, 47) if case.masks[t, 0] >> 39 & 1]
        rows[sees] = False
        assert torch.isnan(out[sees]).all()
        case.cache = clean.cache
        got = torch.where(rows[:, None, None].to(DEV), out, want)
        case.check(got)


def test_missing_pages_are_not_seen():
    case = Case(lens=[300, 90, 515], rows=[4, 3, 2], heads=8, hd=128, seed=3)
    case.tables[0, 3] = -1
    case.tables[0, 5] = case.cache[0].shape[0]
    case.tables[1, :] = -1
    case.tables[2, 7:20] = 2 ** 31 - 1
    out, lse = call(case)
    case.check(out, lse)
    assert (out[4:7] == 0).all() and torch.isneginf(lse[4:7]).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_softmax_scales(dtype, scale):
    case = Case(lens=[40, 300], rows=[2, 5], hd=64, dtype=dtype, seed=2)
    case.check(*call(case, softmax_scale=scale), scale=scale)


@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** 12])
def test_small_and_large_values(size):
    for dtype in ("bf16", "fp16"):
        case = Case(lens=[1, 40, 700], rows=[1, 2, 40], hd=128, heads=8, dtype=dtype, seed=9)
        case.cache[1] = (case.cache[1].double() * size).to(case.dtype)
        case.check(*call(case))


def test_the_largest_bf16_values_stay_finite():
    case = Case(lens=[3000], hd=64, seed=6)
    case.cache[1] = torch.full_like(case.cache[1], 2.0 ** 127)
    out, _ = call(case)
    assert (out == 2.0 ** 127).all()


@pytest.mark.parametrize("longest", [1, 600, 100000])
def test_lengths_past_max_seq_len_and_far_below_it(longest):
    for window, sinks in ((None, 0), (900, 20)):
        case = Case(lens=[5000, 17, 1300], rows=[3, 2, 1], heads=8, hd=128, window=window, sinks=sinks, seed=1)
        case.check(*call(case, max_seq_len=longest))
    case = Case(lens=[1100, 17, 1300], rows=[50, 2, 64], heads=8, hd=128, tree=1, seed=1)
    case.check(*call(case, max_seq_len=longest))


def test_table_rows_with_much_room():
    case = Case(lens=[300, 5], heads=8, hd=128, extra=4000, seed=12)
    case.check(*call(case))


def test_lengths_past_the_table_and_past_32_bits():
    case = Case(lens=[64, 64, 64], rows=[2, 1, 1], hd=64, extra=0, index=torch.int64, seed=7)
    for far in (65, 1000, 2 ** 31, 2 ** 40, 2 ** 62):
        case.lens = np.asarray([64, far, far])
        args = case.args()
        out, lse = musa_aiter.kv_paged_attention(*args, query_starts=case.index_of(case.starts), return_lse=True)
        # Such rows see all that the table names.
        case.lens = np.asarray([64, 64, 64])
        case.check(out, lse)
        out, lse = musa_aiter.kv_paged_attention(*args, query_starts=case.index_of(case.starts), return_lse=True,
                                                 window=1, sinks=2)
        assert torch.isfinite(lse[2:]).all() and torch.isfinite(out).all()  # the first tokens alone


@pytest.mark.parametrize("index", [torch.int16, torch.int32, torch.int64])
def test_index_types(index):
    case = Case(lens=[100, 30], rows=[3, 2], index=index, seed=3)
    case.check(*call(case))


def test_layouts_of_the_arguments():
    case = Case(lens=[100, 330, 8], rows=[3, 20, 2], heads=8, hd=128, window=90, sinks=7, seed=13)
    args = case.args()
    want, want_lse = musa_aiter.kv_paged_attention(*args, **case.sight(), return_lse=True)
    query, key, value, tables, lens = args
    wide = torch.zeros((25, 16, 256), dtype=query.dtype, device=DEV)
    wide[:, ::2, :128] = query
    far = torch.zeros((key.shape[0], 2, *key.shape[1:]), dtype=key.dtype, device=DEV)
    far[:, 1] = key
    turned = value.transpose(2, 3).contiguous().transpose(2, 3)
    shifted = torch.zeros(key.numel() + 1, dtype=key.dtype, device=DEV)[1:].view(key.shape)  # 2-byte aligned
    shifted.copy_(key)
    columns = torch.full((3, 2 * tables.shape[1]), -1, dtype=tables.dtype, device=DEV)
    columns[:, ::2] = tables
    for q in (query, wide[:, ::2, :128], query.transpose(1, 2).contiguous().transpose(1, 2)):
        for k, v, t in ((far[:, 1], value, tables), (key, turned, columns[:, ::2]), (shifted, value, tables)):
            out, lse = musa_aiter.kv_paged_attention(q, k, v, t, lens, **case.sight(), return_lse=True)
            case.check(out, lse)
    base = torch.full((25, 8, 256), 7.0, dtype=query.dtype, device=DEV)
    given = base[:, :, ::2]
    got = musa_aiter.kv_paged_attention(*args, **case.sight(), out=given)
    assert got is given and torch.equal(got, want) and (base[:, :, 1::2] == 7).all()


def test_loose_rows_are_left_in_a_given_output():
    for tree in (0, 1):
        case = Case(lens=[40, 300], rows=[3, 20], pad=70, heads=8, hd=128, tree=tree, seed=13)
        out = torch.full(case.query.shape, 3.0, dtype=case.dtype, device=DEV)
        got, lse = call(case, out=out)
        assert (got[23:] == 3).all() and torch.isneginf(lse[23:]).all()
        case.check(got, lse)


def test_row_starts_that_are_none():
    case = Case(lens=[40, 300, 20], rows=[3, 20, 5], heads=8, hd=128, seed=14)
    case.starts = np.asarray([3, 0, 20, 50])  # runs backwards, then past the rows
    case.check(*call(case))


def test_no_rows_no_sequences_no_pages():
    empty = torch.zeros((0, 4, 64), dtype=torch.bfloat16, device=DEV)
    cache = torch.zeros((2, 2, 64, 16), dtype=torch.bfloat16, device=DEV)
    none = torch.zeros((0, 3), dtype=torch.int32, device=DEV)
    lens = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert musa_aiter.kv_paged_attention(empty, cache, cache, none, lens).shape == (0, 4, 64)
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device=DEV)
    starts = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = musa_aiter.kv_paged_attention(q, cache, cache, none, lens, query_starts=starts, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    room = torch.zeros((3, 0), dtype=torch.int32, device=DEV)
    out, lse = musa_aiter.kv_paged_attention(q, cache, cache, room, torch.full((3,), 9, device=DEV), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("case_of", [
    lambda: Case(lens=[2000, 13], rows=[1, 1], heads=8, hd=128),
    lambda: Case(lens=[2000, 900], rows=[700, 64], heads=8, hd=128, window=500, sinks=9),
    lambda: Case(lens=[1500, 900], rows=[64, 40], heads=8, hd=128, tree=1)])
def test_the_same_call_gives_the_same_bits(case_of):
    case = case_of()
    one, two = call(case), call(case)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_prompt_rows_over_a_long_prefix():
    case = Case(lens=[1500, 700, 333], rows=[600, 300, 333], heads=8, kv_heads=2, hd=128, seed=21)
    case.check(*call(case))
    case = Case(lens=[1500, 700, 333], rows=[600, 300, 333], heads=4, kv_heads=1, hd=64, window=250, sinks=20,
                dtype="fp16", seed=22)
    case.check(*call(case))


def test_addresses_that_are_no_multiples_of_16():
    case = Case(lens=[100, 330, 8], rows=[3, 20, 2], heads=8, hd=128, window=90, sinks=7, seed=15)
    query, key, value, tables, lens = case.args()

    def odd(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape)
        return flat.copy_(t)

    for args in ((odd(query), key, value), (query, odd(key), value), (query, key, odd(value))):
        case.check(*musa_aiter.kv_paged_attention(*args, tables, lens, **case.sight(), return_lse=True))
    out = odd(query)
    got, lse = musa_aiter.kv_paged_attention(query, key, value, tables, lens, **case.sight(), return_lse=True, out=out)
    assert got is out
    case.check(got, lse)
    plain, moved = (torch.zeros((3, 2, 330), device=DEV) for _ in range(2))
    musa_aiter.kv_accumulate_attention_weights(plain, query, key, tables, lens, lse, **case.sight())
    musa_aiter.kv_accumulate_attention_weights(moved, odd(query), odd(key), tables, lens, odd(lse), **case.sight())
    assert torch.allclose(plain, moved, rtol=1e-5)
