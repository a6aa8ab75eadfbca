"""GPU: kv_evict_paged_tokens against a plain implementation, byte for byte."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import cache_attention_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BITS = {1: np.uint8, 2: np.uint16, 4: np.uint32}
TYPES = {1: torch.uint8, 2: torch.int16, 4: torch.int32}


class Case:
    def __init__(self, *, lens, keep, layers=2, kv_heads=2, hd=16, bs=16, size=2, tokens=None, seed=0, spare=3, ties=False,
                 index=torch.int32):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.keep, self.index, self.size = np.asarray(lens), np.asarray(keep), index, size
        pages = -(-np.maximum(self.lens, 0) // bs)
        nb = int(pages.sum()) + spare
        order, used = rng.permutation(nb), 0
        self.tables = np.full((len(lens), int(pages.max(initial=0)) + 1), -1, dtype=np.int64)
        for b, k in enumerate(pages):
            self.tables[b, :k] = order[used:used + k]
            used += int(k)
        lead = () if layers is None else (layers,)
        self.cache = [rng.integers(0, 1 << 8 * size, size=(*lead, nb, kv_heads, hd, bs), dtype=BITS[size]) for _ in range(2)]
        tokens = self.tables.shape[1] * bs if tokens is None else tokens
        self.weights = np.exp(2 * rng.normal(size=(*lead, len(lens), kv_heads, tokens))).astype(np.float32)
        if ties:
            self.weights = np.floor(self.weights)

    def tensors(self, dtype=None):
        caches = [torch.from_numpy(c.view(c.dtype.str.replace("u", "i")) if self.size > 1 else c).to(DEV) for c in self.cache]
        return caches, torch.from_numpy(self.weights).to(DEV)

    def index_of(self, x):
        return torch.from_numpy(np.asarray(x, dtype=np.int64)).to(device=DEV, dtype=self.index)

    def check(self, refs=None, **more):
        caches, weights = self.tensors()
        given = {} if refs is None else {"ref_counts": self.index_of(refs)}
        kept = musa_aiter.kv_evict_paged_tokens(*caches, weights, self.index_of(self.tables), self.index_of(self.lens),
                                                self.index_of(self.keep), **given, **more)
        want = [c.copy() for c in self.cache], self.weights.copy()
        layered = self.cache[0].ndim == 5
        for layer in range(self.cache[0].shape[0] if layered else 1):
            pick = (lambda x: x[layer]) if layered else (lambda x: x)
            lens = ref.evict(pick(want[0][0]), pick(want[0][1]), pick(want[1]), self.tables, self.lens, self.keep,
                             refs=refs, **more)
        assert kept.dtype is torch.int64 and kept.tolist() == lens.tolist()
        for got, w in zip(caches, want[0]):
            assert np.array_equal(got.cpu().numpy().view(w.dtype), w)
        assert np.array_equal(weights.cpu().numpy().view(np.uint32), want[1].view(np.uint32))


@pytest.mark.parametrize("size", [1, 2, 4])
@pytest.mark.parametrize("bs", [1, 5, 8, 16, 24, 32, 64, 128])
def test_lengths_and_blocks(size, bs):
    Case(lens=[1, 0, 2, 16, 63, 64, 65, 300, 700], keep=[0, 0, 1, 7, 20, 63, 64, 90, 256], bs=bs, size=size,
         seed=bs).check(sinks=4, recent=10)


@pytest.mark.parametrize("hd", [1, 7, 33, 64, 80, 128, 256])
@pytest.mark.parametrize("layers", [None, 1, 3])
def test_head_dims_and_layers(hd, layers):
    Case(lens=[100, 333, 257], keep=[30, 100, 256], hd=hd, layers=layers, kv_heads=3, seed=hd).check(sinks=3, recent=20)


@pytest.mark.parametrize("sinks,recent", [(0, 0), (0, 1), (1, 0), (200, 5), (5, 200), (10 ** 12, 10 ** 12), (64, 64)])
def test_first_and_last_tokens(sinks, recent):
    case = Case(lens=[300, 300, 70, 128], keep=[100, 1, 69, 128], seed=2)
    case.check(sinks=sinks, recent=recent)


def test_equal_weights_keep_the_earlier():
    for seed in range(3):
        Case(lens=[700, 300], keep=[200, 150], ties=True, seed=seed).check(sinks=2, recent=30)
    case = Case(lens=[1000], keep=[333], seed=4)
    case.weights[:] = 0.0
    case.check(recent=17)


def test_weights_of_every_kind():
    case = Case(lens=[600, 600], keep=[250, 599], seed=5)
    flat = case.weights.reshape(-1)
    kinds = np.asarray([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5, 1e-45, -1e-45, 3e38, 1.0], dtype=np.float32)
    flat[:] = kinds[case.rng.integers(0, len(kinds), size=flat.size)]
    case.check(sinks=1, recent=3)


def test_what_stays_as_it_is():
    case = Case(lens=[300, 90, -7, 64, 200, 5000], keep=[-1, 90, 3, 65, 100, 20], seed=6)
    case.tables[4, 2] = -1
    case.tables[5, 1] = case.cache[0].shape[1]
    case.check(recent=8)
    case = Case(lens=[64, 64], keep=[10, 10], seed=7)
    case.lens = np.asarray([64, 200])  # past the table's room
    case.check()


def test_shared_pages():
    case = Case(lens=[200, 200, 100], keep=[50, 50, 50], seed=8)
    refs = np.ones(case.cache[0].shape[1], dtype=np.int64)
    refs[case.tables[1, 12]] = 2
    refs[case.tables[2, 6]] = 0
    case.check(refs=refs, recent=5)


def test_weights_shorter_than_the_sequences():
    for tokens in (0, 1, 100, 299):
        Case(lens=[300, 40], keep=[120, 20], tokens=tokens, seed=tokens).check(sinks=2, recent=9)


@pytest.mark.parametrize("index", [torch.int16, torch.int32, torch.int64])
def test_index_types(index):
    Case(lens=[300, 40], keep=[120, 20], index=index, seed=1).check(recent=9)


def test_long_rows():
    Case(lens=[20000, 9001], keep=[3000, 9000], layers=None, kv_heads=1, hd=8, seed=11).check(sinks=4, recent=100)


def test_layouts():
    case = Case(lens=[300, 80], keep=[64, 20], seed=12)
    caches, weights = case.tensors()
    want = [c.clone() for c in caches], weights.clone()
    args = [case.index_of(x) for x in (case.tables, case.lens, case.keep)]
    musa_aiter.kv_evict_paged_tokens(*want[0], want[1], *args, recent=7)
    wide = torch.zeros((2, 2 * caches[0].shape[1], *caches[0].shape[2:]), dtype=caches[0].dtype, device=DEV)
    wide[:, ::2] = caches[0]
    far = torch.full((*weights.shape[:-1], 2 * weights.shape[-1]), 5.0, device=DEV)
    far[..., ::2] = weights
    columns = torch.full((2, 2 * case.tables.shape[1]), -1, dtype=torch.int32, device=DEV)
    columns[:, ::2] = args[0]
    musa_aiter.kv_evict_paged_tokens(wide[:, ::2], caches[1], far[..., ::2], columns[:, ::2], *args[1:], recent=7)
    assert torch.equal(wide[:, ::2], want[0][0]) and torch.equal(caches[1], want[0][1])
    assert torch.equal(far[..., ::2], want[1]) and (far[..., 1::2] == 5).all() and (wide[:, 1::2] == 0).all()


def test_nothing_to_do():
    cache = torch.zeros((2, 3, 2, 8, 16), dtype=torch.float16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    kept = musa_aiter.kv_evict_paged_tokens(cache, cache.clone(), torch.zeros((2, 0, 2, 5), device=DEV),
                                            torch.zeros((0, 4), dtype=torch.int32, device=DEV), none, none)
    assert kept.shape == (0,)


@pytest.mark.parametrize("size,hd", [(1, 128), (2, 64), (4, 32)])
@pytest.mark.parametrize("bs", [8, 16, 24, 32, 64, 128])
def test_many_lines(size, hd, bs):
    """512 lines: the form with 16 bytes of dims a wave."""
    Case(lens=[70, 300, 129, 64, 65, 200, 17, 1], keep=[20, 100, 128, 30, 64, 50, 3, 1], layers=8, kv_heads=8, hd=hd, bs=bs,
         size=size, seed=14).check(sinks=2, recent=9)


@pytest.mark.parametrize("size", [1, 2, 4])
@pytest.mark.parametrize("bs,extra", [(8, 7000), (8, 14000), (8, 30000), (64, 1400), (16, 200000)])
def test_long_table_rows(bs, extra, size):
    """Rows whose entries and marks take 70 KiB of LDS and more, up to none that would hold them."""
    case = Case(lens=[500, 77], keep=[200, 30], bs=bs, size=size, seed=bs)
    case.tables = np.concatenate([case.tables, np.full((2, extra), -1, dtype=np.int64)], axis=1)
    case.check(sinks=2, recent=9)


def test_one_dim_more_than_a_slice():
    for size in (1, 2, 4):
        for hd in (4, 5, 12, 36, 100):
            Case(lens=[300], keep=[77], hd=hd, layers=None, size=size, seed=hd).check(recent=5)


def test_dense_and_sparse_marks():
    for size in (1, 2, 4):
        for keep in (1, 5, 64, 128, 1000, 1990, 1999):
            Case(lens=[2000], keep=[keep], layers=None, size=size, seed=keep).check()
    case = Case(lens=[2000], keep=[1000], layers=None, seed=3)
    case.weights[..., ::2] = 1.0
    case.weights[..., 1::2] = 2.0
    case.check()
    case.weights[..., :1000] = 5.0  # nothing moves
    case.check()
