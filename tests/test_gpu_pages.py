"""GPU: the page bookkeeping (extend, fork, free, compact) against a step-by-step implementation, exactly; and a
run of all the operators of a block-scaled cache together."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Pool:
    """Random state on the device and the same on the host."""

    def __init__(self, rng, *, batch, page, blocks, longest, dtype=torch.int32, layers=2, share=0.0, extra=3,
                 cache=torch.uint8, scales=True, inner=(2, 8)):
        lens = rng.integers(0, longest + 1, size=batch)
        width = -(-longest // page) + extra
        tables, refs = np.full((batch, width), -1, dtype=np.int64), np.zeros(blocks, dtype=np.int64)
        order, used = rng.permutation(blocks), 0
        for b in range(batch):
            if b and rng.random() < share:  # shares a prefix with an earlier row, partial page and all
                o = int(rng.integers(0, b))
                lens[b] = min(lens[b], lens[o])
                own = -(-int(lens[b]) // page)
                tables[b, :own] = tables[o, :own]
            else:
                own = -(-int(lens[b]) // page)
                assert used + own <= blocks
                tables[b, :own] = order[used:used + own]
                used += own
            np.add.at(refs, tables[b, :own], 1)
        self.page, self.layers = page, layers
        shape = ((layers,) if layers else ()) + (blocks, *inner, page)
        self.caches = [torch.randint(0, 200, shape, device=DEV).to(cache) for _ in range(2)]
        self.scales = [torch.rand(shape[:-2], device=DEV) for _ in range(2)] if scales else [None, None]
        self.start(tables, lens, refs, dtype)

    def start(self, tables, lens, refs, dtype):
        self.host = ref.Pages(tables, lens, refs, self.page)
        self.tables, self.lens, self.refs = (torch.from_numpy(np.asarray(x)).to(device=DEV, dtype=dtype)
                                             for x in (tables, lens, refs))
        self.state = (self.tables, self.lens, self.refs)
        self.want = [t.clone() for t in self.caches + self.scales if t is not None]

    def kw(self):
        return {} if self.scales[0] is None else {"k_scales": self.scales[0], "v_scales": self.scales[1]}

    def extend(self, new, most):
        rows = torch.tensor(new, device=DEV)
        slots, left = musa_aiter.kv_extend_paged_sequences(*self.caches, *self.state, rows, most, **self.kw())
        want, want_left = self.host.extend(new, most)
        assert slots.tolist() == want and int(left) == want_left
        self.check()
        return slots

    def fork(self, parents):
        musa_aiter.kv_fork_paged_sequences(*self.state, torch.tensor(parents, device=DEV), block_size=self.page)
        self.host.fork(parents)
        self.check()

    def free(self, keep):
        musa_aiter.kv_free_paged_sequences(*self.state, torch.tensor(keep, device=DEV), block_size=self.page)
        self.host.free(keep)
        self.check()

    def compact(self):
        count = musa_aiter.kv_compact_paged_blocks(*self.caches, self.tables, self.refs, **self.kw())
        assert int(count) == self.host.compact()
        self.check()

    def check(self):
        assert self.tables.tolist() == self.host.tables
        assert self.lens.tolist() == self.host.lens
        assert self.refs.tolist() == self.host.refs
        for src, dst in self.host.moves:
            for t in self.want:
                if self.layers:
                    t[:, dst] = t[:, src]
                else:
                    t[dst] = t[src]
        self.host.moves = []
        for got, want in zip([t for t in self.caches + self.scales if t is not None], self.want):
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("batch", [1, 5, 70])
def test_random_lives(dtype, page, batch):
    rng = np.random.default_rng(page * 100 + batch)
    longest = 5 * page + 3
    pool = Pool(rng, batch=batch, page=page, blocks=batch * 9 + 20, longest=longest, dtype=dtype, share=0.4, extra=12)
    for step in range(6):
        pool.extend(rng.integers(-1, page + 4, size=batch).tolist(), page + 2)
        parents = np.where(rng.random(batch) < 0.4, rng.integers(-1, batch + 1, size=batch), np.arange(batch))
        pool.fork(parents.tolist())
        pool.extend(rng.integers(0, 3, size=batch).tolist(), 2)
        pool.free(np.where(rng.random(batch) < 0.5, -1, rng.integers(0, longest, size=batch)).tolist())
        if step % 2:
            pool.compact()


@pytest.mark.parametrize("batch", [1024, 1500])
def test_more_rows_than_one_round_of_the_scan(batch):
    """Rows past the first thousand grow into pages that earlier rows share."""
    rng = np.random.default_rng(batch)
    pool = Pool(rng, batch=batch, page=16, blocks=9000, longest=40, share=0.6, layers=0, inner=(1, 4), scales=False)
    pool.extend(rng.integers(0, 20, size=batch).tolist(), 19)
    pool.free(np.where(rng.random(batch) < 0.5, 0, -1).tolist())
    pool.compact()
    pool.extend(rng.integers(0, 5, size=batch).tolist(), 4)


@pytest.mark.parametrize("blocks", [8192, 8193, 20000])
def test_pools_of_many_pages(blocks):
    rng = np.random.default_rng(blocks)
    pool = Pool(rng, batch=60, page=4, blocks=blocks, longest=900, layers=1, inner=(1, 4))
    pool.free(np.where(np.arange(60) % 3 == 0, 0, -1).tolist())
    pool.compact()
    pool.extend(np.where(np.arange(60) % 3 == 0, 300, 1).tolist(), 300)
    pool.free([0] * 60)
    pool.compact()


@pytest.mark.parametrize("cache", [torch.uint8, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers", [0, 1, 5])
@pytest.mark.parametrize("inner", [(2, 8), (3, 5), (8, 128)])
def test_page_types_and_sizes(cache, layers, inner):
    rng = np.random.default_rng(5)
    pool = Pool(rng, batch=12, page=16 if inner != (3, 5) else 3, blocks=120, longest=40, layers=layers, inner=inner,
                cache=cache, scales=cache is torch.uint8, share=0.7)
    pool.extend([3] * 12, 3)
    pool.free([0, -1, 5] * 4)
    pool.compact()


def test_too_few_pages_do_nothing():
    rng = np.random.default_rng(6)
    pool = Pool(rng, batch=4, page=4, blocks=30, longest=20, extra=30)
    free = int((pool.refs == 0).sum())
    pool.extend([4 * free, 4, 0, 1], 4 * free)      # too many
    pool.extend([500, 0, 0, 0], 500)                # a table too short, and too many
    pool.extend([0, 0, 0, 0], 0)
    pool.extend([4 * (free - 2), 0, 0, 0], 4 * free)
    pool.compact()


def test_a_table_too_short_is_told_apart():
    rng = np.random.default_rng(7)
    pool = Pool(rng, batch=2, page=4, blocks=60, longest=8, extra=0)
    assert int(musa_aiter.kv_extend_paged_sequences(*pool.caches, *pool.state, torch.tensor([50, 1], device=DEV), 50,
                                                    **pool.kw())[1]) == -(1 << 62)
    pool.check()


def test_owners_that_are_no_rows_keep_their_pages():
    """A page kept by the caller is neither reused nor written, and moves with its count."""
    rng = np.random.default_rng(8)
    pool = Pool(rng, batch=3, page=8, blocks=40, longest=30)
    pool.refs += (torch.arange(40, device=DEV) % 3 == 0).int()
    pool.host.refs = pool.refs.tolist()
    pool.extend([9, 9, 9], 9)
    pool.free([0, 0, 0])
    pool.compact()
    pool.extend([1, 2, 3], 3)


def test_ids_outside_the_cache_are_passed_over():
    rng = np.random.default_rng(9)
    pool = Pool(rng, batch=4, page=4, blocks=40, longest=20)
    tables = np.array(pool.host.tables)
    tables[0, 0], tables[1, 0], tables[2, 2] = 4000, -3, 40
    lens = np.array([6, 7, 10, 90])  # the last one runs past its table
    pool.start(tables, lens, np.array(pool.host.refs), torch.int64)
    pool.fork([1, 0, 3, 2])
    pool.free([5, 1, 0, 2])
    pool.extend([2, 2, 2, 2], 2)
    pool.compact()


def test_tables_with_gaps_between_rows():
    rng = np.random.default_rng(10)
    pool = Pool(rng, batch=6, page=4, blocks=70, longest=30, share=0.5)
    wide = torch.full((6, 40), 77, dtype=torch.int32, device=DEV)
    width = pool.tables.shape[1]
    wide[:, :width] = pool.tables
    pool.tables = wide[:, :width]
    pool.state = (pool.tables, pool.lens, pool.refs)
    pool.extend([3, 0, 5, 1, 1, 1], 5)
    pool.fork([1, 1, 1, 3, 4, -1])
    pool.free([-1, 2, -1, 0, -1, -1])
    pool.compact()
    assert (wide[:, width:] == 77).all()


def test_no_rows():
    state = (torch.zeros((0, 4), dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV),
             torch.zeros(8, dtype=torch.int32, device=DEV))
    caches = [torch.zeros(8, 2, 4, 4, device=DEV) for _ in range(2)]
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    slots, left = musa_aiter.kv_extend_paged_sequences(*caches, *state, none, 3)
    assert slots.shape == (0, 3) and int(left) == 8
    musa_aiter.kv_fork_paged_sequences(*state, none, block_size=4)
    musa_aiter.kv_free_paged_sequences(*state, none, block_size=4)
    assert int(musa_aiter.kv_compact_paged_blocks(*caches, state[0], state[2])) == 0


def test_captured_and_replayed():
    rng = np.random.default_rng(11)
    pool = Pool(rng, batch=8, page=4, blocks=200, longest=30, share=0.5, extra=20)
    rows = [torch.zeros(8, dtype=torch.int32, device=DEV) for _ in range(3)]

    def step():
        musa_aiter.kv_fork_paged_sequences(*pool.state, rows[0], block_size=4)
        slots, left = musa_aiter.kv_extend_paged_sequences(*pool.caches, *pool.state, rows[1], 6, **pool.kw())
        musa_aiter.kv_free_paged_sequences(*pool.state, rows[2], block_size=4)
        return slots, left, musa_aiter.kv_compact_paged_blocks(*pool.caches, pool.tables, pool.refs, **pool.kw())

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        slots, left, count = step()
    for _ in range(5):
        parents = np.where(rng.random(8) < 0.5, rng.integers(0, 8, size=8), np.arange(8)).tolist()
        new, keep = rng.integers(0, 7, size=8).tolist(), rng.integers(-5, 30, size=8).tolist()
        for t, v in zip(rows, (parents, new, keep)):
            t.copy_(torch.tensor(v))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        pool.host.fork(parents)
        want, want_left = pool.host.extend(new, 6)
        pool.host.free(keep)
        assert int(count) == pool.host.compact() and slots.tolist() == want and int(left) == want_left
        pool.check()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_a_serving_run(fmt):
    """Prompts, forks, decode steps, ends and a compaction: the attention of every step matches a dense cache of the
    decoded tokens that every row carries along on the host."""
    rng = np.random.default_rng(12)
    batch, page, nh, hd, heads, blocks = 5, 16, 2, 64, 4, 120
    caches = [torch.zeros(blocks, nh, hd, page, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(blocks, nh, device=DEV) for _ in range(2)]
    tables = torch.full((batch, 20), -1, dtype=torch.int32, device=DEV)
    lens, refs = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (batch, blocks))
    state, kw = (tables, lens, refs), {"k_scales": scales[0], "v_scales": scales[1]}
    history = [[[], []] for _ in range(batch)]  # the rows' tokens, K and V
    top = {"e4m3": 448.0, "e5m2": 57344.0}[fmt]
    step = {"e4m3": 2.0 ** -4, "e5m2": 2.0 ** -3}[fmt]

    def grow(new):
        most = max(new)
        slots, left = musa_aiter.kv_extend_paged_sequences(*caches, *state, torch.tensor(new, device=DEV), most, **kw)
        assert int(left) >= 0
        x = torch.from_numpy(rng.normal(size=(2, batch, most, nh, hd)).astype(np.float32)).to(torch.bfloat16)
        lin = x.to(DEV).view(2, batch * most, nh, hd)
        musa_aiter.kv_linear_to_paged_fp8_block(lin[0], lin[1], *caches, slots.view(-1), *scales, fp8_format=fmt)
        for b, n in enumerate(new):
            for i in range(n):
                for kv in range(2):
                    history[b][kv].append(x[kv, b, i].double().numpy())

    def attend(rows):
        starts = np.concatenate([[0], np.cumsum(rows)])
        q = torch.from_numpy(rng.normal(size=(int(starts[-1]), heads, hd)).astype(np.float32)).to(torch.bfloat16)
        out = musa_aiter.kv_paged_attention_fp8(q.to(DEV), *caches, tables, lens, *scales, fp8_format=fmt,
                                                query_starts=torch.from_numpy(starts).to(DEV)).double().cpu().numpy()
        want = ref.attention(q.double().numpy(), *(c.cpu().numpy() for c in caches), tables.cpu().numpy(),
                             lens.tolist(), *(s.double().cpu().numpy() for s in scales), fmt, starts=starts)
        assert np.abs(out - want[0]).max() <= (2.0 ** -8 * np.abs(want[0]) + 2.0 ** -10 * want[2] + 1e-4).max()
        for b in range(batch):  # what the cache holds is what the row was given, to within the codes' rounding
            n = int(lens[b])
            assert n == len(history[b][0])
            for kv in range(2):
                for pos in range(n):
                    p, o = int(tables[b, pos // page]), pos % page
                    code = caches[kv][p, :, :, o].cpu().numpy()
                    s = scales[kv][p].double().cpu().numpy()[:, None]
                    got, true = ref.decode_table(fmt)[code] * s, history[b][kv][pos]
                    # Encoded at most three times (its block's scale grew), small values flushed each time.
                    assert (np.abs(got - true) <= 3 * step * np.abs(true) + s * 2.0 ** -5).all()
                    assert np.abs(true).max() <= s.max() * top * (1 + step)

    grow([30, 17, 0, 5, 48])
    attend([3, 17, 0, 1, 2])
    musa_aiter.kv_fork_paged_sequences(*state, torch.tensor([0, 0, 0, 4, 4], device=DEV), block_size=page)
    history = [[list(history[p][0]), list(history[p][1])] for p in (0, 0, 0, 4, 4)]
    for _ in range(3):
        grow([1, 1, 1, 1, 0])
        attend([1, 1, 1, 1, 1])
    musa_aiter.kv_free_paged_sequences(*state, torch.tensor([0, -1, 20, -1, -1], device=DEV), block_size=page)
    history[0], history[2] = [[], []], [x[:20] for x in history[2]]
    count = int(musa_aiter.kv_compact_paged_blocks(*caches, tables, refs, **kw))
    assert (refs[:count] > 0).all() and (refs[count:] == 0).all()
    grow([40, 2, 6, 1, 1])
    attend([4, 2, 6, 1, 1])
