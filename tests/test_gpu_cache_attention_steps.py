"""GPU: the operators on plain paged caches as they are used together, captured into graphs and on several streams."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import cache_attention_ref as ref
from tests.test_gpu_cache_attention import DEV, Case, call, tree_masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,extra", [([3, 1, 9], 5), ([200, 64, 129], 300)])
def test_captured_and_replayed(rows, extra):
    lens = [900, 400, 700]
    cases = [Case(lens=lens, rows=rows, heads=12, kv_heads=3, hd=64, extra=extra, window=500, sinks=5, seed=s) for s in range(3)]
    shape = cases[0].cache[0].shape
    masks = [torch.from_numpy(tree_masks(c.rng, rows, 4)).to(DEV) for c in cases]
    gathered = [torch.rand((3, 3, 901), device=DEV) for _ in cases]
    keep = torch.tensor([100, 400, 300], dtype=torch.int32, device=DEV)
    starts = cases[0].index_of(cases[0].starts)
    buffers = [t.clone() for t in cases[0].args()]
    mask, weights = masks[0].clone(), gathered[0].clone()

    def fill(k):
        for to, from_ in zip([*buffers, mask, weights], [*cases[k].args(), masks[k], gathered[k]]):
            to.copy_(from_)

    def step():
        query, key, value, tables, lens = buffers
        sight = dict(query_starts=starts, window=500, sinks=5)
        out, lse = musa_aiter.kv_paged_attention(query, key, value, tables, lens, return_lse=True, **sight)
        tree, tree_lse = musa_aiter.kv_paged_attention_tree(query, key, value, tables, lens, mask, query_starts=starts,
                                                            return_lse=True)
        musa_aiter.kv_accumulate_attention_weights(weights, query, key, tables, lens, lse, **sight)
        kept = musa_aiter.kv_evict_paged_tokens(key, value, weights, tables, lens, keep, sinks=3, recent=40)
        return [out, lse, tree, tree_lse, kept]

    def state():
        return [t.clone() for t in (*buffers[1:3], weights)]

    want = []
    for k in range(3):
        fill(k)
        want.append([t.clone() for t in step()] + state())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        graphs.append((graph, captured))
    for turn, k in enumerate((0, 1, 2, 0, 2, 1)):
        graph, captured = graphs[turn % 2]
        fill(k)
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip([*captured, *state()], want[k]):
            assert torch.equal(got, w)
        fill((k + 1) % 3)
        for got, w in zip([*step(), *state()], want[(k + 1) % 3]):
            assert torch.equal(got, w)
    assert shape == cases[0].cache[0].shape


def test_streams_side_by_side():
    made = [Case(lens=[900, 400, 700], rows=r, heads=12, kv_heads=3, hd=64, extra=100, tree=4, seed=s)
            for s, r in enumerate(([200, 64, 129], [3, 1, 9], [128, 64, 100], [1, 1, 1]))]
    want = [call(c) for c in made]
    args = [(c.args(), c.sight(), torch.from_numpy(c.masks).to(DEV)) for c in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = []
    for _ in range(4):
        for s, (a, sight, masks) in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(musa_aiter.kv_paged_attention_tree(*a, masks, return_lse=True, **sight))
    torch.cuda.synchronize()
    for k, (out, lse) in enumerate(got):
        assert torch.equal(out, want[k % 4][0]) and torch.equal(lse, want[k % 4][1])


class Serving:
    """A small engine over the public calls, next to plain lists of each (sequence, kv head)'s keys and values."""

    def __init__(self, batch, dtype=torch.bfloat16, nh=2, hd=64, bs=16, blocks=200, width=40, tokens=400):
        self.rng, self.dtype, self.nh, self.hd, self.bs, self.batch = np.random.default_rng(5), dtype, nh, hd, bs, batch
        self.key, self.value = (torch.full((blocks, nh, hd, bs), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
        self.tables = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=DEV)
        self.refs = torch.zeros(blocks, dtype=torch.int32, device=DEV)
        self.weights = torch.zeros((batch, nh, tokens), device=DEV)
        self.plain = [[[] for _ in range(nh)] for _ in range(batch)]  # (key, value) of each cached token

    def append(self, counts):
        counts = np.asarray(counts)
        slots, left = musa_aiter.kv_extend_paged_sequences(
            self.key, self.value, self.tables, self.lens, self.refs, torch.tensor(counts, dtype=torch.int32, device=DEV),
            int(counts.max()))
        assert int(left) >= 0
        shape = (self.batch, int(counts.max()), self.nh, self.hd)
        new = [torch.from_numpy(self.rng.normal(size=shape).astype(np.float32)).to(self.dtype) for _ in range(2)]
        musa_aiter.kv_linear_to_paged(*(x.flatten(0, 1).to(DEV) for x in new), self.key, self.value, slots.view(-1))
        for b, n in enumerate(counts):
            for i in range(n):
                for h in range(self.nh):
                    self.plain[b][h].append((new[0][b, i, h].double().numpy(), new[1][b, i, h].double().numpy()))
        return slots

    def rows(self, counts, heads):
        total = int(np.sum(counts))
        query = torch.from_numpy((1.5 * self.rng.normal(size=(total, heads, self.hd))).astype(np.float32)).to(self.dtype)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=DEV)
        return query.to(DEV), starts

    def expect(self, query, counts, masks=None):
        """float64 outputs and logarithms, from the plain lists."""
        q = query.double().cpu().numpy()
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        group, t = q.shape[1] // self.nh, 0
        for b, n in enumerate(counts):
            length = len(self.plain[b][0])
            seen = ref._seen(length, n, None, 0, None if masks is None else masks[t:t + n])
            for i in range(n):
                for g in range(q.shape[1]):
                    k, v = (np.stack([x[p] for x in self.plain[b][g // group]]) for p in (0, 1))
                    s = np.where(seen[i], k @ q[t, g] / self.hd ** 0.5, -np.inf)
                    p = np.exp(s - s.max())
                    out[t, g], lse[t, g] = p @ v / p.sum(), s.max() + np.log(p.sum())
                t += 1
        return out, lse

    def near(self, got, want):
        got = [x.double().cpu().numpy() for x in got]
        # One rounding of the output, one of each weight (2^-8 of sums of weights times sizes of about 1), float32 scores.
        assert np.abs(got[0] - want[0]).max() < 2.0 ** -7
        assert np.abs(got[1] - want[1]).max() < 2.0 ** -14

    def cut(self, keep):
        musa_aiter.kv_free_paged_sequences(self.tables, self.lens, self.refs, keep, block_size=self.bs)


def test_a_serving_run():
    """Prompts, decode steps that gather weights, evictions, drafted trees of which a path is accepted."""
    s, heads = Serving(batch=3), 8
    counts = [130, 70, 1]
    s.append(counts)
    gathered = np.zeros(s.weights.shape)
    for turn in range(4):
        query, starts = s.rows(counts, heads)
        out, lse = musa_aiter.kv_paged_attention(query, s.key, s.value, s.tables, s.lens, query_starts=starts, return_lse=True)
        s.near((out, lse), s.expect(query, counts))
        musa_aiter.kv_accumulate_attention_weights(s.weights, query, s.key, s.tables, s.lens, lse, query_starts=starts)
        total = s.weights.double().sum(dim=2).cpu().numpy()
        gained = np.asarray(counts)[:, None] * heads / s.nh
        assert np.allclose(total - gathered.sum(axis=2), gained, rtol=1e-4)
        gathered = s.weights.double().cpu().numpy()
        counts = [1, 1, 1]
        s.append(counts)
    # Down to 60 tokens, the heaviest of each head; the second sequence is shared with a kept prefix and stays.
    s.refs[s.tables[1, 0].long()] += 1
    before = s.weights.cpu().numpy().copy()
    keep = torch.tensor([60, 60, 60], dtype=torch.int32, device=DEV)
    kept = musa_aiter.kv_evict_paged_tokens(s.key, s.value, s.weights, s.tables, s.lens, keep, sinks=4, recent=20,
                                            ref_counts=s.refs)
    assert kept.tolist() == [60, 74, 5]
    for h in range(s.nh):
        n = len(s.plain[0][h])
        middle = sorted(range(4, n - 20), key=lambda p: (-before[0, h, p], p))[:36]
        stay = [*range(4), *sorted(middle), *range(n - 20, n)]
        s.plain[0][h] = [s.plain[0][h][p] for p in stay]
        assert np.array_equal(s.weights[0, h, :60].cpu().numpy(), before[0, h, stay])
    used = int((s.refs > 0).sum())
    s.cut(kept)
    assert s.lens.tolist() == [60, 74, 5] and int((s.refs > 0).sum()) == used - 5
    # Decode on what is left.
    for turn in range(2):
        s.append([1, 1, 1])
        query, _ = s.rows([1, 1, 1], heads)
        got = musa_aiter.kv_paged_attention(query, s.key, s.value, s.tables, s.lens, return_lse=True)
        s.near(got, s.expect(query, [1, 1, 1]))
    # Trees of drafts; the longest path of each is accepted.
    counts = [9, 20, 3]
    context = s.lens.tolist()
    slots = s.append(counts)
    masks = tree_masks(s.rng, counts)
    query, starts = s.rows(counts, heads)
    got = musa_aiter.kv_paged_attention_tree(query, s.key, s.value, s.tables, s.lens, torch.from_numpy(masks).to(DEV),
                                             query_starts=starts, return_lse=True)
    s.near(got, s.expect(query, counts, masks))
    source, target, keep, first = [], [], [], 0
    for b, n in enumerate(counts):
        bits = max((int(m) for m in masks[first:first + n, 0]), key=lambda m: bin(m).count("1"))
        path = [k for k in range(n) if bits >> k & 1]
        source += [int(slots[b, k]) for k in path]
        target += [int(slots[b, i]) for i in range(len(path))]
        keep.append(context[b] + len(path))
        for h in range(s.nh):
            s.plain[b][h] = s.plain[b][h][:context[b]] + [s.plain[b][h][context[b] + k] for k in path]
        first += n
    moved = musa_aiter.kv_paged_to_linear(s.key, s.value, torch.tensor(source, device=DEV))
    musa_aiter.kv_linear_to_paged(*moved, s.key, s.value, torch.tensor(target, device=DEV))
    s.cut(torch.tensor(keep, dtype=torch.int32, device=DEV))
    s.append([1, 1, 1])
    query, _ = s.rows([1, 1, 1], heads)
    got = musa_aiter.kv_paged_attention(query, s.key, s.value, s.tables, s.lens, return_lse=True)
    s.near(got, s.expect(query, [1, 1, 1]))
