"""GPU: outputs that share memory with what a call reads."""

from __future__ import annotations

import pytest
import torch

import musa_aiter
from tests.test_gpu_cache_attention import DEV, Case, call

pytestmark = pytest.mark.gpu

FORMS = {"any": dict(lens=[40, 300, 7], rows=[2, 3, 1], heads=2, kv_heads=1, hd=40),
         "few": dict(lens=[40, 300, 7], rows=[2, 3, 1], heads=8, hd=64),
         "parts": dict(lens=[40, 3000, 7], rows=[2, 3, 1], heads=8, hd=64),
         "many": dict(lens=[1300, 640, 700], rows=[200, 64, 129], heads=12, kv_heads=3, hd=64, extra=60)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("bad", [0.0, float("inf")])
@pytest.mark.parametrize("tree", [0, 4])
def test_out_is_the_query(form, bad, tree):
    """Also where some rows see an infinity: those are computed a second time."""
    case = Case(**FORMS[form], tree=tree, pad=3, seed=41)
    for b, n in enumerate(case.lens):  # the last token of every sequence
        case.cache[1][case.tables[b, (n - 1) // 16], :, 7, (n - 1) % 16] = bad
    want, want_lse = call(case)
    query = case.query.to(DEV)
    case.query = query
    got, lse = call(case, out=query)
    assert got is query
    rows = query.shape[0] - 3
    assert torch.equal(got[:rows].view(torch.int16), want[:rows].view(torch.int16)) and torch.equal(lse, want_lse)


def test_out_next_to_and_over_the_query():
    """A buffer whose rows the query and the output share in part: the query is read as it was."""
    case = Case(**FORMS["many"], seed=42)
    want, _ = call(case)
    rows, heads, hd = case.query.shape
    base = torch.zeros((rows + 5, heads, hd), dtype=case.dtype, device=DEV)
    for q0, o0 in ((0, 5), (5, 0), (0, 1), (2, 2)):
        base.zero_()
        query, out = base[q0:q0 + rows], base[o0:o0 + rows]
        query.copy_(case.query)
        case.query, plain = query, case.query
        got, _ = call(case, out=out)
        case.query = plain
        assert got is out and torch.equal(got, want)


def test_out_in_the_cache():
    """Output rows in a block of the cache that the call reads."""
    case = Case(lens=[40, 300, 7], rows=[2, 3, 1], heads=8, kv_heads=2, hd=64, seed=43)
    want, _ = call(case)
    query, key, value, tables, lens = case.args()
    block = int(tables[1, 3])
    out = value.view(-1)[block * 2 * 64 * 16:][:query.numel()].view(query.shape)
    got = musa_aiter.kv_paged_attention(query, key, value, tables, lens, **case.sight(), out=out)
    assert torch.equal(got, want)


@pytest.mark.parametrize("form", ["few", "many"])
def test_captured_in_place(form):
    """A captured step that writes over its query, replayed with eager work in between."""
    case = Case(**FORMS[form], seed=44)
    want, _ = call(case)
    source, query = case.query.to(DEV), torch.empty(case.query.shape, dtype=case.dtype, device=DEV)
    _, *caches = case.args()
    case.query = query

    def step():
        query.copy_(source)
        return musa_aiter.kv_paged_attention(query, *caches, **case.sight(), out=query)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph, starts = torch.cuda.CUDAGraph(), case.index_of(case.starts)
    case.sight = lambda: {"query_starts": starts, "window": None, "sinks": 0}
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        query.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(query, want)
        assert torch.equal(step(), want)
