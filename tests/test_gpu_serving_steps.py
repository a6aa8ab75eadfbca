"""GPU: the operators on block-scaled caches and pages in a row, as a server calls them; every output of every step is
held against 64 bits over what the caches hold, element by element, with the bound of test_gpu_block_attention."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests.test_gpu_block_attention import Case

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Server:
    def __init__(self, fmt, *, batch=5, page=16, kv_heads=2, hd=64, heads=4, blocks=120, width=20, layers=2):
        self.fmt, self.page, self.heads, self.batch, self.layers = fmt, page, heads, batch, layers
        self.rng = np.random.default_rng(12)
        self.caches = [torch.zeros(layers, blocks, kv_heads, hd, page, dtype=torch.uint8, device=DEV) for _ in range(2)]
        self.scales = [torch.zeros(layers, blocks, kv_heads, device=DEV) for _ in range(2)]
        self.tables = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
        self.lens, self.refs = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (batch, blocks))
        self.state = (self.tables, self.lens, self.refs)
        self.kw = {"k_scales": self.scales[0], "v_scales": self.scales[1]}

    def normal(self, *shape, size=1.0):
        return torch.from_numpy((self.rng.normal(size=shape) * size).astype(np.float32)).to(DEV, torch.bfloat16)

    def grow(self, new, size=1.0):
        most = max(new)
        slots, left = musa_aiter.kv_extend_paged_sequences(*self.caches, *self.state, torch.tensor(new, device=DEV), most,
                                                           **self.kw)
        assert int(left) >= 0
        _, _, nh, hd, _ = self.caches[0].shape
        for layer in range(self.layers):
            k, v = (self.normal(self.batch * most, nh, hd, size=size) for _ in range(2))
            musa_aiter.kv_linear_to_paged_fp8_block(k, v, *(c[layer] for c in self.caches), slots.view(-1),
                                                    *(s[layer] for s in self.scales), fp8_format=self.fmt)

    def attend(self, rows, window=None):
        case = Case(lens=[1], fmt=self.fmt)
        case.window, case.tables, case.lens = window, self.tables.cpu().numpy().astype(np.int64), self.lens.cpu().numpy()
        case.starts = None if rows is None else np.concatenate([[0], np.cumsum(rows)])
        total = self.batch if rows is None else int(case.starts[-1])
        for layer in range(self.layers):
            query = self.normal(total, self.heads, self.caches[0].shape[3])
            starts = None if rows is None else torch.from_numpy(case.starts).to(DEV)
            out, lse = musa_aiter.kv_paged_attention_fp8(
                query, *(c[layer] for c in self.caches), self.tables, self.lens, *(s[layer] for s in self.scales),
                query_starts=starts, window=window, fp8_format=self.fmt, return_lse=True)
            case.query = query.cpu()
            case.cache, case.scales = ([t[layer].cpu().numpy() for t in pair] for pair in (self.caches, self.scales))
            case.check(out, lse)

    def fork(self, parents):
        musa_aiter.kv_fork_paged_sequences(*self.state, torch.tensor(parents, device=DEV), block_size=self.page)

    def free(self, keep):
        musa_aiter.kv_free_paged_sequences(*self.state, torch.tensor(keep, device=DEV), block_size=self.page)

    def compact(self):
        return int(musa_aiter.kv_compact_paged_blocks(*self.caches, self.tables, self.refs, **self.kw))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_outputs_of_every_step(fmt):
    s = Server(fmt)
    s.grow([30, 17, 0, 5, 48])
    s.attend([3, 17, 0, 1, 2])
    s.attend([30, 17, 0, 5, 48])
    s.fork([0, 0, 0, 4, 4])
    for step in range(3):
        s.grow([1, 1, 1, 1, 0], size=2.0 ** step)
        s.attend(None)
        s.attend(None, window=9)
    s.free([0, -1, 20, -1, -1])
    count = s.compact()
    assert (s.refs[:count] > 0).all() and (s.refs[count:] == 0).all()
    s.attend(None)
    s.grow([90, 2, 6, 1, 1], size=0.01)
    s.attend([90, 2, 6, 1, 1], window=40)
    s.attend([4, 0, 1, 1, 1])
    s.free([0] * 5)
    assert int(s.refs.abs().sum()) == 0 and (s.tables == -1).all()
    s.attend(None)
