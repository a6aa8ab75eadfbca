"""GPU: the host module's calls of the operators on block-scaled caches and pages, against the Python checks."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from musa_aiter.ops import _hip
from tests.test_gpu_block_attention import Case, _go
from tests.test_gpu_block_store import _inputs
from tests.test_gpu_pages import Pool

pytestmark = pytest.mark.gpu
DEV = "cuda"
NATIVE = ("attention_native", "block_store_native", "pages_native")


@pytest.fixture(params=["module", "python"])
def path(request, monkeypatch):
    """Counts the calls that the module took; with "python" it takes none."""
    taken = []
    for name in NATIVE:
        real = getattr(_hip, name)

        def call(*args, real=real, name=name):
            got = None if request.param == "python" else real(*args)
            taken.append((name, got is not None))
            return got

        monkeypatch.setattr(_hip, name, call)
    return request.param, taken


def _took(path, name, most_left=0):
    kind, taken = path
    mine = [took for n, took in taken if n == name]
    assert mine and (not any(mine) if kind == "python" else mine.count(False) <= most_left)


@pytest.mark.parametrize("layers", [0, 3])
@pytest.mark.parametrize("tokens", [5, 700])
def test_stores(path, layers, tokens):
    rng = np.random.default_rng(tokens + layers)
    nb, nh, hd, bs = 60, 2, 64, 16
    cache, scales, lin = _inputs(rng, layers, nb, nh, hd, bs, tokens, torch.bfloat16)
    slots = torch.from_numpy(rng.permutation(nb * bs)[:tokens].astype(np.int64)).to(DEV)
    outs = []
    for _ in range(3):
        c, s = [torch.from_numpy(x).to(DEV) for x in cache], [torch.from_numpy(x).to(DEV) for x in scales]
        musa_aiter.kv_linear_to_paged_fp8_block(*(x.to(DEV) for x in lin), *c, slots, *s)
        outs.append([*c, *s])
    _took(path, "block_store_native", most_left=2)  # a stream's first calls make what the later ones use
    for other in outs[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(outs[0], other))
    slots[tokens // 2] = nb * bs
    kept = [t.clone() for t in outs[0]]
    with pytest.raises(ValueError, match="out of bounds"):
        musa_aiter.kv_linear_to_paged_fp8_block(*(x.to(DEV) for x in lin), *outs[0][:2], slots, *outs[0][2:])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(outs[0], kept))


@pytest.mark.parametrize("lens,rows,dtype", [([70, 0, 300], None, "bf16"), ([5000], None, "fp16"), ([90, 40], [3, 7], "fp32"),
                                             ([300, 200], [120, 90], "bf16")])
def test_attention(path, lens, rows, dtype):
    case = Case(lens=lens, rows=rows, heads=8, kv_heads=2, hd=64, dtype=dtype, seed=3)
    case.check(*_go(case))
    out = torch.full((len(lens) if rows is None else sum(rows), 8, 64), 3.0, dtype=case.dtype, device=DEV)
    args, kw = case.args()
    assert musa_aiter.kv_paged_attention_fp8(*args, **kw, out=out, max_seq_len=max(lens)) is out
    case.check(out)
    _took(path, "attention_native")


@pytest.mark.parametrize("layers", [0, 2])
def test_pages(path, layers):
    rng = np.random.default_rng(layers)
    pool = Pool(rng, batch=6, page=16, blocks=80, longest=100, layers=layers, share=0.5)
    pool.extend([3, 0, 20, 1, 7, 0], 20)
    parents = torch.tensor([0, 0, 2, 2, 4, 1], device=DEV)
    musa_aiter.kv_fork_paged_sequences(*pool.state, parents, block_size=16)
    pool.host.fork(parents.tolist())
    pool.extend([1, 2, 3, 4, 5, 6], 6)
    keep = torch.tensor([0, 5, -1, 40, 1000, 17], device=DEV)
    musa_aiter.kv_free_paged_sequences(*pool.state, keep, block_size=16)
    pool.host.free(keep.tolist())
    pool.check()
    _took(path, "pages_native")


def test_block_of_more_places_than_32_bits_hold():
    """One block of 2^24 tokens a head: places in it are computed in 64 bits."""
    case = Case(lens=[100], heads=4, kv_heads=1, hd=64, bs=128, seed=5, spare=0)
    want, _ = _go(case)
    args, kw = case.args()
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GiB of device memory")
    big = []
    for c in args[1:3]:
        b = torch.zeros(1, 1, 64, 1 << 24, dtype=torch.uint8, device=DEV)
        b[..., :128] = c[int(case.tables[0, 0])]
        big.append(b)
    at = int(case.tables[0, 0])
    tables = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    got = musa_aiter.kv_paged_attention_fp8(args[0], *big, tables, args[4], args[5][at:at + 1], args[6][at:at + 1], **kw)
    case.check(got)
    assert torch.isfinite(want.float()).all()
