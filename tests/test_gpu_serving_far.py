"""GPU: the operators on block-scaled caches and pages at places past 2^32 bytes, against the same call on a small cache."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests.test_gpu_block_attention import Case, _go
from tests.test_gpu_block_store import _inputs, _mapping

pytestmark = pytest.mark.gpu
DEV = "cuda"
NB, NH, HD, BS = 70_000, 8, 128, 64  # 4.6e9 bytes a plane


@pytest.fixture(autouse=True)
def _room():
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GiB of device memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("lens,longest,dtype", [([300, 5000], None, "bf16"), ([300, 700], 700, "bf16"),
                                                ([300, 1000], 1 << 20, "fp16"), ([30, 100], None, "fp32")])
def test_decode_steps(lens, longest, dtype):
    case = Case(lens=lens, heads=16, kv_heads=NH, hd=HD, bs=BS, seed=18, dtype=dtype)
    want, want_lse = _go(case, max_seq_len=longest)
    case.check(want, want_lse)
    args, kw = case.args()
    shift = NB - case.cache[0].shape[0]
    for i in (1, 2):
        far = torch.empty(NB, NH, HD, BS, dtype=torch.uint8, device=DEV)
        far[shift:] = args[i]
        args[i] = far
    for i in (5, 6):
        far = torch.zeros(NB, NH, device=DEV)
        far[shift:] = args[i]
        args[i] = far
    args[3] = torch.where(args[3] >= 0, args[3] + shift, -1)
    out, lse = musa_aiter.kv_paged_attention_fp8(*args, **kw, max_seq_len=longest, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("tokens", [40, 400])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("layers", [0, 2])
def test_stores(tokens, captured, layers):
    rng = np.random.default_rng(tokens)
    few = 30
    blocks = NB // max(layers, 1)
    cache, scales, lin = _inputs(rng, layers, few, NH, HD, BS, tokens, torch.bfloat16)
    slots = torch.from_numpy(_mapping("scattered", rng, few, BS, tokens)).to(DEV)
    lin = [x.to(DEV) for x in lin]
    want = [torch.from_numpy(x).to(DEV) for x in (*cache, *scales)]
    shift, lead = blocks - few, (layers,) if layers else ()
    far = []
    for t in want:
        f = torch.zeros(*lead, blocks, *t.shape[len(lead) + 1:], dtype=t.dtype, device=DEV)
        f.narrow(len(lead), shift, few).copy_(t)
        far.append(f)
    far_slots = torch.where(slots >= 0, slots + shift * BS, -1)
    musa_aiter.kv_linear_to_paged_fp8_block(*lin, *want[:2], slots, *want[2:])
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            musa_aiter.kv_linear_to_paged_fp8_block(*lin, *far[:2], far_slots, *far[2:])
        graph.replay()
    else:
        musa_aiter.kv_linear_to_paged_fp8_block(*lin, *far[:2], far_slots, *far[2:])
    torch.cuda.synchronize()
    for got, w in zip(far, want):
        assert torch.equal(got.narrow(len(lead), shift, few).contiguous().view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("layers", [0, 2])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_page_moves(layers, index):
    blocks = NB // max(layers, 1)
    lead = (layers,) if layers else ()
    caches = [torch.zeros(*lead, blocks, NH, HD, BS, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(*lead, blocks, NH, device=DEV) for _ in range(2)]
    planes = [*caches, *scales]
    at = len(lead)
    shared, spare = blocks - 7, blocks - 2  # a partial page of two rows; the only free page
    kept = []
    for t in planes:
        page = t.select(at, shared)
        page.copy_(torch.randint(0, 200, page.shape, device=DEV))
        kept.append(page.clone())
    refs = torch.ones(blocks, dtype=index, device=DEV)
    refs[shared], refs[spare] = 2, 0
    tables = torch.tensor([[shared, -1], [shared, -1]], dtype=index, device=DEV)
    lens = torch.tensor([5, 5], dtype=index, device=DEV)
    kw = {"k_scales": scales[0], "v_scales": scales[1]}
    slots, left = musa_aiter.kv_extend_paged_sequences(*caches, tables, lens, refs, torch.tensor([1, 1], device=DEV), 1, **kw)
    assert int(left) == 0 and slots.tolist() == [[spare * BS + 5], [shared * BS + 5]]
    assert tables.tolist() == [[spare, -1], [shared, -1]]
    for t, want in zip(planes, kept):
        assert torch.equal(t.select(at, spare), want) and torch.equal(t.select(at, shared), want)
    # Everything else is given back: both pages move to the front.
    refs.zero_()
    refs[shared] = refs[spare] = 1
    for t in planes:
        t.select(at, spare).add_(1)
    assert int(musa_aiter.kv_compact_paged_blocks(*caches, tables, refs, **kw)) == 2
    assert tables.tolist() == [[1, -1], [0, -1]] and refs[:3].tolist() == [1, 1, 0] and int(refs.sum()) == 2
    for t, want in zip(planes, kept):
        assert torch.equal(t.select(at, 0), want) and torch.equal(t.select(at, 1), want + 1)
