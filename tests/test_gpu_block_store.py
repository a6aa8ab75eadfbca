"""GPU: kv_linear_to_paged_fp8_block against the definition, code for code and scale for scale.

The operator's arithmetic is float32 with one rounding per operation, so codes and scales are compared exactly.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import musa_aiter
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODE_TYPE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def _inputs(rng, nl, nb, nh, hd, bs, tokens, dtype, *, fresh=0.5):
    """Random codes of every value, scales some of which are not usable, and tokens of widely differing size."""
    lead = (nl,) if nl else ()
    cache = [rng.integers(0, 256, size=(*lead, nb, nh, hd, bs), dtype=np.uint8) for _ in range(2)]
    scales = []
    for _ in range(2):
        s = np.exp(rng.normal(-4, 1.5, size=(*lead, nb, nh))).astype(np.float32)
        kind = rng.random(s.shape)
        s[kind < 0.1 * fresh] = 0.0
        s[(kind >= 0.1 * fresh) & (kind < 0.14 * fresh)] = np.nan
        s[(kind >= 0.14 * fresh) & (kind < 0.18 * fresh)] = np.inf
        s[(kind >= 0.18 * fresh) & (kind < 0.22 * fresh)] = -1.0
        scales.append(s)
    lin = []
    for _ in range(2):
        x = rng.normal(size=(*lead, tokens, nh, hd)) * np.exp(rng.normal(0, 1, size=(*lead, tokens, 1, 1)))
        lin.append(torch.from_numpy(x.astype(np.float32)).to(dtype))
    return cache, scales, lin


def _expect(cache, scales, lin, slots, fmt):
    cache, scales = [c.copy() for c in cache], [s.copy() for s in scales]
    for c, s, x in zip(cache, scales, lin):
        x = x.float().numpy()
        for layer in range(c.shape[0] if c.ndim == 5 else 1):
            at = layer if c.ndim == 5 else slice(None)
            ref.block_store(x[at], c[at], s[at], slots, fmt)
    return cache, scales


def _check(cache, scales, want_cache, want_scales):
    for name, got, want in zip(("key", "value"), cache, want_cache):
        assert np.array_equal(got.cpu().view(torch.uint8).numpy(), want), name
    for name, got, want in zip(("k_scales", "v_scales"), scales, want_scales):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=True), name


def _run(nl, nb, nh, hd, bs, slots, dtype, fmt, seed=0):
    rng = np.random.default_rng(seed)
    cache, scales, lin = _inputs(rng, nl, nb, nh, hd, bs, len(slots), dtype)
    want = _expect(cache, scales, lin, slots, fmt)
    d_cache = [torch.from_numpy(c).to(DEV) for c in cache]
    d_scales = [torch.from_numpy(s).to(DEV) for s in scales]
    musa_aiter.kv_linear_to_paged_fp8_block(*(x.to(DEV) for x in lin), *d_cache, torch.from_numpy(slots).to(DEV),
                                            *d_scales, fp8_format=fmt)
    torch.cuda.synchronize()
    _check(d_cache, d_scales, *want)


def _mapping(kind, rng, nb, bs, tokens):
    if kind == "sequences":  # contiguous runs, half of them beginning inside a block
        order, out, used = rng.permutation(nb), [], 0
        while len(out) < tokens and used < nb:
            start = int(rng.integers(0, bs)) if rng.random() < 0.5 else 0
            n = int(rng.integers(1, 3 * bs + 2))
            blocks = -(-(start + n) // bs)
            if used + blocks > nb:
                break
            j = start + np.arange(n)
            out += (order[used + j // bs] * bs + j % bs).tolist()
            used += blocks
        s = np.array(out[:tokens])
    elif kind == "scattered":  # any slot, some named twice, some skipped
        s = rng.integers(0, nb * bs, size=tokens)
        s[rng.random(tokens) < 0.15] = -1
        s[tokens // 2] = s[0]
    else:  # "last": one token per block, each at the end
        s = rng.permutation(nb)[:tokens] * bs + bs - 1
    return s.astype(np.int64)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("kind", ["sequences", "scattered", "last"])
@pytest.mark.parametrize("tokens", [1, 37, 256, 257, 700])
def test_matches_the_definition(fmt, dtype, kind, tokens):
    rng = np.random.default_rng(tokens)
    nb, bs = 800 if kind == "last" else 150, 16
    _run(0, nb, 2, 64, bs, _mapping(kind, rng, nb, bs, tokens), DTYPES[dtype], fmt, seed=tokens)


@pytest.mark.parametrize("bs", [1, 3, 8, 16, 32, 48, 64, 128, 200])
@pytest.mark.parametrize("hd", [1, 5, 16, 40, 64, 96, 128, 256, 300])
@pytest.mark.parametrize("tokens", [50, 300])
def test_block_sizes_and_head_dims(bs, hd, tokens):
    rng = np.random.default_rng(bs * 1000 + hd)
    nb = max(6, 3 * tokens // bs)
    for kind in ("sequences", "scattered"):
        _run(0, nb, 3, hd, bs, _mapping(kind, rng, nb, bs, tokens), torch.bfloat16, "e4m3", seed=hd)


@pytest.mark.parametrize("tokens", [9, 500])
@pytest.mark.parametrize("nh,hd,bs", [(8, 128, 16), (1, 128, 64), (5, 96, 32), (2, 64, 48)])
def test_layers_at_once(tokens, nh, hd, bs):
    rng = np.random.default_rng(tokens + nh)
    nb = 60
    for kind in ("sequences", "scattered"):
        _run(3, nb, nh, hd, bs, _mapping(kind, rng, nb, bs, tokens), torch.float16, "e5m2", seed=tokens)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("tokens", [40, 400])
def test_every_kind_of_value(dtype, fmt, tokens):
    """Zeros, NaN, infinities, subnormals, the type's extremes; blocks that hold nothing else."""
    rng = np.random.default_rng(3)
    nb, nh, hd, bs = 40, 2, 64, 16
    cache, scales, lin = _inputs(rng, 0, nb, nh, hd, bs, tokens, DTYPES[dtype])
    info = torch.finfo(DTYPES[dtype])
    odd = torch.tensor([0.0, -0.0, float("nan"), float("inf"), -float("inf"), info.max, -info.max, info.tiny,
                        info.tiny / 4, -info.smallest_normal, 1e-30, 2.0 ** -61 * 448]).to(DTYPES[dtype])
    for x in lin:
        pick = rng.random(x.shape) < 0.2
        pick[::3] = False
        x[torch.from_numpy(pick)] = odd[rng.integers(0, len(odd), size=int(pick.sum()))]
        x[1], x[4], x[7] = 0.0, float("nan"), float("inf")
    slots = _mapping("sequences", rng, nb, bs, tokens)
    slots = np.concatenate([slots, np.full(tokens - len(slots), -1)]) if len(slots) < tokens else slots
    want = _expect(cache, scales, lin, slots, fmt)
    d_cache = [torch.from_numpy(c).to(DEV) for c in cache]
    d_scales = [torch.from_numpy(s).to(DEV) for s in scales]
    musa_aiter.kv_linear_to_paged_fp8_block(*(x.to(DEV) for x in lin), *d_cache, torch.from_numpy(slots).to(DEV),
                                            *d_scales, fp8_format=fmt)
    _check(d_cache, d_scales, *want)


@pytest.mark.parametrize("tokens", [33, 290])
def test_layouts_that_are_not_packed(tokens):
    """Rows cut out of a fused projection, caches interleaved in one tensor, float8 types, scattered scales, int32 slots."""
    rng = np.random.default_rng(8)
    nb, nh, hd, bs = 70, 4, 64, 16
    cache, scales, lin = _inputs(rng, 0, nb, nh, hd, bs, tokens, torch.bfloat16)
    slots = _mapping("scattered", rng, nb, bs, tokens)
    want = _expect(cache, scales, lin, slots, "e4m3")
    fused = torch.cat([x.reshape(tokens, -1) for x in (lin[0], lin[0], lin[1])], dim=1).to(DEV)
    k, v = (fused[:, i * nh * hd:(i + 1) * nh * hd].view(tokens, nh, hd) for i in (0, 2))
    both = torch.from_numpy(np.stack(cache, axis=1)).to(DEV).view(torch.float8_e4m3fn)
    wide = torch.zeros(2, nh, nb, device=DEV)
    wide.copy_(torch.from_numpy(np.stack(scales)).transpose(1, 2))
    d_scales = [wide[i].t() for i in range(2)]
    musa_aiter.kv_linear_to_paged_fp8_block(k, v, both[:, 0], both[:, 1], torch.from_numpy(slots).int().to(DEV), *d_scales)
    _check([both[:, i].contiguous() for i in range(2)], d_scales, *want)
    # A cache whose blocks are not packed goes through a copy.
    odd = [torch.from_numpy(c).to(DEV).transpose(2, 3).contiguous().transpose(2, 3) for c in cache]
    d_scales = [torch.from_numpy(s).to(DEV) for s in scales]
    musa_aiter.kv_linear_to_paged_fp8_block(v.new_tensor(lin[0].tolist()), lin[1].to(DEV).float().double(), *odd,
                                            torch.from_numpy(slots).to(DEV), *d_scales)
    _check([c.contiguous() for c in odd], d_scales, *want)


@pytest.mark.parametrize("tokens", [5, 300])
def test_a_slot_past_the_cache_stores_nothing(tokens):
    nb, nh, hd, bs = 30, 2, 32, 16
    cache = [torch.randint(0, 256, (nb, nh, hd, bs), dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.rand(nb, nh, device=DEV) for _ in range(2)]
    before = [t.clone() for t in (*cache, *scales)]
    lin = [torch.randn(tokens, nh, hd, device=DEV) for _ in range(2)]
    for bad in (nb * bs, 1 << 40):
        slots = torch.arange(tokens, device=DEV)
        slots[tokens // 2] = bad
        with pytest.raises(ValueError, match="out of bounds"):
            musa_aiter.kv_linear_to_paged_fp8_block(*lin, *cache, slots, *scales)
    musa_aiter.kv_linear_to_paged_fp8_block(*lin, *cache, torch.full((tokens,), -7, device=DEV), *scales)
    for got, want in zip((*cache, *scales), before):
        assert torch.equal(got, want)


@pytest.mark.parametrize("tokens", [12, 310])
def test_captured_and_replayed(tokens):
    rng = np.random.default_rng(1)
    nb, nh, hd, bs = 90, 2, 64, 16
    lin = [torch.zeros(tokens, nh, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    slots = torch.full((tokens,), -1, dtype=torch.int64, device=DEV)
    cache = [torch.zeros(nb, nh, hd, bs, dtype=torch.uint8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(nb, nh, device=DEV) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        musa_aiter.kv_linear_to_paged_fp8_block(*lin, *cache, slots, *scales)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        musa_aiter.kv_linear_to_paged_fp8_block(*lin, *cache, slots, *scales)
    for rep in range(5):
        s = _mapping("scattered", rng, nb, bs, tokens)
        s[1] = nb * bs + 5  # skipped in a captured call
        slots.copy_(torch.from_numpy(s))
        for x in lin:
            x.copy_(torch.randn(x.shape) * (rep + 1))
        want_cache, want_scales = [c.clone() for c in cache], [x.clone() for x in scales]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s[1] = -1
        musa_aiter.kv_linear_to_paged_fp8_block(*lin, *want_cache, torch.from_numpy(s).to(DEV), *want_scales)
        torch.cuda.synchronize()
        for got, want in zip((*cache, *scales), (*want_cache, *want_scales)):
            assert torch.equal(got, want), rep


def test_another_stream_than_the_tensors_own():
    rng = np.random.default_rng(2)
    nb, nh, hd, bs, tokens = 50, 2, 64, 16, 400
    side = torch.cuda.Stream()
    cache, scales, lin = _inputs(rng, 0, nb, nh, hd, bs, tokens, torch.bfloat16)
    slots = _mapping("scattered", rng, nb, bs, tokens)
    want = _expect(cache, scales, lin, slots, "e4m3")
    args = [t.to(DEV) for t in lin] + [torch.from_numpy(c).to(DEV) for c in cache] + [torch.from_numpy(slots).to(DEV)]
    d_scales = [torch.from_numpy(s).to(DEV) for s in scales]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        musa_aiter.kv_linear_to_paged_fp8_block(*args, *d_scales)
    side.synchronize()
    _check(args[2:4], d_scales, *want)
