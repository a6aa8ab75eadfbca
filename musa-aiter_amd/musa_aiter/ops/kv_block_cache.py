"""FP8 paged caches with one scale per block and head: the store that fills them and the attention over them.

The caches are the paged ones of kv_transfer (``[blocks, kv_heads, head_dim, block_size]``, uint8 or float8) with
its codec; next to them stand float32 scales ``[blocks, kv_heads]``, one tensor for K and one for V, and a code
means ``decode(code) * scale[block, head]``.  The scales follow the data: the store finds them as tokens arrive.

No counterpart in the reference, which keeps one fixed scale per head and leaves attention to its callers.
Shapes, types and devices are checked on the host and raise ``ValueError``; tensors that are not on a ROCm device
raise ``RuntimeError``.  Both operators run on the current stream of the caches' device and can be captured into a
graph.
"""

from __future__ import annotations

import math
from typing import Literal

import torch

from musa_aiter.ops import _hip
from musa_aiter.ops.kv_transfer import (
    _FP8_CACHE_DTYPES,
    _INDEX_DTYPES,
    _LIN_DTYPE,
    _NATIVE_FORMATS,
    _LinearPair,
    _codec,
    _emit,
    _ensure_slotmapping_vector,
    _fp8_bytes,
    _fp8_linear_input,
    _normalize_fp8_format,
    _require_rocm,
    _validate_paged_shapes,
    _validate_stacked_paged_shapes,
)

_MAX_HEAD_DIM = 512


def _check_fp8_caches(op: str, key_cache: torch.Tensor, value_cache: torch.Tensor) -> tuple[int, int, int, int, int]:
    """(layers, blocks, kv_heads, head_dim, block_size) of 4-D (one layer) or 5-D FP8 caches."""
    for name, cache in (("key_cache_fp8", key_cache), ("value_cache_fp8", value_cache)):
        if cache.dtype is not torch.uint8 and str(cache.dtype) not in _FP8_CACHE_DTYPES:
            raise ValueError(f"{op}: {name} must be torch.uint8 or a supported torch.float8 dtype")
    if key_cache.dim() == 5:
        return _validate_stacked_paged_shapes(key_cache, value_cache, name=op)
    return (1, *_validate_paged_shapes(key_cache, value_cache, name=op))


def _check_scales(op: str, scales: torch.Tensor, which: str, shape: tuple[int, ...], device: torch.device) -> None:
    if tuple(scales.shape) != shape:
        raise ValueError(f"{op}: {which} must be {list(shape)} (one scale per block and head), got {list(scales.shape)}")
    if scales.dtype is not torch.float32:
        raise ValueError(f"{op}: {which} must be float32, got {scales.dtype}")
    if scales.device != device:
        raise ValueError(f"{op}: all tensors must be on the same device")


def _packed_blocks(cache: torch.Tensor) -> bool:
    """Whether every block's ``[kv_heads, head_dim, block_size]`` is packed (blocks and layers may have gaps)."""
    want = 1
    for extent, stride in zip(reversed(cache.shape[-3:]), reversed(cache.stride()[-3:])):
        if extent != 1 and stride != want:
            return False
        want *= extent
    return True


def _spans_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the bytes from one tensor's first element to its last meet another's."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    ends = [t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size() for t in (a, b)]
    return a.data_ptr() < ends[1] and b.data_ptr() < ends[0]


class _Written:
    """A tensor that a call writes: itself where the kernels can write there, else a copy that goes back."""

    def __init__(self, t: torch.Tensor, fits: bool):
        self.user, self.t = t, t if fits else t.clone(memory_format=torch.contiguous_format)

    def finish(self) -> None:
        if self.t is not self.user:
            self.user.copy_(self.t)


def _overlaps(t: torch.Tensor) -> bool:
    """Whether an expanded extent makes several elements share one address."""
    return any(extent > 1 and stride == 0 for extent, stride in zip(t.shape, t.stride()))


def kv_linear_to_paged_fp8_block(
    key_linear: torch.Tensor,
    value_linear: torch.Tensor,
    key_cache_fp8: torch.Tensor,
    value_cache_fp8: torch.Tensor,
    slot_mapping: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    *,
    fp8_format: Literal["e4m3", "e5m2"] = "e4m3",
) -> None:
    """Quantize ``[T, H, D]`` rows into FP8 paged caches that keep one scale per block and head.

    With stacked caches ``[L, NB, H, D, BS]`` the rows are ``[L, T, H, D]`` and the scales ``[L, NB, H]``; with
    single-layer caches ``[NB, H, D, BS]`` the scales are ``[NB, H]``.  For every block that a token goes to, per
    head and for K and V apart,

        scale = max(max|new| / F, 2**-60, old scale),      F = 448 (E4M3) or 57344 (E5M2)

    over the finite new values; tokens that were in the block before are encoded anew if the scale grew.  A call
    that writes the first slot of a block starts the block anew, and so does one that finds a scale there that is
    not positive and finite (a zeroed scale tensor): the old scale does not count, and the block's other slots
    become zeros.  Values are encoded as by kv_linear_to_paged_fp8 (non-finite ones become zeros).

    ``slot < 0`` is skipped and a slot named twice keeps the last token.  A slot past the cache raises
    ``ValueError``, with nothing stored; in a call that is being captured it is skipped.
    """
    op = "kv_linear_to_paged_fp8_block"
    codec = _NATIVE_FORMATS.get(fp8_format)
    if codec is not None and _hip.block_store_native(op, key_linear, value_linear, key_cache_fp8, value_cache_fp8,
                                                     slot_mapping, k_scales, v_scales, codec):
        _emit(op, key_linear, f"gfx950 {fp8_format.upper()} store with block scales")
        return
    fp8_format = _normalize_fp8_format(fp8_format)
    nl, nb, nh, hd, bs = _check_fp8_caches(op, key_cache_fp8, value_cache_fp8)
    layered = key_cache_fp8.dim() == 5
    lead = (nl,) if layered else ()
    if key_linear.shape != value_linear.shape or key_linear.dim() != 3 + layered:
        raise ValueError(f"{op}: key_linear and value_linear must be {'[layers, ' if layered else '['}tokens, "
                         "kv_heads, head_dim]")
    tcount = int(key_linear.shape[layered])
    if tuple(key_linear.shape) != (*lead, tcount, nh, hd):
        raise ValueError(f"{op}: linear shape does not match FP8 cache shape")
    if not key_linear.is_floating_point() or not value_linear.is_floating_point():
        raise ValueError(f"{op}: key_linear and value_linear must be floating-point")
    device = key_cache_fp8.device
    slots = _ensure_slotmapping_vector(slot_mapping, expected_len=tcount, name=op)
    for t in (key_linear, value_linear, value_cache_fp8, slots):
        if t.device != device:
            raise ValueError(f"{op}: all tensors must be on the same device")
    _check_scales(op, k_scales, "k_scales", (*lead, nb, nh), device)
    _check_scales(op, v_scales, "v_scales", (*lead, nb, nh), device)
    for name, t in (("caches", key_cache_fp8), ("caches", value_cache_fp8), ("scales", k_scales), ("scales", v_scales)):
        if _overlaps(t):
            raise ValueError(f"{op}: the {name} are written and must not be expanded")
    _require_rocm(op, key_cache_fp8)
    if tcount == 0:
        return
    key_linear, value_linear = _fp8_linear_input(key_linear), _fp8_linear_input(value_linear)
    if value_linear.dtype != key_linear.dtype:
        key_linear, value_linear = key_linear.to(torch.float32), value_linear.to(torch.float32)
    lin = _LinearPair(key_linear, value_linear, token_dim=int(layered), row=nh * hd, writable=False)
    caches = [_Written(_fp8_bytes(c), _packed_blocks(c)) for c in (key_cache_fp8, value_cache_fp8)]
    scales = [_Written(s, s.is_contiguous()) for s in (k_scales, v_scales)]
    ok = _hip.block_store(
        op=op, device=device, linear=(lin.k, lin.v), caches=[c.t for c in caches], scales=[s.t for s in scales],
        slots=slots, sizes=(nl, tcount, nb, nh, hd, bs), strides=(lin.tok_stride, lin.layer_stride),
        block_strides=[c.t.stride(-4) for c in caches], layer_strides=[c.t.stride(0) if layered else 0 for c in caches],
        codec=_codec(fp8_format), lin_dtype=_LIN_DTYPE[lin.k.dtype])
    if not ok:
        raise ValueError(f"{op}: slot index {int(slots.max())} out of bounds for caches (max {nb * bs - 1})")
    for w in (*caches, *scales):
        w.finish()
    _emit(op, key_linear, f"gfx950 {fp8_format.upper()} store with block scales")


def _read_cache(cache: torch.Tensor) -> torch.Tensor:
    cache = _fp8_bytes(cache)
    return cache if _packed_blocks(cache) else cache.contiguous()


def _index_rows(t: torch.Tensor) -> torch.Tensor:
    """An index tensor the kernels read as it is: int32 or int64, the last extent packed."""
    if t.dtype not in (torch.int32, torch.int64):
        t = t.to(torch.int64)
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def kv_paged_attention_fp8(
    query: torch.Tensor,
    key_cache_fp8: torch.Tensor,
    value_cache_fp8: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    *,
    query_starts: torch.Tensor | None = None,
    max_seq_len: int | None = None,
    softmax_scale: float | None = None,
    window: int | None = None,
    fp8_format: Literal["e4m3", "e5m2"] = "e4m3",
    out: torch.Tensor | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of ``query`` rows ``[T, heads, head_dim]`` over FP8 paged caches with block scales.

    ``heads`` is a multiple of ``kv_heads``; head ``h`` reads kv head ``h // (heads // kv_heads)``.  Sequence ``b``
    has ``seq_lens[b]`` cached tokens, position ``pos`` in slot
    ``block_tables[b, pos // block_size] * block_size + pos % block_size``.  Its query rows are
    ``query_starts[b] : query_starts[b + 1]``, the sequence's last tokens (stored already); without
    ``query_starts`` every sequence has one row (a decode step).  Row ``i`` of ``n`` sees the positions up to
    ``seq_lens[b] - n + i``, with ``window`` only the last ``window`` of them.  ``softmax_scale`` is
    ``head_dim ** -0.5`` by default.

    Tables, lengths and row starts (any integer type) are read on the device only: nothing is synchronised.  A
    position without a table entry, or whose entry lies outside the cache, is not seen.  A row that sees nothing
    gives zeros (``lse`` -inf).  Rows of ``query`` that belong to no sequence (a padded batch) are left as they
    are in ``out``, and are zeros in a new tensor; their ``lse`` is -inf either way.  Scales of blocks that a call's
    rows see are 0 (a block of zeros) or lie in [2**-60, 2**60]; scales may be expanded, e.g.
    ``per_head.expand(blocks, kv_heads)``.  Codes decode as in kv_paged_fp8_to_linear.  Query values are at most
    2**100 in size; E4M3 value scales are at most 4 where a row's scores pass 2**24.

    ``max_seq_len``, an upper bound of ``seq_lens`` that the caller knows, only decides how the work is cut;
    by default it is what ``block_tables`` has room for.  Returns the output, in ``query``'s type, and with
    ``return_lse`` also the float32 ``[T, heads]`` logarithms of the rows' softmax sums.  There is no backward pass:
    the output carries no gradient, also where ``query`` requires one.

    Sums and softmax statistics are float32.  With float32 queries everything is; with 16-bit queries weights are
    rounded to at least 11 bits, and weights (times value scale), and next to E4M3 codes query components, below 2**-28
    of a row's largest may count as zero.
    """
    op = "kv_paged_attention_fp8"
    native = _NATIVE_FORMATS.get(fp8_format)
    if native is not None and (window is None or type(window) is int and window > 0) \
            and (max_seq_len is None or type(max_seq_len) is int and max_seq_len >= 0) \
            and (softmax_scale is None or type(softmax_scale) is float and math.isfinite(softmax_scale)):
        got = _hip.attention_native(
            op, query, key_cache_fp8, value_cache_fp8, block_tables, seq_lens, k_scales, v_scales, query_starts, out,
            -1 if max_seq_len is None else max_seq_len,
            query.shape[-1] ** -0.5 if softmax_scale is None and query.dim() and query.shape[-1] else softmax_scale or 0.0,
            window or 0, native, return_lse)
        if got is not None:
            _emit(op, query, f"gfx950 {fp8_format.upper()} paged attention with block scales")
            return got if return_lse else got[0]
    if query.dim() != 3:
        raise ValueError(f"{op}: query must be [rows, heads, head_dim]")
    if query.dtype not in _LIN_DTYPE:
        raise ValueError(f"{op}: query must be float32, float16 or bfloat16, got {query.dtype}")
    codec = _codec(fp8_format)
    if key_cache_fp8.dim() == 5:
        raise ValueError(f"{op}: caches must be 4-D [blocks, kv_heads, head_dim, block_size] (one layer)")
    _, nb, nh, hd, bs = _check_fp8_caches(op, key_cache_fp8, value_cache_fp8)
    rows, heads = int(query.shape[0]), int(query.shape[1])
    if int(query.shape[2]) != hd or hd > _MAX_HEAD_DIM:
        raise ValueError(f"{op}: query head_dim {int(query.shape[2])} must match the caches' {hd} (at most {_MAX_HEAD_DIM})")
    if heads < 1 or heads % nh:
        raise ValueError(f"{op}: heads ({heads}) must be a multiple of kv_heads ({nh})")
    if block_tables.dim() != 2:
        raise ValueError(f"{op}: block_tables must be [batch, max_blocks]")
    batch = int(block_tables.shape[0])
    if seq_lens.dim() != 1 or seq_lens.shape[0] != batch:
        raise ValueError(f"{op}: seq_lens must be [batch]")
    indices = [block_tables, seq_lens]
    if query_starts is not None:
        if query_starts.dim() != 1 or query_starts.shape[0] != batch + 1:
            raise ValueError(f"{op}: query_starts must be [batch + 1]")
        indices.append(query_starts)
    elif rows != batch:
        raise ValueError(f"{op}: without query_starts there is one query row per sequence ({rows} rows, {batch} sequences)")
    if any(t.dtype not in _INDEX_DTYPES for t in indices):
        raise ValueError(f"{op}: block_tables, seq_lens and query_starts must be integer tensors")
    device = query.device
    if any(t.device != device for t in (key_cache_fp8, value_cache_fp8, *indices)):
        raise ValueError(f"{op}: all tensors must be on the same device")
    _check_scales(op, k_scales, "k_scales", (nb, nh), device)
    _check_scales(op, v_scales, "v_scales", (nb, nh), device)
    if rows * heads >= 1 << 31 or int(block_tables.shape[1]) * bs > 1 << 29:
        raise ValueError(f"{op}: at most 2**31 - 1 rows times heads and 2**29 positions per sequence")
    if window is not None and window < 1:
        raise ValueError(f"{op}: window must be positive")
    if max_seq_len is not None and max_seq_len < 0:
        raise ValueError(f"{op}: max_seq_len must be non-negative")
    scale = hd ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not math.isfinite(scale):
        raise ValueError(f"{op}: softmax_scale must be finite")
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or out.device != device):
        raise ValueError(f"{op}: out must match query's shape, dtype and device")
    _require_rocm(op, query)
    if query.shape[2] > 1 and query.stride(2) != 1:
        query = query.contiguous()
    result = torch.empty(query.shape, dtype=query.dtype, device=device) if out is None else out
    target = result if result.is_contiguous() else torch.empty(query.shape, dtype=query.dtype, device=device)
    if target is not result:
        target.copy_(result)
    lse = torch.empty((rows, heads), dtype=torch.float32, device=device) if return_lse else None
    tables, lens = _index_rows(block_tables), _index_rows(seq_lens)
    starts = None if query_starts is None else _index_rows(query_starts)
    _hip.attention(
        op=op, query=query, out=target, lse=lse, caches=[_read_cache(key_cache_fp8), _read_cache(value_cache_fp8)],
        scales=(k_scales, v_scales), tables=tables, lens=lens, starts=starts,
        sizes=(rows, batch, heads, nh, hd, bs, nb, int(tables.shape[1])), window=window or 0, softmax_scale=scale,
        longest=int(tables.shape[1]) * bs if max_seq_len is None else int(max_seq_len), dtype=_LIN_DTYPE[query.dtype],
        codec=codec, fill_rows=out is None)
    if target is not result:
        result.copy_(target)
    _emit(op, query, f"gfx950 {_normalize_fp8_format(fp8_format).upper()} paged attention with block scales")
    return (result, lse) if return_lse else result


__all__ = ["kv_linear_to_paged_fp8_block", "kv_paged_attention_fp8"]
