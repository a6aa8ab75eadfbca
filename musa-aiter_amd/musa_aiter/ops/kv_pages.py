"""Pages of a paged cache: growing, forking, cutting and compacting sequences on the device.

State, all on the caches' device and changed in place:

- ``block_tables [batch, max_blocks]`` and ``seq_lens [batch]``: row ``b`` owns the pages named by the first
  ``ceil(seq_lens[b] / block_size)`` entries of its table row;
- ``ref_counts [blocks]``: how many rows own each page; 0 means free.  A caller may count further owners (a prefix
  kept for later requests): such pages are neither reused nor written.

The three share one type, int32 or int64, are packed (table rows may have gaps), and hold what these functions and
the caller wrote; entries outside the cache are passed over.  Nothing is read by the host: the calls do not
synchronise and can be captured into a graph.  Results depend on the state alone: rows are served in order and free
pages are taken lowest id first.  No counterpart in the reference, whose callers keep their pages on the host.
"""

from __future__ import annotations

import torch

from musa_aiter.ops import _hip
from musa_aiter.ops.kv_block_cache import _check_scales, _overlaps, _packed_blocks
from musa_aiter.ops.kv_transfer import _INDEX_DTYPES, _emit, _require_rocm

_STATE_DTYPES = (torch.int32, torch.int64)


def _check_state(op: str, block_tables: torch.Tensor, seq_lens: torch.Tensor | None, ref_counts: torch.Tensor) -> int:
    """Checks the state tensors; returns the batch size."""
    if block_tables.dim() != 2:
        raise ValueError(f"{op}: block_tables must be [batch, max_blocks]")
    batch = int(block_tables.shape[0])
    if seq_lens is not None and (seq_lens.dim() != 1 or seq_lens.shape[0] != batch):
        raise ValueError(f"{op}: seq_lens must be [batch]")
    if ref_counts.dim() != 1:
        raise ValueError(f"{op}: ref_counts must be [blocks]")
    state = [t for t in (block_tables, seq_lens, ref_counts) if t is not None]
    if any(t.dtype not in _STATE_DTYPES or t.dtype != block_tables.dtype for t in state):
        raise ValueError(f"{op}: block_tables, seq_lens and ref_counts must share one dtype, int32 or int64")
    if any(t.device != block_tables.device for t in state):
        raise ValueError(f"{op}: all tensors must be on the same device")
    width = int(block_tables.shape[1])
    packed = (width <= 1 or block_tables.stride(1) == 1) and (batch <= 1 or block_tables.stride(0) >= width)
    if not packed or not ref_counts.is_contiguous() or (seq_lens is not None and not seq_lens.is_contiguous()):
        raise ValueError(f"{op}: block_tables (each row), seq_lens and ref_counts are written and must be contiguous")
    return batch


def _row_values(op: str, name: str, values: torch.Tensor, batch: int, device: torch.device) -> torch.Tensor:
    if values.dim() != 1 or values.shape[0] != batch:
        raise ValueError(f"{op}: {name} must be [batch]")
    if values.dtype not in _INDEX_DTYPES:
        raise ValueError(f"{op}: {name} must use an integer dtype")
    if values.device != device:
        raise ValueError(f"{op}: all tensors must be on the same device")
    return values.contiguous() if values.dtype in _STATE_DTYPES else values.to(torch.int64).contiguous()


def _check_block_size(op: str, block_size: int) -> int:
    if block_size < 1:
        raise ValueError(f"{op}: block_size must be positive")
    return int(block_size)


def _check_pool(op: str, key_cache: torch.Tensor, value_cache: torch.Tensor, k_scales: torch.Tensor | None,
                v_scales: torch.Tensor | None, ref_counts: torch.Tensor) -> tuple[int, dict]:
    """(block_size, arguments of the launch) of the caches whose pages a call may move."""
    if key_cache.dim() not in (4, 5) or key_cache.shape != value_cache.shape or key_cache.dtype != value_cache.dtype:
        raise ValueError(f"{op}: caches must be 4-D [blocks, kv_heads, head_dim, block_size] or 5-D [layers, ...] "
                         "tensors of one shape and dtype")
    blocks = int(key_cache.shape[-4])
    if any(int(extent) < 1 for extent in key_cache.shape):
        raise ValueError(f"{op}: all cache extents must be positive")
    if ref_counts.shape[0] != blocks:
        raise ValueError(f"{op}: ref_counts must be [blocks] ({blocks})")
    if key_cache.device != ref_counts.device or value_cache.device != ref_counts.device:
        raise ValueError(f"{op}: all tensors must be on the same device")
    if any(not _packed_blocks(c) or _overlaps(c) for c in (key_cache, value_cache)):
        raise ValueError(f"{op}: the blocks of the caches are written and must be contiguous")
    if (k_scales is None) != (v_scales is None):
        raise ValueError(f"{op}: k_scales and v_scales come together")
    lead = tuple(key_cache.shape[:-3])
    for name, scales in (("k_scales", k_scales), ("v_scales", v_scales)):
        if scales is not None:
            _check_scales(op, scales, name, (*lead, int(key_cache.shape[-3])), key_cache.device)
            if not scales.is_contiguous():
                raise ValueError(f"{op}: {name} are written and must be contiguous")
    layered = key_cache.dim() == 5
    block = key_cache.element_size()
    for extent in key_cache.shape[-3:]:
        block *= int(extent)
    caches = (key_cache, value_cache)
    return int(key_cache.shape[-1]), dict(
        caches=caches, scales=(k_scales, v_scales), layers=int(key_cache.shape[0]) if layered else 1,
        block_bytes=block, block_strides=[c.stride(-4) * c.element_size() for c in caches],
        layer_strides=[c.stride(0) * c.element_size() if layered else 0 for c in caches],
        scale_values=int(key_cache.shape[-3]))


def kv_extend_paged_sequences(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    new_lens: torch.Tensor,
    max_new: int,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Give every row room for ``new_lens[b]`` more tokens and return their slots.

    Row ``b`` takes the free pages that ``seq_lens[b] + new_lens[b]`` tokens need (``new_lens`` is cut to
    [0, max_new]).  If its last page is only partly filled and others own it too, the row gets a copy of the page
    first (all layers, with the scales of a block-scaled cache), unless the other owners are rows that grow into it
    in this call and copy it themselves: the last of them keeps it.  Caches are 4-D, or 5-D with several layers, of
    any element type.

    Returns ``(slots, pages_left)``: int64 ``[batch, max_new]`` slots of the new tokens, -1 past ``new_lens[b]``
    (``slots.view(-1)`` is a slot_mapping), and an int64 scalar: the pages still free, or, if it is negative, that
    nothing was done and all slots are -1, since so many pages were missing (-2**62: since a row of
    ``block_tables`` is too short, or int32 ``seq_lens`` for its length).
    """
    op = "kv_extend_paged_sequences"
    if type(max_new) is int and max_new >= 0:
        got = _hip.pages_native("extend", op, key_cache, value_cache, block_tables, seq_lens, ref_counts, new_lens,
                                k_scales, v_scales, 0, max_new)
        if got is not None:
            _emit(op, key_cache, "gfx950 page allocation with copy of shared pages")
            return got
    batch = _check_state(op, block_tables, seq_lens, ref_counts)
    block_size, pool = _check_pool(op, key_cache, value_cache, k_scales, v_scales, ref_counts)
    device = block_tables.device
    rows = _row_values(op, "new_lens", new_lens, batch, device)
    if max_new < 0:
        raise ValueError(f"{op}: max_new must be non-negative")
    _require_rocm(op, block_tables)
    slots = torch.empty((batch, int(max_new)), dtype=torch.int64, device=device)
    left = torch.empty((), dtype=torch.int64, device=device)
    _hip.pages("extend", op=op, device=device, tables=block_tables, lens=seq_lens, refs=ref_counts, rows=rows,
               block_size=block_size, slots=slots, result=left, max_new=int(max_new), **pool)
    _emit(op, key_cache, "gfx950 page allocation with copy of shared pages")
    return slots, left


def kv_fork_paged_sequences(
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    parents: torch.Tensor,
    *,
    block_size: int,
) -> None:
    """Make every row ``b`` a copy of the row ``parents[b]`` as it was before the call (``b`` itself: unchanged).

    All rows change at once.  Pages are shared, not copied: reference counts gain the new owners and lose the old
    ones, and a page shared while partly filled is copied when a row grows into it (kv_extend_paged_sequences).  A
    row whose parent is not in [0, batch) becomes empty.
    """
    op = "kv_fork_paged_sequences"
    if type(block_size) is int and block_size > 0 and _hip.pages_native(
            "fork", op, None, None, block_tables, seq_lens, ref_counts, parents, None, None, block_size, 0) is not None:
        _emit(op, block_tables, "gfx950 page table fork")
        return
    batch = _check_state(op, block_tables, seq_lens, ref_counts)
    rows = _row_values(op, "parents", parents, batch, block_tables.device)
    block_size = _check_block_size(op, block_size)
    _require_rocm(op, block_tables)
    if batch == 0:
        return
    _hip.pages("fork", op=op, device=block_tables.device, tables=block_tables, lens=seq_lens, refs=ref_counts,
               rows=rows, block_size=block_size)
    _emit(op, block_tables, "gfx950 page table fork")


def kv_free_paged_sequences(
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    keep_lens: torch.Tensor,
    *,
    block_size: int,
) -> None:
    """Cut every row to its first ``keep_lens[b]`` tokens (0: the row ends; negative, or past the row: unchanged).

    Pages past the kept tokens lose an owner, and their table entries become -1.
    """
    op = "kv_free_paged_sequences"
    if type(block_size) is int and block_size > 0 and _hip.pages_native(
            "free", op, None, None, block_tables, seq_lens, ref_counts, keep_lens, None, None, block_size, 0) is not None:
        _emit(op, block_tables, "gfx950 page release")
        return
    batch = _check_state(op, block_tables, seq_lens, ref_counts)
    rows = _row_values(op, "keep_lens", keep_lens, batch, block_tables.device)
    block_size = _check_block_size(op, block_size)
    _require_rocm(op, block_tables)
    if batch == 0:
        return
    _hip.pages("free", op=op, device=block_tables.device, tables=block_tables, lens=seq_lens, refs=ref_counts,
               rows=rows, block_size=block_size)
    _emit(op, block_tables, "gfx950 page release")


def kv_compact_paged_blocks(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    ref_counts: torch.Tensor,
    *,
    k_scales: torch.Tensor | None = None,
    v_scales: torch.Tensor | None = None,
) -> torch.Tensor:
    """Move the pages in use to the front of the cache; returns their number ``n`` (an int64 scalar).

    The k-th page in use at or past ``n`` moves to the k-th free page before ``n``, in all layers and with its
    scales and reference count; table entries that named it follow.  Pages from ``n`` on are free afterwards.
    """
    op = "kv_compact_paged_blocks"
    got = _hip.pages_native("compact", op, key_cache, value_cache, block_tables, None, ref_counts, None, k_scales,
                            v_scales, 0, 0)
    if got is not None:
        _emit(op, key_cache, "gfx950 page compaction")
        return got[1]
    _check_state(op, block_tables, None, ref_counts)
    block_size, pool = _check_pool(op, key_cache, value_cache, k_scales, v_scales, ref_counts)
    device = block_tables.device
    _require_rocm(op, block_tables)
    count = torch.empty((), dtype=torch.int64, device=device)
    _hip.pages("compact", op=op, device=device, tables=block_tables, lens=None, refs=ref_counts, rows=None,
               block_size=block_size, result=count, **pool)
    _emit(op, key_cache, "gfx950 page compaction")
    return count


__all__ = [
    "kv_extend_paged_sequences",
    "kv_fork_paged_sequences",
    "kv_free_paged_sequences",
    "kv_compact_paged_blocks",
]
