"""Attention over paged caches of plain values, the weight that cached tokens gather, and the eviction by it.

The caches are the paged ones of kv_transfer, ``[blocks, kv_heads, head_dim, block_size]`` of float32, float16 or
bfloat16.  Sequence ``b`` has ``seq_lens[b]`` cached tokens, position ``pos`` in slot
``block_tables[b, pos // block_size] * block_size + pos % block_size``; its query rows are its last tokens (stored
already).  Head ``h`` reads kv head ``h // (heads // kv_heads)``.

Tables, lengths, row starts, tree masks and the numbers of tokens to keep are read on the device only: nothing is
synchronised, and the calls can be captured into a graph.  They run on the current stream of the caches' device.
Shapes, types and devices are checked on the host and raise ``ValueError``; tensors that are not on a ROCm device raise
``RuntimeError``.  No counterpart in the reference, which leaves attention and eviction to its callers.
"""

from __future__ import annotations

import math

import torch

from musa_aiter.ops import _hip
from musa_aiter.ops.kv_block_cache import _index_rows, _overlaps, _packed_blocks, _spans_meet, _Written
from musa_aiter.ops.kv_transfer import (
    _INDEX_DTYPES,
    _LIN_DTYPE,
    _emit,
    _require_rocm,
    _validate_paged_shapes,
    _validate_stacked_paged_shapes,
)

_MAX_HEAD_DIM = 512
_MAX_ROOM = 1 << 29


def _blocks_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a packed block of one of two caches of the same shape shares bytes with one of the other."""
    if not _spans_meet(a, b):
        return False
    if any(n > 1 and s != t for n, s, t in zip(a.shape[:-3], a.stride(), b.stride())):
        return True  # not looked at further
    size = a.element_size()
    packed, apart = a[(0,) * (a.dim() - 3)].numel() * size, b.data_ptr() - a.data_ptr()
    layers, layer = (a.shape[0], a.stride(0) * size) if a.dim() == 5 else (1, 0)
    last = a.shape[-4] - 1
    block = a.stride(-4) * size if last else 1
    for i in range(1 - layers, layers):
        off = apart + i * layer
        near = -off // block
        if any(abs(off + min(max(j, -last), last) * block) < packed for j in (near, near + 1)):
            return True
    return False


class _Rows:
    """The checked arguments that the three operators on query rows share."""

    def __init__(self, op: str, query: torch.Tensor, caches: tuple[torch.Tensor, ...], block_tables: torch.Tensor,
                 seq_lens: torch.Tensor, query_starts: torch.Tensor | None, max_seq_len: int | None,
                 softmax_scale: float | None, window: int | None, sinks: int):
        if query.dim() != 3:
            raise ValueError(f"{op}: query must be [rows, heads, head_dim]")
        if query.dtype not in _LIN_DTYPE:
            raise ValueError(f"{op}: query must be float32, float16 or bfloat16, got {query.dtype}")
        nb, nh, hd, bs = _validate_paged_shapes(caches[0], caches[-1], name=op)
        if any(c.dtype != query.dtype for c in caches):
            raise ValueError(f"{op}: query and caches must share one dtype")
        rows, heads = int(query.shape[0]), int(query.shape[1])
        if int(query.shape[2]) != hd or hd > _MAX_HEAD_DIM:
            raise ValueError(f"{op}: query head_dim {int(query.shape[2])} must match the caches' {hd} (at most {_MAX_HEAD_DIM})")
        if heads < 1 or heads % nh:
            raise ValueError(f"{op}: heads ({heads}) must be a multiple of kv_heads ({nh})")
        if block_tables.dim() != 2:
            raise ValueError(f"{op}: block_tables must be [batch, max_blocks]")
        batch, width = map(int, block_tables.shape)
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
        if any(t.device != device for t in (*caches, *indices)):
            raise ValueError(f"{op}: all tensors must be on the same device")
        if rows * heads >= 1 << 31 or rows > _MAX_ROOM or heads > 65535 or width * bs > _MAX_ROOM:
            raise ValueError(f"{op}: at most 2**31 - 1 rows times heads, 65535 heads, 2**29 rows and 2**29 positions per sequence")
        if window is not None and window < 1:
            raise ValueError(f"{op}: window must be positive")
        if sinks < 0:
            raise ValueError(f"{op}: sinks must be non-negative")
        if max_seq_len is not None and max_seq_len < 0:
            raise ValueError(f"{op}: max_seq_len must be non-negative")
        scale = hd ** -0.5 if softmax_scale is None else float(softmax_scale)
        if not math.isfinite(scale):
            raise ValueError(f"{op}: softmax_scale must be finite")
        self.rows, self.heads, self.kv_heads, self.batch, self.room = rows, heads, nh, batch, width * bs
        self.query, self.device = query, device
        self._caches, self._indices = caches, (block_tables, seq_lens, query_starts)
        self.read = (query, *caches, *indices)
        self._shape = (rows, batch, heads, nh, hd, bs, nb, width)
        self._scale, self._window, self._sinks = scale, min(int(window or 0), _MAX_ROOM), min(int(sinks), _MAX_ROOM) if window else 0
        self._longest = width * bs if max_seq_len is None else min(int(max_seq_len), 1 << 62)

    def call(self) -> dict:
        """The arguments of the launch, in layouts that the kernels read."""
        query = self.query
        if query.shape[2] > 1 and query.stride(2) != 1:
            query = query.contiguous()
        tables, lens, starts = self._indices
        return dict(
            query=query, caches=[c if _packed_blocks(c) else c.contiguous() for c in self._caches],
            tables=_index_rows(tables), lens=_index_rows(lens), starts=None if starts is None else _index_rows(starts),
            sizes=self._shape, window=self._window, sinks=self._sinks, longest=self._longest,
            softmax_scale=self._scale, dtype=_LIN_DTYPE[query.dtype])


def _native_sight(query: torch.Tensor, max_seq_len, softmax_scale, window, sinks) -> tuple | None:
    """(longest, scale, window, sinks) as the host module takes them, or None for what the checks have to look at."""
    if not (window is None or type(window) is int and 0 < window < 1 << 62) \
            or not (type(sinks) is int and 0 <= sinks < 1 << 62) \
            or not (max_seq_len is None or type(max_seq_len) is int and 0 <= max_seq_len < 1 << 62) \
            or not (softmax_scale is None or type(softmax_scale) is float and math.isfinite(softmax_scale)) \
            or query.dim() != 3 or query.shape[2] < 1:
        return None
    return (-1 if max_seq_len is None else max_seq_len, query.shape[2] ** -0.5 if softmax_scale is None else softmax_scale,
            window or 0, sinks)


def _attention(op: str, rows: _Rows, masks: torch.Tensor | None, out: torch.Tensor | None, return_lse: bool):
    query, device = rows.query, rows.device
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or out.device != device):
        raise ValueError(f"{op}: out must match query's shape, dtype and device")
    if out is not None and out.numel() and _overlaps(out):
        raise ValueError(f"{op}: out is written and must not be expanded")
    _require_rocm(op, query)
    result = torch.empty(query.shape, dtype=query.dtype, device=device) if out is None else out
    read = rows.read if masks is None else (*rows.read, masks)
    target = _Written(result, result.is_contiguous() and (out is None or not any(_spans_meet(out, t) for t in read)))
    lse = torch.empty((rows.rows, rows.heads), dtype=torch.float32, device=device) if return_lse else None
    _hip.paged_attention(op=op, out=target.t, lse=lse, masks=masks, fill_rows=out is None, **rows.call())
    target.finish()
    return (result, lse) if return_lse else result


def kv_paged_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    query_starts: torch.Tensor | None = None,
    max_seq_len: int | None = None,
    softmax_scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Causal attention of ``query`` rows ``[T, heads, head_dim]`` over paged caches of the same type.

    The rows of sequence ``b`` are ``query_starts[b] : query_starts[b + 1]`` (ascending), its last tokens; without ``query_starts``
    every sequence has one row (a decode step).  Row ``i`` of ``n`` sits at position ``seq_lens[b] - n + i`` and sees
    the positions up to there: all of them, or with ``window`` the last ``window`` and next to them the sequence's
    first ``sinks`` (their pages may be the only ones in front of the window that are still there).
    ``softmax_scale`` is ``head_dim ** -0.5`` by default.

    A position without a table entry, or whose entry lies outside the cache, is not seen.  A row that sees nothing
    gives zeros (``lse`` -inf).  Rows of ``query`` that belong to no sequence (a padded batch) are left as they are in
    ``out``, and are zeros in a new tensor; their ``lse`` is -inf either way.  What positions that a row does not see
    hold does not reach it, infinities and NaN included.  An ``out`` that shares memory with an argument, ``query``
    itself among them, is computed apart and copied.

    ``max_seq_len``, an upper bound of ``seq_lens`` that the caller knows, only decides how the work is cut; by
    default it is what ``block_tables`` has room for.  Returns the output, in ``query``'s type, and with
    ``return_lse`` also the float32 ``[T, heads]`` logarithms of the rows' softmax sums.  There is no backward pass:
    the output carries no gradient, also where ``query`` requires one.

    Scores, softmax statistics and sums are float32.  With 16-bit caches a weight enters its products as two numbers of
    their type, 2**-16 (float16 2**-22) of it off at most; float16 ones lose what lies below 2**-28 of a row's largest.
    With float32 caches no weight is rounded.
    """
    op = "kv_paged_attention"
    sight = _native_sight(query, max_seq_len, softmax_scale, window, sinks)
    if sight is not None:
        got = _hip.paged_attention_native(op, query, key_cache, value_cache, block_tables, seq_lens, None, query_starts,
                                          out, *sight, return_lse)
        if got is not None:
            _emit(op, query, "gfx950 paged attention")
            return got if return_lse else got[0]
    rows = _Rows(op, query, (key_cache, value_cache), block_tables, seq_lens, query_starts, max_seq_len, softmax_scale,
                 window, sinks)
    got = _attention(op, rows, None, out, return_lse)
    _emit(op, query, "gfx950 paged attention")
    return got


def kv_paged_attention_tree(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    tree_masks: torch.Tensor,
    *,
    query_starts: torch.Tensor | None = None,
    max_seq_len: int | None = None,
    softmax_scale: float | None = None,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """Attention of trees of drafted tokens over paged caches: kv_paged_attention, with masks among a sequence's rows.

    The ``n`` rows of a sequence are its last ``n`` cached tokens (drafts, stored already, in any order in which the
    caller numbers the tree).  Each row sees all ``seq_lens[b] - n`` tokens in front of them, and of the drafts those
    that its mask names: bit ``k % 64`` of ``tree_masks[row, k // 64]`` (int64 ``[T, words]``) stands for the
    sequence's draft ``k``, the row itself included.  Drafts past ``64 * words`` are not seen, and bits past the
    sequence's drafts mean nothing.

    Everything else is as in kv_paged_attention.
    """
    op = "kv_paged_attention_tree"
    sight = _native_sight(query, max_seq_len, softmax_scale, None, 0)
    if sight is not None and tree_masks is not None:
        got = _hip.paged_attention_native(op, query, key_cache, value_cache, block_tables, seq_lens, tree_masks,
                                          query_starts, out, *sight, return_lse)
        if got is not None:
            _emit(op, query, "gfx950 paged attention of draft trees")
            return got if return_lse else got[0]
    rows = _Rows(op, query, (key_cache, value_cache), block_tables, seq_lens, query_starts, max_seq_len, softmax_scale,
                 None, 0)
    if tree_masks.dim() != 2 or tree_masks.shape[0] != rows.rows or tree_masks.shape[1] < 1:
        raise ValueError(f"{op}: tree_masks must be [rows, words]")
    if tree_masks.dtype is not torch.int64:
        raise ValueError(f"{op}: tree_masks must be int64, got {tree_masks.dtype}")
    if tree_masks.device != rows.device:
        raise ValueError(f"{op}: all tensors must be on the same device")
    got = _attention(op, rows, _index_rows(tree_masks), out, return_lse)
    _emit(op, query, "gfx950 paged attention of draft trees")
    return got


def kv_accumulate_attention_weights(
    weights: torch.Tensor,
    query: torch.Tensor,
    key_cache: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    lse: torch.Tensor,
    *,
    query_starts: torch.Tensor | None = None,
    max_seq_len: int | None = None,
    softmax_scale: float | None = None,
    window: int | None = None,
    sinks: int = 0,
) -> None:
    """Add to ``weights[b, kv_head, pos]`` the attention weight that position ``pos`` got from the rows.

    That is the sum of ``exp(score - lse)`` over the rows of sequence ``b`` that see the position and over the heads
    of the kv head, with the ``lse`` ``[T, heads]`` that kv_paged_attention returned for the same arguments.
    ``weights`` is float32 ``[batch, kv_heads, tokens]``; positions past its last extent are passed over.  Rows whose
    ``lse`` is -inf give nothing.  Sums are float32 and made in the same order in every call: no atomics.
    """
    op = "kv_accumulate_attention_weights"
    sight = _native_sight(query, max_seq_len, softmax_scale, window, sinks)
    if sight is not None and _hip.attention_weights_native(op, weights, query, key_cache, block_tables, seq_lens, lse,
                                                           query_starts, *sight):
        _emit(op, query, "gfx950 gathered attention weights")
        return
    rows = _Rows(op, query, (key_cache,), block_tables, seq_lens, query_starts, max_seq_len, softmax_scale, window,
                 sinks)
    if weights.dim() != 3 or tuple(weights.shape[:2]) != (rows.batch, rows.kv_heads):
        raise ValueError(f"{op}: weights must be [batch, kv_heads, tokens]")
    if tuple(lse.shape) != (rows.rows, rows.heads):
        raise ValueError(f"{op}: lse must be [rows, heads]")
    if weights.dtype is not torch.float32 or lse.dtype is not torch.float32:
        raise ValueError(f"{op}: weights and lse must be float32")
    if weights.device != rows.device or lse.device != rows.device:
        raise ValueError(f"{op}: all tensors must be on the same device")
    if weights.numel() and _overlaps(weights):
        raise ValueError(f"{op}: weights are written and must not be expanded")
    if rows.batch > 65535 or rows.kv_heads > 65535:
        raise ValueError(f"{op}: at most 65535 sequences and kv_heads")
    _require_rocm(op, query)
    target = _Written(weights, weights.shape[2] <= 1 or weights.stride(2) == 1)
    _hip.attention_weights(op=op, weights=target.t, lse=lse.contiguous(), **rows.call())
    target.finish()
    _emit(op, query, "gfx950 gathered attention weights")


def kv_evict_paged_tokens(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    weights: torch.Tensor,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    keep_lens: torch.Tensor,
    *,
    sinks: int = 0,
    recent: int = 0,
    ref_counts: torch.Tensor | None = None,
) -> torch.Tensor:
    """Cut every sequence to the ``keep_lens[b]`` tokens that count most, in every kv head on its own.

    Each kv head keeps the first ``sinks`` tokens, the last ``recent`` and, up to ``keep_lens[b]`` in all, those
    between with the largest ``weights`` (float32 ``[batch, kv_heads, tokens]``, as kv_accumulate_attention_weights
    gathers them); of equal weights the earlier token stays, a NaN counts as lighter than any number and a position
    past the last extent of ``weights`` as 0.  Where ``keep_lens[b]`` does not hold both, the first go before the last.
    The kept tokens move, in their order, to positions ``0 .. keep_lens[b] - 1`` of the sequence's pages, and their
    weights with them; the weights of the positions behind, up to ``seq_lens[b]``, become 0.  With stacked caches
    ``[L, NB, H, D, BS]`` the weights are ``[L, batch, kv_heads, tokens]`` and every layer chooses for itself.
    Elements are moved as they are, of any 1-, 2- or 4-byte type (not block-scaled codes, whose scales would not move).

    Returns the sequences' new lengths, int64 ``[batch]``; ``kv_free_paged_sequences`` with these as its ``keep_lens``
    then cuts the table rows and releases the pages behind.  A sequence stays as it is, and its length is returned,
    where ``keep_lens[b]`` is negative or not below it, where a page of it is missing or outside the cache, and where
    ``ref_counts`` (as in kv_pages) is given and counts another owner of one of its pages.  Without ``ref_counts`` the
    caller knows that no two sequences share a page.
    """
    op = "kv_evict_paged_tokens"
    if type(sinks) is int and 0 <= sinks < 1 << 62 and type(recent) is int and 0 <= recent < 1 << 62:
        kept = _hip.evict_native(op, key_cache, value_cache, weights, block_tables, seq_lens, keep_lens, ref_counts,
                                 sinks, recent)
        if kept is not None:
            _emit(op, key_cache, "gfx950 eviction by gathered weight")
            return kept
    if key_cache.dtype != value_cache.dtype or key_cache.element_size() not in (1, 2, 4):
        raise ValueError(f"{op}: caches must share one dtype of 1, 2 or 4 bytes")
    layered = key_cache.dim() == 5
    nl, nb, nh, hd, bs = (_validate_stacked_paged_shapes(key_cache, value_cache, name=op) if layered else
                          (1, *_validate_paged_shapes(key_cache, value_cache, name=op)))
    if block_tables.dim() != 2:
        raise ValueError(f"{op}: block_tables must be [batch, max_blocks]")
    batch, width = map(int, block_tables.shape)
    for name, t in (("seq_lens", seq_lens), ("keep_lens", keep_lens)):
        if t.dim() != 1 or t.shape[0] != batch:
            raise ValueError(f"{op}: {name} must be [batch]")
    if ref_counts is not None and (ref_counts.dim() != 1 or ref_counts.shape[0] != nb):
        raise ValueError(f"{op}: ref_counts must be [blocks] ({nb})")
    lead = (nl,) if layered else ()
    if weights.dim() != 3 + layered or tuple(weights.shape[:-1]) != (*lead, batch, nh):
        raise ValueError(f"{op}: weights must be {'[layers, ' if layered else '['}batch, kv_heads, tokens]")
    if weights.dtype is not torch.float32:
        raise ValueError(f"{op}: weights must be float32, got {weights.dtype}")
    indices = [t for t in (block_tables, seq_lens, keep_lens, ref_counts) if t is not None]
    if any(t.dtype not in _INDEX_DTYPES for t in indices):
        raise ValueError(f"{op}: block_tables, seq_lens, keep_lens and ref_counts must be integer tensors")
    device = key_cache.device
    if any(t.device != device for t in (value_cache, weights, *indices)):
        raise ValueError(f"{op}: all tensors must be on the same device")
    if any(not _packed_blocks(c) or _overlaps(c) for c in (key_cache, value_cache)):
        raise ValueError(f"{op}: the blocks of the caches are written and must be contiguous")
    if key_cache.data_ptr() == value_cache.data_ptr():
        raise ValueError(f"{op}: key_cache and value_cache are moved each on its own and must not be one tensor")
    if _blocks_meet(key_cache, value_cache):
        raise ValueError(f"{op}: key_cache and value_cache are moved each on its own and must not share memory")
    if weights.numel() and _overlaps(weights):
        raise ValueError(f"{op}: weights are written and must not be expanded")
    if sinks < 0 or recent < 0:
        raise ValueError(f"{op}: sinks and recent must be non-negative")
    if width * bs > _MAX_ROOM or hd > 65535 or nl * batch * nh >= 1 << 31:
        raise ValueError(f"{op}: at most 2**29 positions per sequence, 65535 dims and 2**31 - 1 layers times batch times kv_heads")
    _require_rocm(op, key_cache)
    kept = torch.empty(batch, dtype=torch.int64, device=device)
    target = _Written(weights, weights.shape[-1] <= 1 or weights.stride(-1) == 1)
    _hip.evict(op=op, caches=(key_cache, value_cache), weights=target.t, tables=_index_rows(block_tables),
               lens=_index_rows(seq_lens), keep=_index_rows(keep_lens),
               refs=None if ref_counts is None else _index_rows(ref_counts), kept=kept,
               sizes=(nl, batch, nh, hd, bs, nb, width), sinks=min(int(sinks), _MAX_ROOM),
               recent=min(int(recent), _MAX_ROOM))
    target.finish()
    _emit(op, key_cache, "gfx950 eviction by gathered weight")
    return kept


__all__ = [
    "kv_paged_attention",
    "kv_paged_attention_tree",
    "kv_accumulate_attention_weights",
    "kv_evict_paged_tokens",
]
