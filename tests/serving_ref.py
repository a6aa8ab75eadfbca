"""Plain 64-bit implementations of the block-scaled FP8 store, the attention over such a cache and the page
bookkeeping, one element or one step at a time on the CPU.  Oracles, not product code."""

from __future__ import annotations

import math

import numpy as np

# Mantissa bits, exponent bias, the largest value that a block's scale aims at.
FORMATS = {"e4m3": (3, 7, 448.0), "e5m2": (2, 15, 57344.0)}
SCALE_FLOOR = 2.0 ** -60


def decode_table(fmt: str) -> np.ndarray:
    """float64 value of every code."""
    mant, bias, _ = FORMATS[fmt]
    codes = np.arange(256)
    e, m = (codes & 127) >> mant, codes & ((1 << mant) - 1)
    v = np.where(e > 0, (1 + m / (1 << mant)) * 2.0 ** (e - bias), 0.0)
    return np.where(codes & 128, -v, v)


def encode32(x: np.ndarray, fmt: str) -> np.ndarray:
    """Codes of float32 quotients: round half to even, flush below the smallest normal, non-finite to a zero."""
    mant, bias, _ = FORMATS[fmt]
    emax = 8 if fmt == "e4m3" else 16
    x = x.astype(np.float32)
    a = np.abs(x.astype(np.float64))
    a = np.where(np.isfinite(a), a, 0.0)
    a = np.minimum(a, (2 - 2.0 ** -mant) * 2.0 ** emax)
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -40)))
    q = np.round(a / 2.0 ** (e - mant))                # in [2^mant, 2^(mant + 1)]
    e, q = np.where(q == 2 << mant, e + 1, e), np.where(q == 2 << mant, 1 << mant, q)
    code = ((e + bias) * (1 << mant) + (q - (1 << mant))).astype(np.int64)
    code = np.where(a < 2.0 ** (1 - bias), 0, code)
    return (code | np.where(x < 0, 128, 0)).astype(np.uint8)


def block_store(new: np.ndarray, cache: np.ndarray, scales: np.ndarray, slots: np.ndarray, fmt: str) -> None:
    """One layer and plane: new [T, H, D] float32, cache [NB, H, D, BS] uint8 and scales [NB, H] changed in place.
    The arithmetic is float32 with one rounding per operation, as the definition says."""
    top, bs = np.float32(FORMATS[fmt][2]), cache.shape[-1]
    table = decode_table(fmt).astype(np.float32)
    blocks: dict[int, dict[int, int]] = {}
    for t, slot in enumerate(slots.tolist()):
        if slot >= 0:
            blocks.setdefault(slot // bs, {})[slot % bs] = t
    with np.errstate(all="ignore"):
        for b, cols in blocks.items():
            for h in range(cache.shape[1]):
                x = np.stack([new[t, h] for t in cols.values()]).astype(np.float32)
                finite = x[np.isfinite(x)]
                most = np.float32(np.abs(finite).max()) if finite.size else np.float32(0)
                before = scales[b, h]
                anew = 0 in cols or not (before > 0 and np.isfinite(before))
                now = max(most / top, np.float32(SCALE_FLOOR))
                if not anew:
                    now = max(now, before)
                old = cache[b, h]
                if anew:
                    old = np.zeros_like(old)
                elif now != before:
                    old = encode32(table[old] * before / now, fmt)
                for c, row in zip(cols, x):
                    old[:, c] = encode32(row / now, fmt)
                cache[b, h], scales[b, h] = old, now


def attention(query, key, value, tables, lens, k_scales, v_scales, fmt, *, starts=None, scale=None, window=None):
    """float64 (out [T, Hq, D], lse [T, Hq], weight [T, Hq, D], spread [T, Hq], faint [T, Hq, D]) of float64 query and
    uint8 caches.

    weight is sum_j p_j |v_jd|, spread the largest sum_d |q_d k_jd| * |scale| that a row meets, and faint
    max_j(p_j vs_j) * sum_j |code_jd|: what the error of a computation in fewer bits grows with.  Rows of no
    sequence are NaN."""
    table = decode_table(fmt)
    rows, heads, hd = query.shape
    nb, nh, _, bs = key.shape
    scale = hd ** -0.5 if scale is None else scale
    starts = list(range(len(lens) + 1)) if starts is None else list(starts)
    out, lse = np.full(query.shape, np.nan), np.full((rows, heads), np.nan)
    weight, spread, faint = np.zeros(query.shape), np.zeros((rows, heads)), np.zeros(query.shape)
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        room = min(max(int(n), 0), tables.shape[1] * bs)
        blk = np.repeat(tables[b, :-(-room // bs)], bs)[:room].astype(np.int64)
        off = np.arange(room) % bs
        there = (blk >= 0) & (blk < nb)
        safe = np.where(there, blk, 0)
        for h in range(nh):
            k = table[key[safe, h, :, off]] * k_scales[safe, h][:, None]
            codes, vs = table[value[safe, h, :, off]], v_scales[safe, h]
            v = codes * vs[:, None]
            for t in range(lo, hi):
                pos = int(n) - (hi - lo) + (t - lo)
                j = np.arange(room)
                seen = there & (j <= pos) & (True if window is None else j > pos - window)
                for g in range(h * heads // nh, (h + 1) * heads // nh):
                    if not seen.any():
                        out[t, g], lse[t, g] = 0.0, -np.inf
                        continue
                    s = (k[seen] @ query[t, g]) * scale
                    p = np.exp(s - s.max())
                    lse[t, g] = s.max() + math.log(p.sum())
                    p /= p.sum()
                    out[t, g] = p @ v[seen]
                    weight[t, g] = p @ np.abs(v[seen])
                    faint[t, g] = (p * vs[seen]).max() * np.abs(codes[seen]).sum(axis=0)
                    spread[t, g] = (np.abs(k[seen]) @ np.abs(query[t, g])).max() * abs(scale)
    return out, lse, weight, spread, faint


class Pages:
    """The page bookkeeping, one row and one page at a time."""

    def __init__(self, tables, lens, refs, page: int):
        self.tables = [list(map(int, row)) for row in tables]
        self.lens, self.refs, self.page = list(map(int, lens)), list(map(int, refs)), page
        self.moves: list[tuple[int, int]] = []  # page copies, in order

    def owned(self, n: int) -> int:
        return -(-max(n, 0) // self.page)

    def add(self, row, first: int, last: int, by: int) -> None:
        for p in row[first:last]:
            if 0 <= p < len(self.refs):
                self.refs[p] += by

    def free(self, keep) -> None:
        for b, k in enumerate(keep):
            k = self.lens[b] if k < 0 or k > self.lens[b] else int(k)
            first, last = self.owned(k), self.owned(self.lens[b])
            self.add(self.tables[b], first, last, -1)
            for i in range(first, min(last, len(self.tables[b]))):
                self.tables[b][i] = -1
            self.lens[b] = k

    def fork(self, parents) -> None:
        width = len(self.tables[0]) if self.tables else 0
        new = []
        for b, p in enumerate(parents):
            inside = 0 <= p < len(self.tables)
            new.append((list(self.tables[p]), self.lens[p]) if inside else ([-1] * width, 0))
        for row, n in new:
            self.add(row, 0, self.owned(n), 1)
        for b, (row, n) in enumerate(new):
            self.add(self.tables[b], 0, self.owned(self.lens[b]), -1)
            self.tables[b], self.lens[b] = row, n

    def extend(self, new, most: int):
        new = [min(max(int(n), 0), most) for n in new]
        none = [[-1] * most for _ in new]
        if any(self.owned(self.lens[b] + n) > len(self.tables[b]) for b, n in enumerate(new)):
            return none, -(1 << 62)
        before = ([list(r) for r in self.tables], list(self.lens), list(self.refs), list(self.moves))
        free = [p for p, r in enumerate(self.refs) if r == 0]
        need, slots = 0, []

        def take():
            nonlocal need
            need += 1
            return free[need - 1] if need <= len(free) else None

        for b, n in enumerate(new):
            row, first = self.tables[b], self.lens[b]
            if n and first % self.page:
                last = row[self.owned(first) - 1]
                if 0 <= last < len(self.refs) and self.refs[last] > 1:
                    to = take()
                    self.refs[last] -= 1
                    if to is not None:
                        self.moves.append((last, to))
                        self.refs[to], row[self.owned(first) - 1] = 1, to
            for i in range(self.owned(first), self.owned(first + n)):
                to = take()
                if to is not None:
                    self.refs[to], row[i] = 1, to
            self.lens[b] = first + n
            slots.append([row[i // self.page] * self.page + i % self.page
                          if i < first + n and 0 <= row[i // self.page] < len(self.refs) else -1
                          for i in range(first, first + most)])
        if need > len(free):
            self.tables, self.lens, self.refs, self.moves = before
            return none, len(free) - need
        return slots, len(free) - need

    def compact(self) -> int:
        live = [p for p, r in enumerate(self.refs) if r > 0]
        holes = [p for p in range(len(live)) if self.refs[p] <= 0]
        to = {}
        for src, dst in zip([p for p in live if p >= len(live)], holes):
            self.moves.append((src, dst))
            self.refs[dst], self.refs[src], to[src] = self.refs[src], 0, dst
        self.tables = [[to.get(p, p) for p in row] for row in self.tables]
        return len(live)
