"""Plain 64-bit implementations of the attention over paged caches of plain values (windows, first tokens, trees), of
the weight that cached tokens gather, and of the eviction by it.  Oracles on the CPU, not product code."""

from __future__ import annotations

import numpy as np


def _seen(n: int, rows: int, window, sinks: int, masks) -> np.ndarray:
    """[rows, max(n, 0)]: which positions each of a sequence's rows sees."""
    j = np.arange(max(n, 0))
    seen = np.zeros((rows, max(n, 0)), dtype=bool)
    for i in range(rows):
        if masks is None:
            at = n - rows + i
            seen[i] = j <= at
            if window is not None:
                seen[i] &= (j > at - window) | (j < sinks)
        else:
            words = [int(w) for w in masks[i]]
            for p in range(max(n, 0)):
                k = p - (n - rows)
                seen[i, p] = k < 0 or (k < 64 * len(words) and (words[k // 64] >> (k % 64)) & 1 != 0)
    return seen


class Rows:
    """Scores of every (row, head): ``each`` yields (row, head, kv head, sequence, positions seen, scores there,
    values there, the sizes that their rounding errors grow with)."""

    def __init__(self, query, key, value, tables, lens, *, starts=None, scale=None, window=None, sinks=0, masks=None):
        self.query, self.key, self.value = (np.asarray(x, dtype=np.float64) for x in (query, key, value))
        self.tables, self.lens = np.asarray(tables), [int(n) for n in lens]
        self.starts = list(range(len(self.lens) + 1)) if starts is None else [int(s) for s in starts]
        self.scale = query.shape[2] ** -0.5 if scale is None else scale
        self.window, self.sinks, self.masks = window, sinks, masks

    def each(self):
        nb, nh, _, bs = self.key.shape
        heads = self.query.shape[1]
        for b, n in enumerate(self.lens):
            lo, hi = self.starts[b], self.starts[b + 1]
            if not 0 <= lo <= hi <= self.query.shape[0]:
                continue
            rows = None if self.masks is None else self.masks[lo:hi]
            seen = _seen(n, hi - lo, self.window, self.sinks, rows)
            room = min(max(n, 0), self.tables.shape[1] * bs)
            blk = np.repeat(self.tables[b, :-(-room // bs)], bs)[:room].astype(np.int64)
            off = np.arange(room) % bs
            there = (blk >= 0) & (blk < nb)
            safe = np.where(there, blk, 0)
            for h in range(nh):
                k, v = self.key[safe, h, :, off], self.value[safe, h, :, off]
                for t in range(lo, hi):
                    at = np.nonzero(there & seen[t - lo, :room])[0]
                    for g in range(h * heads // nh, (h + 1) * heads // nh):
                        q = self.query[t, g]
                        with np.errstate(all="ignore"):
                            yield t, g, h, b, at, (k[at] @ q) * self.scale, v[at], np.abs(k[at]) @ np.abs(q) * abs(self.scale)


def attention(query, key, value, tables, lens, **more):
    """float64 (out, lse, weight, spread, faint): weight is sum_j p_j |v_jd|, spread the largest sum_d |q_d k_jd| *
    |scale| of a row, faint max_j(p_j) * sum_j |v_jd|.  Rows of no sequence are NaN."""
    out, lse = np.full(query.shape, np.nan), np.full(query.shape[:2], np.nan)
    weight, spread, faint = np.zeros(query.shape), np.zeros(query.shape[:2]), np.zeros(query.shape)
    for t, g, _, _, at, s, v, size in Rows(query, key, value, tables, lens, **more).each():
        if at.size == 0:
            out[t, g], lse[t, g] = 0.0, -np.inf
            continue
        with np.errstate(all="ignore"):
            p = np.exp(s - s.max())
            lse[t, g] = s.max() + np.log(p.sum())
            p /= p.sum()
            out[t, g] = p @ v
            weight[t, g] = p @ np.abs(v)
            faint[t, g] = p.max() * np.abs(v).sum(axis=0)
        spread[t, g] = size.max()
    return out, lse, weight, spread, faint


def gathered(weights, query, key, tables, lens, lse, **more):
    """float64 (weights after the call, the largest sizes of scores behind each, how many terms each gained)."""
    out, spread, terms = np.array(weights, dtype=np.float64), np.zeros(weights.shape), np.zeros(weights.shape)
    tokens = weights.shape[2]
    for t, g, h, b, at, s, _, size in Rows(query, key, key, tables, lens, **more).each():
        if np.isneginf(lse[t, g]):
            continue
        keep = at < tokens
        at, s, size = at[keep], s[keep], size[keep]
        with np.errstate(all="ignore"):
            out[b, h, at] += np.exp(s - float(lse[t, g]))
        spread[b, h, at] = np.maximum(spread[b, h, at], size + abs(float(lse[t, g])))
        terms[b, h, at] += 1
    return out, spread, terms


def evict(key, value, weights, tables, lens, keep, *, sinks=0, recent=0, refs=None):
    """One layer: key and value [NB, H, D, BS] and weights [B, H, M] float32 changed in place; returns the lengths."""
    nb, nh, _, bs = key.shape
    kept = []
    old = key.copy(), value.copy()
    for b, n in enumerate(int(x) for x in lens):
        k, n = int(keep[b]), max(n, 0)
        pages = [int(p) for p in tables[b, :-(-n // bs)]]
        whole = n <= tables.shape[1] * bs and all(0 <= p < nb for p in pages)
        if k < 0 or k >= n or not whole or (refs is not None and any(refs[p] > 1 for p in pages)):
            kept.append(n)
            continue
        kept.append(k)
        first = min(sinks, k)
        last = min(recent, k - first)
        for h in range(nh):
            w = np.zeros(n, dtype=np.float32)
            w[:min(n, weights.shape[2])] = weights[b, h, :n]
            rank = np.where(np.isnan(w), -np.inf, w)
            # Heavier first; a NaN behind -inf; of equal ones the earlier.
            middle = sorted(range(first, n - last), key=lambda p: (-rank[p], bool(np.isnan(w[p])), p))
            stay = [*range(first), *sorted(middle[:k - first - last]), *range(n - last, n)]
            for dst, src in enumerate(stay):
                for new, was in ((key, old[0]), (value, old[1])):
                    new[pages[dst // bs], h, :, dst % bs] = was[pages[src // bs], h, :, src % bs]
            fresh = np.zeros(n, dtype=np.float32)
            fresh[:k] = w[stay]
            weights[b, h, :n] = fresh[:min(n, weights.shape[2])]
    return np.asarray(kept)
