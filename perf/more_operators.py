"""Workloads of the operators on 16-bit paged caches: attention with a sliding window and first tokens that stay
visible, attention for trees of drafted tokens, the attention weight that every cached token gathers, and the eviction
of the tokens that gathered least.

A case is a dict of plain values.  ``listed()`` names the cases that are measured by default, ``draw()`` makes
further ones over the same ranges, ``prepare()`` builds a case's inputs on the GPU and ``run()`` makes one pass:
with ``own`` through the public entry points, else in plain torch operations, written from the definitions below.
``exact()`` gives the same outputs in 64 bits.

Caches are ``[blocks, kv_heads, head_dim, page]`` (evictions: one more leading extent, the layers).  Sequence b has
``lens[b]`` cached tokens, position j in page ``tables[b, j // page]``, place ``j % page``.  Its n query rows are its
last n tokens; head h reads kv head ``h // (heads // kv_heads)``.

* ``attention``: row i sits at position ``at = len - n + i`` and sees the positions up to there; with a window only the
  last ``window`` of them and the first ``sinks`` of the sequence.  Returned with the logarithms of the softmax sums.
* ``tree``: the n rows are drafted tokens.  Each sees the ``len - n`` tokens in front of them, and of the drafted ones
  those whose bit is set in its mask (its ancestors and itself).
* ``weights``: to ``weights[b, kv head, j]`` is added what the rows' softmax gives position j, summed over the rows and
  the heads of the kv head, with the logarithms that the attention returned.
* ``evict``: every layer, row and kv head keeps ``keep`` tokens: the first ``sinks``, the last ``recent`` and the
  heaviest of the others (of equal ones the earliest).  They move, in order, to the front of the row's pages, and their
  weights with them; the weights behind become 0.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed() -> list[dict]:
    return [
        # A decode step of a few short chats that see their last 128 tokens: launch latency counts.
        {"name": "recent_small", "path": "attention", "batch": 4, "q_lo": 1, "q_hi": 1, "pad": 0, "len_lo": 17,
         "len_hi": 500, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 128, "sinks": 4,
         "dtype": "bf16"},
        # A full decode batch of ragged lengths, everything visible: the cache is read once, at memory speed.
        {"name": "decode_batch", "path": "attention", "batch": 48, "q_lo": 1, "q_hi": 1, "pad": 0, "len_lo": 256,
         "len_hi": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # Long streams that keep their first 64 tokens next to a window: what lies between them is not read.
        {"name": "streams_batch", "path": "attention", "batch": 16, "q_lo": 1, "q_hi": 1, "pad": 3, "len_lo": 2001,
         "len_hi": 16001, "heads": 40, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 2048, "sinks": 64,
         "dtype": "fp16"},
        # Prompt chunks against a cached prefix, a window and four sinks: matrix products, not bandwidth.
        {"name": "prompt_chunks", "path": "attention", "batch": 2, "q_lo": 1500, "q_hi": 2048, "pad": 0,
         "len_lo": 4096, "len_hi": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 4000,
         "sinks": 4, "dtype": "bf16"},
        # Trees of a few drafted tokens of three short chats.
        {"name": "tree_small", "path": "tree", "batch": 3, "q_lo": 7, "q_hi": 13, "pad": 0, "len_lo": 20,
         "len_hi": 400, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "bf16"},
        # A batch of wide trees over contexts of ragged lengths, in a padded batch.
        {"name": "tree_batch", "path": "tree", "batch": 16, "q_lo": 33, "q_hi": 64, "pad": 5, "len_lo": 500,
         "len_hi": 4001, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "bf16"},
        # The weights of a decode step, gathered at every token.
        {"name": "weights_decode", "path": "weights", "batch": 16, "q_lo": 1, "q_hi": 1, "pad": 0, "len_lo": 300,
         "len_hi": 4097, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0, "sinks": 0,
         "dtype": "bf16"},
        # The weights of two prompt chunks: as many products as half of their attention.
        {"name": "weights_chunks", "path": "weights", "batch": 2, "q_lo": 600, "q_hi": 1024, "pad": 0, "len_lo": 2000,
         "len_hi": 6001, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "window": 0, "sinks": 0,
         "dtype": "fp16"},
        # A few short rows of one layer cut to 128 tokens.
        {"name": "evict_small", "path": "evict", "batch": 3, "layers": 1, "len_lo": 200, "len_hi": 500, "keep": 128,
         "sinks": 4, "recent": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "bf16"},
        # A batch cut to 1024 tokens in all layers of a small model: hundreds of megabytes are read and moved.
        {"name": "evict_batch", "path": "evict", "batch": 8, "layers": 8, "len_lo": 900, "len_hi": 6000, "keep": 1024,
         "sinks": 4, "recent": 256, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "bf16"},
        # One long document: a fifth of it stays.
        {"name": "evict_long", "path": "evict", "batch": 1, "layers": 2, "len_lo": 40001, "len_hi": 40001,
         "keep": 8000, "sinks": 16, "recent": 500, "kv_heads": 8, "head_dim": 128, "page": 64, "dtype": "fp16"},
    ]


# What a drawn case may cost at most (the largest listed one of its path does).
MAX_DENSE = 3.2e8       # values of K in a dense batch
MAX_SCORES = 9.0e8      # scores of a dense batch
MAX_PRODUCTS = 1.2e11   # products of the scores with one side
MAX_POOL = 4.5e8        # values of K that evictions look at


def _log_int(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng) -> dict:
    path = rng.choice(["attention", "attention", "attention", "tree", "tree", "weights", "evict", "evict"])
    head_dim, page = rng.choice([64, 96, 128, 128, 256]), rng.choice([16, 16, 32, 64])
    kv_heads, dtype = rng.choice([1, 2, 4, 8, 8]), rng.choice(["bf16", "bf16", "fp16"])
    shape = {"kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}
    if path == "evict":
        layers, batch = rng.choice([1, 2, 4, 8]), _log_int(rng, 1, 16)
        len_hi = _log_int(rng, 40, min(40000.0, MAX_POOL / (layers * batch * kv_heads * head_dim)))
        keep = max(1, int(len_hi * rng.choice([0.05, 0.2, 0.5, 0.9])))
        return {"path": path, "batch": batch, "layers": layers, "len_lo": max(1, len_hi // rng.choice([1, 2, 10])),
                "len_hi": len_hi, "keep": keep, "sinks": rng.choice([0, 4, 16]), "recent": keep // rng.choice([1, 3, 20]),
                **shape}
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    kind = "tree" if path == "tree" else rng.choice(["decode", "decode", "verify", "prompt"])
    q_hi = {"decode": 1, "verify": rng.randrange(2, 17), "prompt": _log_int(rng, 64, 2048),
            "tree": _log_int(rng, 2, 150)}[kind]
    batch = rng.randrange(1, 4) if kind == "prompt" else _log_int(rng, 1, 48)
    most = min(MAX_DENSE / (batch * kv_heads * head_dim), MAX_SCORES / (batch * heads * q_hi),
               MAX_PRODUCTS / (batch * heads * q_hi * head_dim), 100000.0)
    len_hi = max(q_hi, _log_int(rng, 16, max(32.0, most)))
    case = {"path": path, "batch": batch, "q_lo": max(1, q_hi // 2), "q_hi": q_hi, "pad": rng.choice([0, 0, 7]),
            "len_lo": max(1, len_hi // rng.choice([1, 3, 30])), "len_hi": len_hi, "heads": heads, **shape}
    if path != "tree":
        window = rng.choice([0, 0, _log_int(rng, 8, 4096)])
        case.update(window=window, sinks=rng.choice([0, 1, 4, 100]) if window else 0)
    return case


# ----- inputs -----------------------------------------------------------------------------------


def _device() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _on(device, values, dtype=torch.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(np.asarray(values, dtype=np.int64))).to(device=device, dtype=dtype)


def _values(gen, shape, dtype) -> torch.Tensor:
    """Normal values, one layer at a time, whose size varies by channel (the last extent but one)."""
    out = torch.empty(shape, dtype=dtype, device=gen.device)
    channel = torch.exp(0.3 * torch.randn((shape[-2], 1), generator=gen, device=gen.device))
    for part in (out if len(shape) == 5 else out[None]):
        part.copy_(torch.randn(part.shape, generator=gen, device=gen.device).mul_(channel))
    return out


def _lengths(rng, case) -> tuple[np.ndarray, np.ndarray]:
    """Cached tokens and query rows of each sequence, uniform in their ranges (one of them the longest).  The seed
    deals them out to the sequences: what they add up to, and so every output's shape, belongs to the case."""
    own_rng, count = np.random.default_rng(20), case["batch"]
    lens = own_rng.integers(case["len_lo"], case["len_hi"] + 1, size=count)
    lens[0] = case["len_hi"]
    rows = own_rng.integers(case.get("q_lo", 1), case.get("q_hi", 1) + 1, size=count)
    rows[0] = case.get("q_hi", 1)
    deal = rng.permutation(count)
    return lens[deal], np.minimum(rows, lens)[deal]


def _tables(rng, lens, page: int) -> tuple[np.ndarray, int]:
    """Page tables over a pool in random order, and the pool's pages."""
    pages = -(-lens // page)
    blocks = int(pages.sum()) + 7
    order, used = rng.permutation(blocks), 0
    tables = np.full((len(lens), int(pages.max())), -1, dtype=np.int64)
    for b, k in enumerate(pages):
        tables[b, :k] = order[used:used + k]
        used += int(k)
    return tables, blocks


def _tree_masks(rng, rows, total: int, words: int) -> np.ndarray:
    """Bits of each row's ancestors and itself; a row's parent is one of the rows before it, or the context."""
    masks, first = np.zeros((total, words), dtype=np.uint64), 0
    for n in rows:
        seen = [0] * int(n)
        for i in range(int(n)):
            parent = int(rng.integers(max(-1, i - 12), i)) if i else -1
            seen[i] = (seen[parent] if parent >= 0 else 0) | 1 << i
            for w in range(words):
                masks[first + i, w] = seen[i] >> 64 * w & (1 << 64) - 1
        first += int(n)
    return masks.view(np.int64)


def _query_inputs(case, gen, rng) -> dict:
    lens, queries = _lengths(rng, case)
    tables, blocks = _tables(rng, lens, case["page"])
    shape, dtype = (blocks, case["kv_heads"], case["head_dim"], case["page"]), DTYPES[case["dtype"]]
    rows = int(queries.sum()) + case["pad"]
    query = torch.randn((rows, case["heads"], case["head_dim"]), generator=gen, device=gen.device).mul_(1.5)
    starts = np.concatenate([[0], np.cumsum(queries)])
    state = {"query": query.to(dtype), "key": _values(gen, shape, dtype), "tables": _on(gen.device, tables),
             "lens": _on(gen.device, lens), "longest": int(lens.max()), "most_rows": int(queries.max()),
             # One row per sequence needs no row table; a padded or ragged batch comes with one.
             "starts": None if case["q_hi"] == 1 and not case["pad"] else _on(gen.device, starts), "masks": None}
    if case["path"] == "tree":
        state["masks"] = _on(gen.device, _tree_masks(rng, queries, rows, -(-case["q_hi"] // 64)), torch.int64)
    if case["path"] != "weights":
        return {**state, "value": _values(gen, shape, dtype)}
    # What the attention before returned, and weights that earlier steps gathered.
    scores, _, place, _ = _scores({"case": case, **state})
    lse = torch.full((rows, case["heads"]), -math.inf, device=gen.device)
    lse[place[0]] = torch.logsumexp(scores, dim=-1).view(*_split(case), -1).permute(0, 3, 1, 2).flatten(2)[place[1]]
    del scores
    lead = (case["batch"], case["kv_heads"], -(-state["longest"] // case["page"]) * case["page"])
    return {**state, "lse": lse, "weights": torch.rand(lead, generator=gen, device=gen.device).pow_(8)}


def _evict_inputs(case, gen, rng) -> dict:
    lens, _ = _lengths(rng, case)
    tables, blocks = _tables(rng, lens, case["page"])
    shape = (case["layers"], blocks, case["kv_heads"], case["head_dim"], case["page"])
    dtype = DTYPES[case["dtype"]]
    longest = int(lens.max())
    # Sums of softmax weights: over orders of magnitude, and the last few tokens have none yet.
    gathered = torch.exp(2.0 * torch.randn((case["layers"], case["batch"], case["kv_heads"],
                                            tables.shape[1] * case["page"]), generator=gen, device=gen.device))
    gathered[..., -max(1, case["recent"] // 2):] = 0.0
    return {"key": _values(gen, shape, dtype), "value": _values(gen, shape, dtype), "tables": _on(gen.device, tables),
            "lens": _on(gen.device, lens), "longest": longest, "keep": _on(gen.device, np.full(len(lens), case["keep"])),
            "gathered": gathered, "weights": torch.empty_like(gathered)}


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=_device()).manual_seed(seed)
    make = _evict_inputs if case["path"] == "evict" else _query_inputs
    return {"case": case, **make(case, gen, np.random.default_rng(seed))}


# ----- the plain forms --------------------------------------------------------------------------


def _split(case: dict) -> tuple[int, int, int]:
    return case["batch"], case["kv_heads"], case["heads"] // case["kv_heads"]


def _dense(s: dict, cache: torch.Tensor) -> torch.Tensor:
    """float32 [batch, kv_heads, head_dim, tokens] of a cache's pages."""
    case = s["case"]
    tables = s["tables"][:, :-(-s["longest"] // case["page"])].long().clamp(min=0)
    x = cache[tables].permute(0, 2, 3, 1, 4).float()
    return x.reshape(case["batch"], case["kv_heads"], case["head_dim"], -1)


def _scores(s: dict):
    """float32 scores [batch, kv_heads, group * rows, tokens], -inf where a row does not see, which of them are seen,
    the places of the rows (in ``query`` and in the dense batch), and the dense rows."""
    case, query = s["case"], s["query"]
    batch, hk, group = _split(case)
    hd, most, device, lens = case["head_dim"], s["most_rows"], query.device, s["lens"].long()
    starts = torch.arange(batch + 1, device=device) if s["starts"] is None else s["starts"].long()
    i = torch.arange(most, device=device)
    n = starts[1:] - starts[:-1]
    there = i < n[:, None]
    rows = torch.where(there, starts[:-1, None] + i, 0)
    q = query[rows].float().view(batch, most, hk, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, hd)
    scores = torch.matmul(q, _dense(s, s["key"])).mul_(1.0 / math.sqrt(hd))
    j = torch.arange(scores.shape[-1], device=device)
    if s["masks"] is None:
        at = ((lens - n)[:, None] + i)[..., None]
        seen = j <= at
        if case["window"]:
            seen = seen & ((j > at - case["window"]) | (j < case["sinks"]))
    else:
        bit = j - (lens - n)[:, None]                                   # [batch, tokens]: place among the drafted ones
        word = (bit.clamp(min=0) // 64).clamp(max=s["masks"].shape[1] - 1)
        words = s["masks"][rows].gather(2, word[:, None].expand(batch, most, -1))
        drafted = (words >> (bit.clamp(min=0) % 64)[:, None]) & 1 != 0
        seen = (bit < 0)[:, None] | (drafted & (bit < n[:, None])[:, None])
    seen = (seen & there[..., None])[:, None, None].expand(batch, 1, group, most, -1).reshape(batch, 1, group * most, -1)
    return scores.masked_fill_(~seen, -math.inf), seen, (rows[there], there), rows


def _plain_attention(s: dict) -> list:
    case, query = s["case"], s["query"]
    batch, hk, group = _split(case)
    scores, _, (place, there), _ = _scores(s)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    p = scores.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p, _dense(s, s["value"]).transpose(2, 3).contiguous())
    o = o / total.clamp(min=torch.finfo(torch.float32).tiny)
    o = o.view(batch, hk, group, -1, case["head_dim"]).permute(0, 3, 1, 2, 4).flatten(2, 3)
    out = torch.zeros(query.shape, dtype=query.dtype, device=query.device)
    out[place] = o[there].to(query.dtype)
    lse = torch.full(query.shape[:2], -math.inf, device=query.device)
    lse[place] = (top + torch.log(total)).view(batch, hk, group, -1).permute(0, 3, 1, 2).flatten(2)[there]
    return [out, lse]


def _plain_weights(s: dict) -> torch.Tensor:
    batch, hk, group = _split(s["case"])
    scores, seen, _, rows = _scores(s)
    lse = s["lse"][rows].view(batch, -1, hk, group).permute(0, 2, 3, 1).reshape(batch, hk, -1, 1)
    given = torch.where(seen & torch.isfinite(lse), (scores - lse).exp(), 0.0).sum(dim=2)
    s["weights"][..., :given.shape[-1]] += given
    return s["weights"]


def _evict_outputs(s: dict, kept: torch.Tensor) -> list:
    return [s["key"], s["value"], s["weights"], kept]


def _plain_evict(s: dict) -> list:
    case, weights = s["case"], s["weights"]
    page, longest, lens = case["page"], s["longest"], s["lens"].long()
    weights.copy_(s["gathered"])
    kept = torch.minimum(s["keep"].long(), lens)
    j = torch.arange(weights.shape[-1], device=weights.device)
    first = torch.clamp(kept, max=case["sinks"])
    last = lens - torch.clamp(kept - first, max=case["recent"])
    always = (j < first[:, None]) | ((j >= last[:, None]) & (j < lens[:, None]))
    rank = torch.where(always[:, None], math.inf, weights)
    rank = torch.where((j < lens[:, None])[:, None], rank, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True)[1]
    chosen = torch.zeros(weights.shape, dtype=torch.bool, device=weights.device)
    chosen.scatter_(-1, order, (j < kept[:, None])[:, None].expand(weights.shape))
    src = torch.where(chosen, j, weights.shape[-1]).sort(dim=-1)[0][..., :int(case["keep"])]  # [layers, batch, heads, keep]
    real = src < weights.shape[-1]
    src = src.clamp(max=weights.shape[-1] - 1)
    tables = s["tables"].long().clamp(min=0)
    dst = torch.arange(src.shape[-1], device=src.device).expand(src.shape)
    layer, row, head, _ = torch.where(real)
    src, dst = src[real], dst[real]
    block = [tables[row, at // page] for at in (src, dst)]
    for cache in (s["key"], s["value"]):
        cache[layer, block[1], head, :, dst % page] = cache[layer, block[0], head, :, src % page]
    moved = weights[layer, row, head, src]
    weights.masked_fill_((j < lens[:, None])[:, None], 0.0)
    weights[layer, row, head, dst] = moved
    return _evict_outputs(s, kept)


# ----- the framework's calls --------------------------------------------------------------------


def _framework():
    package = str(Path(__file__).resolve().parents[1] / "musa-aiter_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import musa_aiter

    return musa_aiter


def _own(s: dict):
    lib, case = _framework(), s["case"]
    path = case["path"]
    if path == "evict":
        s["weights"].copy_(s["gathered"])
        kept = lib.kv_evict_paged_tokens(s["key"], s["value"], s["weights"], s["tables"], s["lens"], s["keep"],
                                         sinks=case["sinks"], recent=case["recent"])
        return _evict_outputs(s, kept)
    if path == "tree":
        return list(lib.kv_paged_attention_tree(
            s["query"], s["key"], s["value"], s["tables"], s["lens"], s["masks"], query_starts=s["starts"],
            max_seq_len=s["longest"], return_lse=True))
    sight = {"query_starts": s["starts"], "max_seq_len": s["longest"], "window": case["window"] or None,
             "sinks": case["sinks"]}
    if path == "attention":
        return list(lib.kv_paged_attention(s["query"], s["key"], s["value"], s["tables"], s["lens"], return_lse=True,
                                           **sight))
    lib.kv_accumulate_attention_weights(s["weights"], s["query"], s["key"], s["tables"], s["lens"], s["lse"], **sight)
    return s["weights"]


def run(state: dict):
    if own:
        return _own(state)
    path = state["case"]["path"]
    if path == "evict":
        return _plain_evict(state)
    return _plain_weights(state) if path == "weights" else _plain_attention(state)


# ----- what a pass cannot do without ------------------------------------------------------------


def work(case: dict) -> dict:
    lens, rows = _lengths(np.random.default_rng(0), case)
    lens, rows = lens.astype(float), rows.astype(float)
    elt, hk, hd = DTYPES[case["dtype"]].itemsize, case["kv_heads"], case["head_dim"]
    if case["path"] == "evict":
        # The weights (gathered, then read and written), and the kept tokens but the first ones, read and written.
        kept = np.minimum(case["keep"], lens)
        moved = np.where(kept < lens, np.maximum(kept - case["sinks"], 0), 0).sum()
        return {"bytes": case["layers"] * hk * (4 * hd * elt * moved + 12 * lens.sum()), "flops": 0}
    window = case.get("window") or np.inf
    outside = np.minimum(case.get("sinks", 0), np.maximum(lens - window, 0))
    reach = np.minimum(lens, window + rows - 1 + outside)               # positions that a sequence's rows see together
    seen = np.minimum(lens - (rows - 1) / 2, window + outside)          # and each on average
    read = hk * hd * elt * reach.sum()
    values = rows.sum() * case["heads"] * hd
    products = 2 * case["heads"] * hd * (rows * seen).sum()
    if case["path"] == "weights":
        return {"bytes": read + 8 * hk * reach.sum() + values * elt + 4 * rows.sum() * case["heads"], "flops": products}
    return {"bytes": 2 * read + 2 * values * elt + 4 * rows.sum() * case["heads"], "flops": 2 * products}


# ----- the same in 64 bits ----------------------------------------------------------------------


def _exact_rows(s: dict):
    """For each sequence and kv head: their numbers, the rows, which positions each row sees, the scores of the
    group's heads in 64 bits, and the pages."""
    case, query = s["case"], s["query"]
    group, hd, device = case["heads"] // case["kv_heads"], case["head_dim"], query.device
    lens = s["lens"].tolist()
    starts = list(range(len(lens) + 1)) if s["starts"] is None else s["starts"].tolist()
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        ids = s["tables"][b, :-(-n // case["page"])].long()
        at = torch.arange(n - (hi - lo), n, device=device)[:, None]
        j = torch.arange(n, device=device)
        if s["masks"] is not None:
            bits = [[(w >> k) & 1 for w in row for k in range(64)] for row in s["masks"][lo:hi].tolist()]
            seen = torch.ones((hi - lo, n), dtype=torch.bool, device=device)
            seen[:, n - (hi - lo):] = torch.tensor(bits, device=device)[:, :hi - lo] != 0
        else:
            seen = j <= at
            if case["window"]:
                seen = seen & ((at - j < case["window"]) | (j < case["sinks"]))
        for h in range(case["kv_heads"]):
            k = s["key"][ids, h].double().permute(1, 0, 2).reshape(hd, -1)[:, :n]
            for g in range(h * group, (h + 1) * group):
                x = query[lo:hi, g].double() @ k / hd ** 0.5
                yield b, h, g, slice(lo, hi), x.masked_fill_(~seen, -math.inf), ids


def _exact_attention(s: dict) -> list:
    case, query = s["case"], s["query"]
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    lse = torch.full(query.shape[:2], -math.inf, dtype=torch.float64, device=query.device)
    for _, h, g, rows, x, ids in _exact_rows(s):
        v = s["value"][ids, h].double().permute(0, 2, 1).reshape(-1, case["head_dim"])[:x.shape[1]]
        out[rows, g] = torch.softmax(x, dim=-1) @ v
        lse[rows, g] = torch.logsumexp(x, dim=-1)
    return [out, lse]


def _exact_weights(s: dict) -> torch.Tensor:
    weights = s["weights"].double()
    for b, h, g, rows, x, _ in _exact_rows(s):
        weights[b, h, :x.shape[1]] += torch.exp(x - s["lse"][rows, g].double()[:, None]).sum(dim=0)
    return weights


def _exact_evict(s: dict) -> list:
    case, page = s["case"], s["case"]["page"]
    key, value = s["key"].clone(), s["value"].clone()
    gathered = s["gathered"].cpu().numpy()
    weights = gathered.astype(np.float64)
    kept = []
    for b, n in enumerate(s["lens"].tolist()):
        k = min(case["keep"], n)
        kept.append(k)
        first = min(case["sinks"], k)
        last = min(case["recent"], k - first)
        table = s["tables"][b].long()
        for layer in range(case["layers"]):
            for h in range(case["kv_heads"]):
                middle = gathered[layer, b, h, first:n - last]
                heavy = np.lexsort((np.arange(middle.size), -middle))[:k - first - last] + first
                stay = np.concatenate([np.arange(first), np.sort(heavy), np.arange(n - last, n)])
                src = torch.from_numpy(stay).to(key.device)
                dst = torch.arange(k, device=key.device)
                for new, old in ((key, s["key"]), (value, s["value"])):
                    new[layer, table[dst // page], h, :, dst % page] = old[layer, table[src // page], h, :, src % page]
                weights[layer, b, h, :n] = 0.0
                weights[layer, b, h, :k] = gathered[layer, b, h, stay]
    whole = [x.double() if x.numel() < 1 << 28 else None for x in (key, value)]
    return [*whole, torch.from_numpy(weights).to(key.device), torch.tensor(kept, device=key.device)]


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["path"] == "evict":
        return _exact_evict(state)
    return _exact_weights(state) if case["path"] == "weights" else _exact_attention(state)
