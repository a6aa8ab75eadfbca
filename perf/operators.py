"""Workloads of the operators on block-scaled FP8 caches: the store that writes such a cache, the attention that
reads it, and the bookkeeping of its pages.

A case is a dict of plain values.  ``listed()`` names the cases that are measured by default, ``draw()`` makes
further ones over the same ranges, ``prepare()`` builds a case's inputs on the GPU and ``run()`` makes one pass:
with ``own`` through the public entry points, else in plain torch operations, written from the definitions below.
``exact()`` gives the same outputs in 64 bits.

Caches are ``[blocks, kv_heads, head_dim, page]`` (several layers: one more leading extent) with one float32 scale
per block and head, for K and V apart.  A code stands for ``decode(code) * scale``; the codec has no subnormals,
no infinities and no NaN (exponent field 0 is a signed zero, the all-ones field is an ordinary one).

* ``attention``: query rows ``[rows, heads, head_dim]``; row i of the n of a sequence with ``len`` cached tokens
  sits at position ``len - n + i`` and sees the tokens up to there (the last ``window`` of them, if there is one).
* ``store``: new tokens are encoded into their slots.  A block's scale is the largest of max|new| / F, 2^-60 and its
  old scale; its older tokens are encoded anew if the scale grew.  A call that writes a block's first slot starts
  the block anew: the old scale and the old tokens are gone.
* ``draft``: one step of drafting several continuations per request.  Every row of a request takes over the accepted
  row's pages (fork), gets room for its draft tokens (extend: a shared partial last page is copied first) and gives
  back what was rejected (free).
* ``turnover``: requests that ended free their pages, the pages in use move together (compact), and new requests of
  the same lengths come in their place (extend).
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Per format: mantissa bits, exponent bias, largest finite value a scale aims at, the torch type of its codes.
FORMATS = {"e4m3": (3, 7, 448.0, torch.float8_e4m3fn), "e5m2": (2, 15, 57344.0, torch.float8_e5m2)}
SCALE_FLOOR = 2.0 ** -60


def listed() -> list[dict]:
    return [
        # One decode step of a few short chats (Llama-3-8B heads): launch latency counts.
        {"name": "decode_small", "path": "attention", "batch": 4, "q_lo": 1, "q_hi": 1, "pad": 0, "len_lo": 17,
         "len_hi": 500, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0, "dtype": "bf16",
         "format": "e4m3"},
        # A full decode batch of ragged lengths: the cache is read once, at memory speed.
        {"name": "decode_batch", "path": "attention", "batch": 64, "q_lo": 1, "q_hi": 1, "pad": 0, "len_lo": 256,
         "len_hi": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0, "dtype": "bf16",
         "format": "e4m3"},
        # Two very long contexts: few rows, so the work has to be split along the cache.
        {"name": "decode_long", "path": "attention", "batch": 2, "q_lo": 1, "q_hi": 1, "pad": 0, "len_lo": 100001,
         "len_hi": 131000, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "window": 0, "dtype": "fp16",
         "format": "e4m3"},
        # Drafts of one to eight tokens verified in a padded batch, odd lengths, a wider exponent.
        {"name": "verify_drafts", "path": "attention", "batch": 24, "q_lo": 1, "q_hi": 8, "pad": 13, "len_lo": 65,
         "len_hi": 3001, "heads": 16, "kv_heads": 2, "head_dim": 64, "page": 32, "window": 1000, "dtype": "bf16",
         "format": "e5m2"},
        # Prompt chunks against a cached prefix: matrix products, not bandwidth.
        {"name": "prefill_chunks", "path": "attention", "batch": 2, "q_lo": 1500, "q_hi": 2048, "pad": 0,
         "len_lo": 2048, "len_hi": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "window": 0,
         "dtype": "bf16", "format": "e4m3"},
        # The new token of each of 64 sequences, stored into one layer's cache.
        {"name": "store_decode", "path": "store", "decode": True, "layers": 1, "tokens": 64, "seq_lo": 1, "seq_hi": 1,
         "blocks": 1024, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "bf16", "format": "e4m3", "skip": 0.0},
        # Prompts stored into one layer, some of them going on inside a half-filled block.
        {"name": "store_prefill", "path": "store", "decode": False, "layers": 1, "tokens": 30977, "seq_lo": 128,
         "seq_hi": 4096, "blocks": 2560, "kv_heads": 8, "head_dim": 128, "page": 16, "dtype": "bf16",
         "format": "e4m3", "skip": 0.0},
        # A cached prefix brought back into all layers at once, 64-token pages, some tokens padded.
        {"name": "store_layers", "path": "store", "decode": False, "layers": 16, "tokens": 4001, "seq_lo": 64,
         "seq_hi": 2048, "blocks": 128, "kv_heads": 8, "head_dim": 128, "page": 64, "dtype": "fp16",
         "format": "e5m2", "skip": 0.01},
        # A draft step of a few requests over two layers: almost only bookkeeping.
        {"name": "draft_small", "path": "draft", "groups": 3, "width": 3, "len_lo": 5, "len_hi": 300, "draft": 5,
         "layers": 2, "kv_heads": 8, "head_dim": 128, "page": 16, "spare": 100},
        # A draft step of a full batch over all layers: the copied pages count.
        {"name": "draft_batch", "path": "draft", "groups": 32, "width": 4, "len_lo": 100, "len_hi": 700, "draft": 7,
         "layers": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "spare": 77},
        # One request in eight of a small pool is replaced.
        {"name": "turnover_small", "path": "turnover", "batch": 16, "every": 8, "len_lo": 30, "len_hi": 400,
         "layers": 4, "kv_heads": 8, "head_dim": 64, "page": 32, "spare": 9},
        # A quarter of a large batch is replaced: hundreds of megabytes of pages move.
        {"name": "turnover_batch", "path": "turnover", "batch": 64, "every": 4, "len_lo": 100, "len_hi": 1500,
         "layers": 16, "kv_heads": 8, "head_dim": 128, "page": 16, "spare": 500},
    ]


# What a drawn case may cost at most (the largest listed one of its path does).
MAX_CACHE_BYTES = 5.5e8     # codes an attention call reads
MAX_PREFILL = 2.0e11        # flops of an attention call
MAX_STORE = 7.0e7           # values of a store call
MAX_POOL = 9.0e8            # bytes of a page pool


def _log_int(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    path = rng.choice(["attention", "attention", "attention", "store", "store", "draft", "turnover"])
    head_dim, page = rng.choice([64, 96, 128, 128, 256]), rng.choice([16, 16, 32, 64])
    if path == "attention":
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
        kind = rng.choice(["decode", "decode", "verify", "prefill"])
        q_hi = {"decode": 1, "verify": rng.randrange(2, 17), "prefill": _log_int(rng, 64, 2048)}[kind]
        batch = rng.randrange(1, 4) if kind == "prefill" else _log_int(rng, 1, 96)
        most = MAX_CACHE_BYTES / (2 * batch * kv_heads * head_dim)
        if kind == "prefill":
            most = min(most, MAX_PREFILL / (4 * batch * q_hi * heads * head_dim))
        len_hi = max(q_hi, _log_int(rng, 16, max(32.0, min(131072.0, most))))
        return {"path": path, "batch": batch, "q_lo": 1 if kind != "prefill" else q_hi // 2, "q_hi": q_hi,
                "pad": 0 if kind == "decode" else rng.choice([0, 7]), "len_lo": max(1, len_hi // rng.choice([1, 3, 30])),
                "len_hi": len_hi, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "window": rng.choice([0, 0, 0, _log_int(rng, 8, 4096)]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
                "format": rng.choice(["e4m3", "e4m3", "e5m2"])}
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    if path == "store":
        decode, layers = rng.random() < 0.4, rng.choice([1, 1, 4, 16])
        if decode:
            tokens, lo, hi = _log_int(rng, 1, 512), 1, 1
            blocks = tokens + rng.randrange(16, 512)
        else:
            tokens = _log_int(rng, 20, MAX_STORE / (2 * layers * kv_heads * head_dim))
            tokens = min(tokens, 60000)
            hi = max(16, min(4096, tokens // 2))
            lo = max(8, hi // 16)
            blocks = tokens // page + 2 * (tokens // lo + 2) + rng.randrange(1, 64)
        return {"path": path, "decode": decode, "layers": layers, "tokens": tokens, "seq_lo": lo, "seq_hi": hi,
                "blocks": blocks, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "format": rng.choice(["e4m3", "e4m3", "e5m2"]),
                "skip": rng.choice([0.0, 0.02])}
    layers, len_hi = rng.choice([1, 2, 16, 32]), _log_int(rng, 20, 2000)
    page_bytes = 2 * layers * kv_heads * head_dim * page
    if path == "draft":
        width, deep = rng.randrange(1, 9), rng.randrange(1, 20)
        pages = len_hi / page + width * (2 + deep / page)
        return {"path": path, "groups": max(1, min(_log_int(rng, 1, 64), int(MAX_POOL / (page_bytes * pages)))),
                "width": width, "len_lo": max(1, len_hi // 8), "len_hi": len_hi, "draft": deep, "layers": layers,
                "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "spare": rng.randrange(0, 64)}
    batch = max(2, min(_log_int(rng, 2, 128), int(MAX_POOL / (page_bytes * (1 + len_hi / page)))))
    return {"path": path, "batch": batch, "every": rng.randrange(2, 9), "len_lo": max(1, len_hi // 8), "len_hi": len_hi,
            "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "spare": rng.randrange(0, 64)}


# ----- inputs -----------------------------------------------------------------------------------


def _device() -> torch.device:
    return torch.device("cuda", torch.cuda.current_device())


def _on(device, values, dtype=torch.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(np.asarray(values, dtype=np.int64))).to(device=device, dtype=dtype)


def _cache(gen, shape, fmt: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes ``shape`` and float32 scales ``shape[:-2]`` of normal values whose size varies by block, head and channel."""
    mant, bias, most, code_type = FORMATS[fmt]
    lead, (hd, page) = tuple(shape[:-2]), shape[-2:]
    codes = torch.empty(lead + (hd, page), dtype=torch.uint8, device=gen.device)
    scales = torch.empty(lead, dtype=torch.float32, device=gen.device)
    flat, flat_scales = codes.view(-1, hd, page), scales.view(-1)
    step = max(1, (1 << 26) // (hd * page))
    channel = torch.exp(0.3 * torch.randn((hd, 1), generator=gen, device=gen.device))
    for i in range(0, flat.shape[0], step):
        part = flat[i:i + step]
        x = torch.randn(part.shape, generator=gen, device=gen.device).mul_(channel)
        x.mul_(torch.exp(0.25 * torch.randn((part.shape[0], 1, 1), generator=gen, device=gen.device)))
        s = x.abs().amax(dim=(1, 2)).div_(most)
        x.div_(s[:, None, None])
        x.masked_fill_(x.abs() < 2.0 ** (1 - bias), 0.0)
        part.copy_(x.to(code_type).view(torch.uint8))
        flat_scales[i:i + step] = s
    return codes, scales


def _lengths(rng, case) -> tuple[np.ndarray, np.ndarray]:
    """Cached tokens and query rows of each sequence, uniform in their ranges (one of them the longest).  The seed
    deals them out to the sequences: what they add up to, and so every output's shape, belongs to the case."""
    own_rng, count = np.random.default_rng(20), case.get("batch") or case["groups"]
    lens = own_rng.integers(case["len_lo"], case["len_hi"] + 1, size=count)
    lens[0] = case["len_hi"]
    rows = own_rng.integers(case.get("q_lo", 1), case.get("q_hi", 1) + 1, size=count)
    rows[0] = case.get("q_hi", 1)
    deal = rng.permutation(count)
    return lens[deal], np.minimum(rows, lens)[deal]


def _attention_inputs(case, gen, rng) -> dict:
    lens, queries = _lengths(rng, case)
    page = case["page"]
    pages = -(-lens // page)
    blocks = int(pages.sum()) + 7
    order, used = rng.permutation(blocks), 0
    tables = np.full((case["batch"], int(pages.max())), -1, dtype=np.int64)
    for b, k in enumerate(pages):
        tables[b, :k] = order[used:used + k]
        used += int(k)
    shape = (blocks, case["kv_heads"], case["head_dim"], page)
    key, k_scales = _cache(gen, shape, case["format"])
    value, v_scales = _cache(gen, shape, case["format"])
    rows = int(queries.sum()) + case["pad"]
    query = torch.randn((rows, case["heads"], case["head_dim"]), generator=gen, device=gen.device).mul_(1.5)
    starts = np.concatenate([[0], np.cumsum(queries)])
    return {"query": query.to(DTYPES[case["dtype"]]), "key": key, "value": value, "k_scales": k_scales,
            "v_scales": v_scales, "tables": _on(gen.device, tables), "lens": _on(gen.device, lens),
            # One row per sequence needs no row table; a padded or ragged batch comes with one.
            "starts": None if case["q_hi"] == 1 and not case["pad"] else _on(gen.device, starts),
            "longest": int(lens.max()), "most_rows": int(queries.max())}


def _store_inputs(case, gen, rng) -> dict:
    page, tokens, layers = case["page"], case["tokens"], case["layers"]
    order = rng.permutation(case["blocks"])
    if case["decode"]:
        slots = order[:tokens] * page + rng.integers(0, page, size=tokens)
    else:
        ends = np.cumsum(rng.integers(case["seq_lo"], case["seq_hi"] + 1, size=tokens // case["seq_lo"] + 1))
        counts = np.diff(np.append(ends[ends < tokens], tokens), prepend=0)
        parts, used = [], 0
        for n in counts:
            # Half of the sequences go on inside a block that holds older tokens.
            j = np.arange(n) + (rng.integers(0, page) if rng.random() < 0.5 else 0)
            parts.append(order[used + j // page] * page + j % page)
            used += int(j[-1]) // page + 1
        slots = np.concatenate(parts)
    slots[rng.random(tokens) < case["skip"]] = -1
    lead = (layers,) if layers > 1 else ()
    shape = lead + (case["blocks"], case["kv_heads"], case["head_dim"], page)
    key, k_scales = _cache(gen, shape, case["format"])
    value, v_scales = _cache(gen, shape, case["format"])
    new = [torch.randn(lead + (tokens, case["kv_heads"], case["head_dim"]), generator=gen, device=gen.device)
           .to(DTYPES[case["dtype"]]) for _ in range(2)]
    return {"new": new, "slots": _on(gen.device, slots, torch.int64), "key": key, "value": value,
            "k_scales": k_scales, "v_scales": v_scales}


def _pool(case, gen, blocks: int) -> dict:
    shape = (case["layers"], blocks, case["kv_heads"], case["head_dim"], case["page"])
    # Codes of ordinary values: neither a subnormal nor an all-ones exponent.
    key, value = (torch.randint(8, 120, shape, generator=gen, device=gen.device, dtype=torch.uint8) for _ in range(2))
    k_scales, v_scales = (torch.rand(shape[:3], generator=gen, device=gen.device) + 0.5 for _ in range(2))
    return {"key": key, "value": value, "k_scales": k_scales, "v_scales": v_scales}


def _draft_inputs(case, gen, rng) -> dict:
    groups, width, page, deep = case["groups"], case["width"], case["page"], case["draft"]
    lens, _ = _lengths(rng, case)
    pages = -(-lens // page)
    blocks = int(pages.sum()) + groups * width * (2 + (deep + page - 1) // page) + case["spare"]
    order, used = rng.permutation(blocks), 0
    tables = np.full((groups * width, int((-(-(lens + deep) // page)).max())), -1, dtype=np.int64)
    refs = np.zeros(blocks, dtype=np.int64)
    for g, k in enumerate(pages):  # the rows of a request share its pages
        ids = order[used:used + k]
        tables[g * width:(g + 1) * width, :k] = ids
        refs[ids] = width
        used += int(k)
    accepted = np.arange(groups) * width + rng.integers(0, width, size=groups)
    return {**_pool(case, gen, blocks), "tables": _on(gen.device, tables), "refs": _on(gen.device, refs),
            "lens": _on(gen.device, np.repeat(lens, width)), "parents": _on(gen.device, np.repeat(accepted, width)),
            "drafts": _on(gen.device, rng.integers(1, deep + 1, size=groups * width)),
            "keep": _on(gen.device, np.repeat(lens, width))}


def _turnover_inputs(case, gen, rng) -> dict:
    page, batch, every = case["page"], case["batch"], case["every"]
    lens, _ = _lengths(rng, case)
    pages = -(-lens // page)
    blocks = int(pages.sum()) + case["spare"]
    order, used = rng.permutation(int(pages.sum())), 0
    tables = np.full((batch, int(pages.max())), -1, dtype=np.int64)
    refs = np.zeros(blocks, dtype=np.int64)
    for b, k in enumerate(pages):
        tables[b, :k] = order[used:used + k]
        used += int(k)
    refs[:used] = 1
    rows = np.arange(batch)
    return {**_pool(case, gen, blocks), "tables": _on(gen.device, tables), "refs": _on(gen.device, refs),
            "lens": _on(gen.device, lens), "turn": 0, "longest": int(lens.max()),
            # Which rows end at each turn (0 tokens kept; -1: the row stays), and the tokens of those that follow.
            "keep": [_on(gen.device, np.where(rows % every == t, 0, -1)) for t in range(every)],
            "come": [_on(gen.device, np.where(rows % every == t, lens, 0)) for t in range(every)]}


_INPUTS = {"attention": _attention_inputs, "store": _store_inputs, "draft": _draft_inputs, "turnover": _turnover_inputs}


def prepare(case: dict, seed: int) -> dict:
    device = _device()
    gen = torch.Generator(device=device).manual_seed(seed)
    return {"case": case, **_INPUTS[case["path"]](case, gen, np.random.default_rng(seed))}


# ----- the plain forms --------------------------------------------------------------------------


def _decoded(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    """float32 values of codes that hold no subnormal and no all-ones exponent (as the caches here)."""
    return codes.view(FORMATS[fmt][3]).float()


def _encoded(w: torch.Tensor, fmt: str) -> torch.Tensor:
    """Codes of float32 quotients whose size is at most the format's largest (to within one rounding)."""
    _, bias, _, code_type = FORMATS[fmt]
    w = torch.where(torch.isfinite(w) & (w.abs() >= 2.0 ** (1 - bias)), w, 0.0)
    return w.to(code_type).view(torch.uint8)


def _plain_attention(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"]
    page, hq, hk, hd = case["page"], case["heads"], case["kv_heads"], case["head_dim"]
    batch, group, device = case["batch"], hq // hk, query.device
    lens = s["lens"].long()
    tables = s["tables"][:, :-(-s["longest"] // page)].long().clamp(min=0)
    most = s["most_rows"]
    starts = torch.arange(batch + 1, device=device) if s["starts"] is None else s["starts"].long()
    i = torch.arange(most, device=device)
    n = starts[1:] - starts[:-1]
    there = i < n[:, None]
    rows = torch.where(there, starts[:-1, None] + i, 0)

    def dense(cache, scales):  # [batch, kv_heads, head_dim, tokens]
        x = _decoded(cache[tables], case["format"]) * scales[tables][..., None, None]
        return x.permute(0, 2, 3, 1, 4).reshape(batch, hk, hd, -1)

    q = query[rows].float().view(batch, most, hk, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, hd)
    scores = torch.matmul(q, dense(s["key"], s["k_scales"])).mul_(1.0 / math.sqrt(hd))
    at = (lens - n)[:, None] + i                                             # position of each row
    j = torch.arange(scores.shape[-1], device=device)
    seen = there[..., None] & (j <= at[..., None])
    if case["window"]:
        seen = seen & (j > at[..., None] - case["window"])
    seen = seen[:, None, None].expand(batch, 1, group, most, -1).reshape(batch, 1, group * most, -1)
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(top), top, 0.0))
    o = torch.matmul(p, dense(s["value"], s["v_scales"]).transpose(2, 3).contiguous())
    o = o / p.sum(dim=-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    o = o.view(batch, hk, group, most, hd).permute(0, 3, 1, 2, 4).reshape(batch, most, hq, hd)
    out = torch.zeros(query.shape, dtype=query.dtype, device=device)
    out[rows[there]] = o[there].to(query.dtype)
    return out


def _plain_store(s: dict) -> list:
    case = s["case"]
    fmt, page, blocks, most = case["format"], case["page"], case["blocks"], FORMATS[case["format"]][2]
    slots = s["slots"]
    order = torch.arange(slots.numel(), device=slots.device)
    last = torch.full((blocks * page + 1,), -1, dtype=torch.int64, device=slots.device)
    last.scatter_reduce_(0, torch.where(slots >= 0, slots, blocks * page), order, "amax")
    last = last[:-1].view(blocks, page)
    ids = (last >= 0).any(dim=1).nonzero()[:, 0]
    last = last[ids]
    wrote = (last >= 0)[None, :, None, None, :]                              # layers, blocks, heads, dims, page

    def one(new, cache, scales):
        if cache.dim() == 4:
            new, cache, scales = new[None], cache[None], scales[None]
        x = new[:, last.clamp(min=0)].permute(0, 1, 3, 4, 2).float()         # [layers, blocks, heads, dims, page]
        size = torch.where(wrote & torch.isfinite(x), x.abs(), 0.0).amax(dim=(3, 4))
        before = scales[:, ids]
        anew = (last[:, 0] >= 0)[None, :, None] | ~((before > 0) & torch.isfinite(before))
        now = torch.maximum(torch.where(anew, 0.0, before), size / most).clamp(min=SCALE_FLOOR)
        old = cache[:, ids]
        back = _encoded(_decoded(old, fmt) * before[..., None, None] / now[..., None, None], fmt)
        same = torch.where((now == before)[..., None, None], old, back)
        same = torch.where(anew[..., None, None], 0, same)
        cache[:, ids] = torch.where(wrote, _encoded(x / now[..., None, None], fmt), same)
        scales[:, ids] = now

    one(s["new"][0], s["key"], s["k_scales"])
    one(s["new"][1], s["value"], s["v_scales"])
    return _store_outputs(s)


def _store_outputs(s: dict) -> list:
    code_type = FORMATS[s["case"]["format"]][3]
    return [s["key"].view(code_type), s["value"].view(code_type), s["k_scales"], s["v_scales"]]


def _owners(refs, tables, used, by: int) -> None:
    """Adds ``by`` to the reference count of every table entry marked ``used``."""
    refs.scatter_add_(0, tables.clamp(min=0).long().view(-1), (used & (tables >= 0)).to(refs.dtype).mul_(by).view(-1))


def _plain_fork(s: dict) -> None:
    page, tables, lens, parents = s["case"]["page"], s["tables"], s["lens"], s["parents"].long()
    at = torch.arange(tables.shape[1], device=tables.device)
    has = (parents >= 0) & (parents < tables.shape[0])
    parents = torch.where(has, parents, 0)
    new_tables = torch.where(has[:, None], tables[parents], -1)
    new_lens = torch.where(has, lens[parents], 0)
    _owners(s["refs"], new_tables, at < (new_lens[:, None] + page - 1) // page, 1)
    _owners(s["refs"], tables, at < (lens[:, None] + page - 1) // page, -1)
    tables.copy_(new_tables)
    lens.copy_(new_lens)


def _plain_free(s: dict, keep: torch.Tensor) -> None:
    page, tables, lens = s["case"]["page"], s["tables"], s["lens"]
    at = torch.arange(tables.shape[1], device=tables.device)
    keep = torch.where(keep < 0, lens, torch.minimum(keep, lens))
    gone = (at >= (keep[:, None] + page - 1) // page) & (at < (lens[:, None] + page - 1) // page)
    _owners(s["refs"], tables, gone, -1)
    tables.masked_fill_(gone, -1)
    lens.copy_(keep)


def _move_pages(s: dict, src, dst) -> None:
    for x in (s["key"], s["value"], s["k_scales"], s["v_scales"]):
        x[:, dst] = x[:, src]


def _plain_extend(s: dict, new: torch.Tensor, most: int) -> list:
    page, tables, refs, lens = s["case"]["page"], s["tables"], s["refs"], s["lens"].long()
    batch, width = tables.shape
    new = new.long().clamp(0, most)
    at = torch.arange(width, device=tables.device)
    had, has = (lens + page - 1) // page, (lens + new + page - 1) // page
    last = tables.long().gather(1, (had - 1).clamp(min=0)[:, None])[:, 0]
    open_ = (new > 0) & (lens % page != 0) & (last >= 0)
    # A shared page is copied by all of its owners but the last that is asked.
    row = torch.arange(batch, device=tables.device)
    earlier = ((last[:, None] == last) & open_[:, None] & open_ & (row < row[:, None])).sum(dim=1)
    copy = open_ & (earlier < refs.long()[last.clamp(min=0)] - 1)
    need = has - had + copy
    first = need.cumsum(0) - need
    free = refs == 0
    fits = (need.sum() <= free.sum()) & (has <= width).all()
    ids = torch.arange(refs.numel(), device=tables.device)
    free_ids = torch.where(free, ids, refs.numel()).sort()[0]
    take = free_ids[(first[:, None] + copy[:, None] + at - had[:, None]).clamp(0, refs.numel() - 1)]
    fresh = fits & (at >= had[:, None]) & (at < has[:, None])
    copied = fits & copy[:, None] & (at == had[:, None] - 1)
    take = torch.where(copied, free_ids[first.clamp(max=refs.numel() - 1)][:, None], take)
    pick = (copy & fits).nonzero()[:, 0]
    src, dst = last[pick], free_ids[first[pick]]
    _move_pages(s, src, dst)
    refs.scatter_add_(0, src, torch.full_like(src, -1).to(refs.dtype))
    tables.copy_(torch.where(fresh | copied, take.to(tables.dtype), tables))
    _owners(refs, tables, fresh | copied, 1)
    s["lens"].copy_(torch.where(fits, lens + new, lens))
    i = torch.arange(most, device=tables.device)
    pos = lens[:, None] + i
    slots = tables.long().gather(1, (pos // page).clamp(max=width - 1)) * page + pos % page
    slots = torch.where(fits & (i < new[:, None]), slots, -1)
    return [slots, free.sum() - need.sum()]


def _plain_compact(s: dict) -> torch.Tensor:
    refs, tables = s["refs"], s["tables"]
    live = refs > 0
    count = live.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    src, dst = (live & (ids >= count)).nonzero()[:, 0], (~live & (ids < count)).nonzero()[:, 0]
    _move_pages(s, src, dst)
    to = ids.to(tables.dtype)
    to[src] = dst.to(tables.dtype)
    refs[dst] = refs[src]
    refs[src] = 0
    tables.copy_(torch.where(tables >= 0, to[tables.clamp(min=0).long()], tables))
    return count


def _page_outputs(s: dict, *more) -> list:
    code_type = FORMATS["e4m3"][3]
    return [*more, s["tables"], s["lens"], s["refs"], s["key"].view(code_type), s["value"].view(code_type),
            s["k_scales"], s["v_scales"]]


def _plain(s: dict):
    path = s["case"]["path"]
    if path == "attention":
        return _plain_attention(s)
    if path == "store":
        return _plain_store(s)
    if path == "draft":
        _plain_fork(s)
        slots, left = _plain_extend(s, s["drafts"], s["case"]["draft"])
        _plain_free(s, s["keep"])
        return _page_outputs(s, slots, left)
    turn = s["turn"]
    s["turn"] = (turn + 1) % s["case"]["every"]
    _plain_free(s, s["keep"][turn])
    count = _plain_compact(s)
    slots, left = _plain_extend(s, s["come"][turn], s["longest"])
    return _page_outputs(s, slots, left, count)


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
    if path == "attention":
        return lib.kv_paged_attention_fp8(
            s["query"], s["key"], s["value"], s["tables"], s["lens"], s["k_scales"], s["v_scales"],
            query_starts=s["starts"], max_seq_len=s["longest"], window=case["window"] or None,
            fp8_format=case["format"])
    if path == "store":
        lib.kv_linear_to_paged_fp8_block(*s["new"], s["key"], s["value"], s["slots"], s["k_scales"], s["v_scales"],
                                         fp8_format=case["format"])
        return _store_outputs(s)
    caches = (s["key"], s["value"])
    scales = {"k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    state = (s["tables"], s["lens"], s["refs"])
    if path == "draft":
        lib.kv_fork_paged_sequences(*state, s["parents"], block_size=case["page"])
        slots, left = lib.kv_extend_paged_sequences(*caches, *state, s["drafts"], case["draft"], **scales)
        lib.kv_free_paged_sequences(*state, s["keep"], block_size=case["page"])
        return _page_outputs(s, slots, left)
    turn = s["turn"]
    s["turn"] = (turn + 1) % case["every"]
    lib.kv_free_paged_sequences(*state, s["keep"][turn], block_size=case["page"])
    count = lib.kv_compact_paged_blocks(*caches, s["tables"], s["refs"], **scales)
    slots, left = lib.kv_extend_paged_sequences(*caches, *state, s["come"][turn], s["longest"], **scales)
    return _page_outputs(s, slots, left, count)


def run(state: dict):
    if own:
        return _own(state)
    return _plain(state)


# ----- what a pass cannot do without ------------------------------------------------------------


def work(case: dict) -> dict:
    page, path = case["page"], case["path"]
    row = case["kv_heads"] * case["head_dim"]
    if path == "attention":
        # Lengths and rows are uniform in their ranges, the first the longest.
        batch, elt = case["batch"], DTYPES[case["dtype"]].itemsize
        mean = (case["len_hi"] + (batch - 1) * (case["len_lo"] + case["len_hi"]) / 2) / batch
        rows = min(mean, (case["q_hi"] + (batch - 1) * (case["q_lo"] + case["q_hi"]) / 2) / batch)
        reach = min(mean, case["window"] + rows) if case["window"] else mean
        seen = min(mean - (rows - 1) / 2, case["window"] or mean)
        codes = batch * reach * (2 * row + 8 * case["kv_heads"] / page + 4 / page)
        values = 2 * (batch * rows) * case["heads"] * case["head_dim"]
        return {"bytes": codes + values * elt, "flops": 2 * values * seen}
    if path == "store":
        # The tokens, their codes, the scales of their blocks (read and written).
        n, elt = case["layers"] * case["tokens"], DTYPES[case["dtype"]].itemsize
        blocks = n if case["decode"] else n / page
        return {"bytes": 2 * n * row * (elt + 1) + 16 * blocks * case["kv_heads"] + 8 * case["tokens"], "flops": 0}
    # Pages that move are read and written in every layer; every row's page list is read.
    page_bytes = 2 * case["layers"] * (row * page + 4 * case["kv_heads"])
    mean = (case["len_lo"] + case["len_hi"]) / 2
    if path == "draft":
        rows = case["groups"] * case["width"]
        moved, entries = case["groups"] * (case["width"] - 1) * (1 - 1 / page), rows * mean / page
        return {"bytes": 2 * moved * page_bytes + 4 * entries + 8 * rows * case["draft"], "flops": 0}
    moved = case["batch"] / case["every"] * mean / page
    return {"bytes": 2 * moved * page_bytes + 4 * case["batch"] * mean / page + 8 * case["batch"] * case["len_hi"],
            "flops": 0}


# ----- the same in 64 bits ----------------------------------------------------------------------


def _table64(fmt: str, device) -> torch.Tensor:
    """The value of every code: (1 + m / 2^M) * 2^(E - bias), a zero where E is 0."""
    mant, bias, _, _ = FORMATS[fmt]
    values = []
    for code in range(256):
        e, m = (code & 127) >> mant, code & ((1 << mant) - 1)
        v = (1 + m / (1 << mant)) * 2.0 ** (e - bias) if e else 0.0
        values.append(-v if code & 128 else v)
    return torch.tensor(values, dtype=torch.float64, device=device)


def _round64(w: torch.Tensor, fmt: str) -> torch.Tensor:
    """The value the encoder keeps of each quotient."""
    mant, bias, most, _ = FORMATS[fmt]
    unit = torch.exp2(torch.frexp(w)[1].double() - 1 - mant)
    r = (torch.round(w / unit) * unit).clamp(-most, most)
    return torch.where(w.abs() < 2.0 ** (1 - bias), 0.0, r)


def _exact_attention(s: dict) -> torch.Tensor:
    case, query = s["case"], s["query"]
    page, hk, hd = case["page"], case["kv_heads"], case["head_dim"]
    group = case["heads"] // hk
    table = _table64(case["format"], query.device)
    lens = s["lens"].tolist()
    starts = list(range(len(lens) + 1)) if s["starts"] is None else s["starts"].tolist()
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    for b, n in enumerate(lens):
        rows = starts[b + 1] - starts[b]
        ids = s["tables"][b, :-(-n // page)].long()
        at = n - rows + torch.arange(rows, device=query.device)
        j = torch.arange(n, device=query.device)
        seen = j[None] <= at[:, None]
        if case["window"]:
            seen &= j[None] > at[:, None] - case["window"]
        for h in range(hk):
            k, v = ((table[c[ids, h].long()] * z[ids, h].double()[:, None, None]).permute(1, 0, 2).reshape(hd, -1)[:, :n]
                    for c, z in ((s["key"], s["k_scales"]), (s["value"], s["v_scales"])))
            for g in range(h * group, (h + 1) * group):
                x = query[starts[b]:starts[b + 1], g].double() @ k / hd ** 0.5
                x = torch.softmax(x.masked_fill(~seen, -math.inf), dim=-1)
                out[starts[b]:starts[b + 1], g] = x @ v.t().contiguous()
    return out


def _exact_store(s: dict) -> list:
    case = s["case"]
    fmt, page, device = case["format"], case["page"], s["slots"].device
    most, table = FORMATS[fmt][2], _table64(fmt, device)
    columns: dict[int, dict[int, int]] = {}
    for t, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            columns.setdefault(slot // page, {})[slot % page] = t
    groups: dict[tuple, list] = {}  # blocks that write the same columns go together
    for block, by in columns.items():
        groups.setdefault(tuple(sorted(by)), []).append((block, [by[c] for c in sorted(by)]))
    outs, sizes = [], []
    for new, cache, scales in zip(s["new"], (s["key"], s["value"]), (s["k_scales"], s["v_scales"])):
        lead = cache.dim() == 5
        new, codes, scale = (x if lead else x[None] for x in (new, cache, scales.double()))
        values, scale = table[codes.long()], scale.clone()
        for cols, members in groups.items():
            ids = torch.tensor([m[0] for m in members], device=device)
            x = new[:, torch.tensor([m[1] for m in members], device=device)].double().permute(0, 1, 3, 4, 2)
            before = scale[:, ids]
            floor = torch.zeros_like(before) if cols[0] == 0 else before
            now = torch.maximum(floor, x.abs().amax(dim=(3, 4)) / most).clamp(min=SCALE_FLOOR)
            old = values[:, ids]
            grown = _round64(old * (before / now)[..., None, None], fmt)
            old = torch.where((now == before)[..., None, None], old, grown) * (cols[0] != 0)
            old[..., list(cols)] = _round64(x / now[..., None, None], fmt)
            values[:, ids], scale[:, ids] = old, now
        outs.append(values if lead else values[0])
        sizes.append(scale if lead else scale[0])
    return outs + sizes


class _Pages:
    """The page bookkeeping, one step at a time on the host."""

    def __init__(self, s: dict):
        self.s, self.page = s, s["case"]["page"]
        self.tables, self.lens, self.refs = s["tables"].tolist(), s["lens"].tolist(), s["refs"].tolist()

    def count(self, n: int) -> int:
        return -(-n // self.page)

    def copy(self, src: int, dst: int) -> None:
        for x in (self.s["key"], self.s["value"], self.s["k_scales"], self.s["v_scales"]):
            x[:, dst] = x[:, src].clone()

    def fork(self, parents) -> None:
        rows = [(list(self.tables[p]), self.lens[p]) for p in parents]
        for row, n in rows:
            for p in row[:self.count(n)]:
                self.refs[p] += 1
        for b, (row, n) in enumerate(rows):
            for p in self.tables[b][:self.count(self.lens[b])]:
                self.refs[p] -= 1
            self.tables[b], self.lens[b] = row, n

    def free(self, keep) -> None:
        for b, k in enumerate(keep):
            k = self.lens[b] if k < 0 else min(k, self.lens[b])
            for i in range(self.count(k), self.count(self.lens[b])):
                self.refs[self.tables[b][i]] -= 1
                self.tables[b][i] = -1
            self.lens[b] = k

    def extend(self, new, most: int):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        taken, slots = iter(free), []
        for b, n in enumerate(new):
            first, row = self.lens[b], self.tables[b]
            if n and first % self.page:
                last = row[self.count(first) - 1]
                if self.refs[last] > 1:
                    to = next(taken)
                    self.copy(last, to)
                    self.refs[last] -= 1
                    self.refs[to] = 1
                    row[self.count(first) - 1] = to
            for i in range(self.count(first), self.count(first + n)):
                row[i] = next(taken)
                self.refs[row[i]] = 1
            self.lens[b] = first + n
            slots.append([row[i // self.page] * self.page + i % self.page if i < first + n else -1
                          for i in range(first, first + most)])
        return slots, sum(1 for _ in taken)

    def compact(self) -> int:
        live = [p for p, r in enumerate(self.refs) if r > 0]
        to = {p: p for p in live}
        holes = [p for p in range(len(live)) if self.refs[p] == 0]
        for src, dst in zip([p for p in live if p >= len(live)], holes):
            self.copy(src, dst)
            self.refs[dst], self.refs[src] = self.refs[src], 0
            to[src] = dst
        self.tables = [[to.get(p, p) for p in row] for row in self.tables]
        return len(live)

    def outputs(self, *more) -> list:
        s, device = self.s, self.s["refs"].device
        table = _table64("e4m3", device)
        whole = [torch.tensor(x, device=device) for x in (*more, self.tables, self.lens, self.refs)]
        return whole + [torch.cat([table[layer.long()][None] for layer in s[x]]) if s[x].numel() < 1 << 28 else None
                        for x in ("key", "value")] + [s["k_scales"].double(), s["v_scales"].double()]


def _exact_pages(s: dict) -> list:
    pages, case = _Pages(s), s["case"]
    if case["path"] == "draft":
        pages.fork(s["parents"].tolist())
        slots, left = pages.extend(s["drafts"].tolist(), case["draft"])
        pages.free(s["keep"].tolist())
        return pages.outputs(slots, left)
    pages.free(s["keep"][0].tolist())
    count = pages.compact()
    slots, left = pages.extend(s["come"][0].tolist(), s["longest"])
    return pages.outputs(slots, left, count)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["path"] == "attention":
        return _exact_attention(state)
    if case["path"] == "store":
        return _exact_store(state)
    return _exact_pages(state)
