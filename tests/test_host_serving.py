"""CPU: argument checks of the operators on block-scaled caches and pages, and the packed calls' layouts."""

from __future__ import annotations

import ctypes
import pathlib
import re

import pytest
import torch

import musa_aiter
from musa_aiter import registry
from musa_aiter.ops import _hip

HEADER = pathlib.Path(__file__).resolve().parents[1] / "include" / "musa_aiter_kv_serving.h"
NAMES = ("kv_linear_to_paged_fp8_block", "kv_paged_attention_fp8", "kv_extend_paged_sequences",
         "kv_fork_paged_sequences", "kv_free_paged_sequences", "kv_compact_paged_blocks")


def test_registered_and_exported():
    caps = registry.list_capabilities("kvblock") + registry.list_capabilities("kvpages")
    assert {c.name for c in caps} == set(NAMES)
    for cap in caps:
        assert cap.backends == ("rocm-hip",) and callable(getattr(musa_aiter, cap.name))


@pytest.mark.parametrize("name,packed", [("block_store", "_BLOCK_STORE_CALL"), ("attention", "_ATTENTION_CALL"),
                                         ("pages", "_PAGES_CALL")])
def test_packed_calls_match_the_header(name, packed):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct musa_aiter_hip_%s_call \{(.*?)\}" % name, text, re.S).group(1)
    codes = ""
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind = "Q" if "*" in decl else {"int64_t": "q", "int32_t": "i", "double": "d"}[decl.split()[0]]
        for field in decl.split(None, 1)[1].split(","):
            size = re.search(r"\[(\d+)\]", field)
            codes += kind * (int(size.group(1)) if size else 1)
    got = getattr(_hip, packed).format.lstrip("<")
    assert re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), got) == codes


def test_workspace_fields_are_where_they_are_written():
    call = bytearray(_hip._ATTENTION_CALL.pack(*range(1, 39)))
    assert _hip._ATTENTION_WORKSPACE.unpack_from(call, _hip._ATTENTION_WORKSPACE_AT) == (11, 12)
    fields = _hip._ATTENTION_CALL.unpack(call)
    at = _hip._ATTENTION_SPLITS_AT // 8
    assert fields[at] == at + 1 and _hip._ATTENTION_CALL.format == "<11Qq8q2q2q4q3qd6i" and at == 30  # splits
    pages = bytearray(_hip._PAGES_CALL.pack(*range(1, 28)))
    assert _hip._PAGES_CALL.unpack(pages)[6:8] == (7, 8) and _hip._PAGES_WORKSPACE_AT == 48


def test_entries_exported_and_refuse_nothing_to_do():
    lib = ctypes.CDLL(str(_hip.LIB_PATH))
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for symbol in re.findall(r"(?:int64_t|int)\s+(musa_aiter_hip_\w+)\s*\(", text):
        assert hasattr(lib, symbol)
        f = _hip.fn(symbol)
        if symbol.split("_")[-1] in ("splits", "workspace"):
            continue
        assert f(None, None) != 0
        # All sizes zero or pointers missing: an error, before any launch.
        size = {"store": _hip._BLOCK_STORE_CALL, "attention": _hip._ATTENTION_CALL}.get(symbol.split("_")[-1], _hip._PAGES_CALL).size
        assert f(bytes(size), None) != 0


def _store(**change):
    a = dict(key_linear=torch.zeros(3, 2, 8), value_linear=torch.zeros(3, 2, 8),
             key_cache_fp8=torch.zeros(4, 2, 8, 16, dtype=torch.uint8), value_cache_fp8=torch.zeros(4, 2, 8, 16, dtype=torch.uint8),
             slot_mapping=torch.zeros(3, dtype=torch.int64), k_scales=torch.zeros(4, 2), v_scales=torch.zeros(4, 2))
    a.update(change)
    return musa_aiter.kv_linear_to_paged_fp8_block(**a)


@pytest.mark.parametrize("change,match", [
    (dict(fp8_format="int8"), "unsupported"),
    (dict(key_cache_fp8=torch.zeros(4, 2, 8, 16)), "uint8"),
    (dict(value_cache_fp8=torch.zeros(4, 2, 8, 8, dtype=torch.uint8)), "match"),
    (dict(key_linear=torch.zeros(3, 2, 9), value_linear=torch.zeros(3, 2, 9)), "does not match"),
    (dict(value_linear=torch.zeros(2, 2, 8)), "must be"),
    (dict(key_linear=torch.zeros(3, 2, 8, dtype=torch.int32), value_linear=torch.zeros(3, 2, 8, dtype=torch.int32)), "floating"),
    (dict(slot_mapping=torch.zeros(2, dtype=torch.int64)), "length"),
    (dict(slot_mapping=torch.zeros(3)), "integer"),
    (dict(k_scales=torch.zeros(2)), "one scale per block"),
    (dict(k_scales=torch.zeros(4, 2, dtype=torch.float16)), "float32"),
    (dict(v_scales=torch.zeros(2).expand(4, 2)), "expanded"),
    (dict(key_cache_fp8=torch.zeros(1, 2, 8, 16, dtype=torch.uint8).expand(4, 2, 8, 16)), "expanded"),
    (dict(k_scales=torch.zeros(4, 2, device="meta")), "device"),
])
def test_store_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        _store(**change)


def _attention(**change):
    a = dict(query=torch.zeros(2, 4, 8), key_cache_fp8=torch.zeros(4, 2, 8, 16, dtype=torch.uint8),
             value_cache_fp8=torch.zeros(4, 2, 8, 16, dtype=torch.uint8), block_tables=torch.zeros(2, 3, dtype=torch.int32),
             seq_lens=torch.zeros(2, dtype=torch.int32), k_scales=torch.zeros(4, 2), v_scales=torch.zeros(4, 2))
    a.update(change)
    return musa_aiter.kv_paged_attention_fp8(**a)


@pytest.mark.parametrize("change,match", [
    (dict(query=torch.zeros(2, 32)), "query must be"),
    (dict(query=torch.zeros(2, 4, 8, dtype=torch.float64)), "float32, float16 or bfloat16"),
    (dict(query=torch.zeros(2, 4, 9)), "head_dim"),
    (dict(query=torch.zeros(2, 3, 8)), "multiple"),
    (dict(query=torch.zeros(2, 0, 8)), "multiple"),
    (dict(query=torch.zeros(3, 4, 8)), "one query row"),
    (dict(fp8_format="e3m4"), "unsupported"),
    (dict(key_cache_fp8=torch.zeros(1, 4, 2, 8, 16, dtype=torch.uint8)), "one layer"),
    (dict(key_cache_fp8=torch.zeros(4, 2, 8, 16, dtype=torch.int8)), "uint8"),
    (dict(block_tables=torch.zeros(2, dtype=torch.int32)), "max_blocks"),
    (dict(block_tables=torch.zeros(2, 3)), "integer"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), "seq_lens"),
    (dict(query_starts=torch.zeros(2, dtype=torch.int32)), "batch \\+ 1"),
    (dict(query_starts=torch.zeros(3)), "integer"),
    (dict(k_scales=torch.zeros(2)), "one scale per block"),
    (dict(v_scales=torch.zeros(4, 2, dtype=torch.float64)), "float32"),
    (dict(window=0), "window"),
    (dict(max_seq_len=-1), "max_seq_len"),
    (dict(softmax_scale=float("nan")), "finite"),
    (dict(out=torch.zeros(2, 4, 8, dtype=torch.float16)), "out must match"),
    (dict(out=torch.zeros(2, 4, 7)), "out must match"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32, device="meta")), "device"),
])
def test_attention_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        _attention(**change)


def test_head_dims_past_the_kernels():
    with pytest.raises(ValueError, match="at most 512"):
        _attention(query=torch.zeros(2, 4, 513), key_cache_fp8=torch.zeros(4, 2, 513, 16, dtype=torch.uint8),
                   value_cache_fp8=torch.zeros(4, 2, 513, 16, dtype=torch.uint8))


def _pages(which, **change):
    a = dict(key_cache=torch.zeros(4, 2, 8, 16), value_cache=torch.zeros(4, 2, 8, 16),
             block_tables=torch.zeros(2, 3, dtype=torch.int32), seq_lens=torch.zeros(2, dtype=torch.int32),
             ref_counts=torch.zeros(4, dtype=torch.int32))
    rows = torch.zeros(2, dtype=torch.int32)
    if which == "extend":
        a |= dict(new_lens=rows, max_new=2)
    elif which == "compact":
        del a["seq_lens"]
    else:
        del a["key_cache"], a["value_cache"]
        a |= {"parents" if which == "fork" else "keep_lens": rows, "block_size": 16}
    a.update(change)
    call = {"extend": musa_aiter.kv_extend_paged_sequences, "fork": musa_aiter.kv_fork_paged_sequences,
            "free": musa_aiter.kv_free_paged_sequences, "compact": musa_aiter.kv_compact_paged_blocks}[which]
    return call(**a)


@pytest.mark.parametrize("which,change,match", [
    ("extend", dict(max_new=-1), "max_new"),
    ("extend", dict(new_lens=torch.zeros(3, dtype=torch.int32)), "new_lens"),
    ("extend", dict(new_lens=torch.zeros(2)), "integer"),
    ("extend", dict(value_cache=torch.zeros(4, 2, 8, 8)), "one shape"),
    ("extend", dict(k_scales=torch.zeros(4, 2)), "together"),
    ("extend", dict(k_scales=torch.zeros(4, 2), v_scales=torch.zeros(2).expand(4, 2)), "contiguous"),
    ("extend", dict(key_cache=torch.zeros(4, 2, 16, 8).transpose(2, 3)), "contiguous"),
    ("extend", dict(ref_counts=torch.zeros(5, dtype=torch.int32)), "ref_counts"),
    ("extend", dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "share one dtype"),
    ("extend", dict(block_tables=torch.zeros(2, 3, dtype=torch.int16), seq_lens=torch.zeros(2, dtype=torch.int16),
                    ref_counts=torch.zeros(4, dtype=torch.int16)), "int32 or int64"),
    ("compact", dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).t()), "contiguous"),
    ("compact", dict(block_tables=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), "contiguous"),
    ("compact", dict(ref_counts=torch.zeros(8, dtype=torch.int32)[::2]), "contiguous"),
    ("fork", dict(parents=torch.zeros(2, 1, dtype=torch.int32)), "parents"),
    ("fork", dict(block_size=0), "block_size"),
    ("fork", dict(ref_counts=torch.zeros(4, 1, dtype=torch.int32)), "ref_counts"),
    ("free", dict(keep_lens=torch.zeros(1, dtype=torch.int32)), "keep_lens"),
    ("free", dict(keep_lens=torch.zeros(2, dtype=torch.bool)), "integer"),
    ("free", dict(seq_lens=torch.zeros(4, dtype=torch.int32)[::2]), "contiguous"),
])
def test_page_refusals(which, change, match):
    with pytest.raises(ValueError, match=match):
        _pages(which, **change)


def test_only_rocm_tensors():
    for call in (_store, _attention, *(lambda w=w: _pages(w) for w in ("extend", "fork", "free", "compact"))):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()
