"""CPU: argument checks of the operators on paged caches of plain values, and the packed calls' layouts."""

from __future__ import annotations

import ctypes
import pathlib
import re

import pytest
import torch

import musa_aiter
from musa_aiter import registry
from musa_aiter.ops import _hip

HEADER = pathlib.Path(__file__).resolve().parents[1] / "include" / "musa_aiter_kv_paged_attention.h"
NAMES = ("kv_paged_attention", "kv_paged_attention_tree", "kv_accumulate_attention_weights", "kv_evict_paged_tokens")


def test_registered_and_exported():
    caps = registry.list_capabilities("kvattention")
    assert {c.name for c in caps} == set(NAMES)
    for cap in caps:
        assert cap.backends == ("rocm-hip",) and callable(getattr(musa_aiter, cap.name))


def _header() -> str:
    return re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)


@pytest.mark.parametrize("name,packed", [("paged_attention", "_CACHE_ATTENTION_CALL"), ("evict", "_EVICT_CALL")])
def test_packed_calls_match_the_header(name, packed):
    body = re.search(r"typedef struct musa_aiter_hip_%s_call \{(.*?)\}" % name, _header(), re.S).group(1)
    codes, fields = "", []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind = "Q" if "*" in decl else {"int64_t": "q", "int32_t": "i", "double": "d"}[decl.split()[0]]
        for field in decl.split(None, 1)[1].split(","):
            size = re.search(r"\[(\d+)\]", field)
            fields += [field.split()[-1]] * (int(size.group(1)) if size else 1)
            codes += kind * (int(size.group(1)) if size else 1)
    got = getattr(_hip, packed).format.lstrip("<")
    assert re.sub(r"(\d+)(\w)", lambda m: m.group(2) * int(m.group(1)), got) == codes
    at = {"paged_attention": _hip._CACHE_ATTENTION_WORKSPACE_AT, "evict": _hip._EVICT_WORKSPACE_AT}[name]
    assert at % 8 == 0 and fields[at // 8].endswith("workspace") and fields[at // 8 + 1] == "workspace_bytes"


def test_entries_exported_and_refuse_nothing_to_do():
    lib = ctypes.CDLL(str(_hip.LIB_PATH))
    symbols = re.findall(r"(?:int64_t|int)\s+(musa_aiter_hip_\w+)\s*\(", _header())
    assert len(symbols) == 5
    for symbol in symbols:
        assert hasattr(lib, symbol)
        f = _hip.fn(symbol)
        size = (_hip._EVICT_CALL if "evict" in symbol else _hip._CACHE_ATTENTION_CALL).size
        if symbol.endswith("workspace"):
            assert f(None) == 0 and f(bytes(size)) == 0
            continue
        assert f(None, None) != 0
        assert f(bytes(size), None) != 0  # all sizes zero or pointers missing: an error, before any launch


def _attention(op, **change):
    a = dict(query=torch.zeros(3, 4, 8), key_cache=torch.zeros(5, 2, 8, 16), value_cache=torch.zeros(5, 2, 8, 16),
             block_tables=torch.zeros(3, 4, dtype=torch.int32), seq_lens=torch.zeros(3, dtype=torch.int32))
    if op == "kv_paged_attention_tree":
        a["tree_masks"] = torch.zeros(3, 1, dtype=torch.int64)
    if op == "kv_accumulate_attention_weights":
        del a["value_cache"]
        a.update(weights=torch.zeros(3, 2, 64), lse=torch.zeros(3, 4))
    a.update(change)
    return getattr(musa_aiter, op)(**a)


COMMON = [
    (dict(query=torch.zeros(3, 32)), "query must be"),
    (dict(query=torch.zeros(3, 4, 8, dtype=torch.int32)), "float32"),
    (dict(query=torch.zeros(3, 4, 8, dtype=torch.float64)), "float32"),
    (dict(query=torch.zeros(3, 4, 8, dtype=torch.float16)), "share one dtype"),
    (dict(query=torch.zeros(3, 4, 16)), "head_dim"),
    (dict(query=torch.zeros(3, 3, 8)), "multiple of kv_heads"),
    (dict(query=torch.zeros(3, 0, 8)), "multiple of kv_heads"),
    (dict(key_cache=torch.zeros(5, 2, 16)), "4-D"),
    (dict(key_cache=torch.zeros(0, 2, 8, 16), value_cache=torch.zeros(0, 2, 8, 16)), "positive"),
    (dict(block_tables=torch.zeros(12, dtype=torch.int32)), "block_tables"),
    (dict(block_tables=torch.zeros(3, 4)), "integer"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32)), "seq_lens"),
    (dict(query_starts=torch.zeros(3, dtype=torch.int32)), "query_starts"),
    (dict(query=torch.zeros(4, 4, 8)), "one query row per sequence"),
    (dict(max_seq_len=-1), "max_seq_len"),
    (dict(softmax_scale=float("inf")), "finite"),
    (dict(block_tables=torch.zeros(3, 1, dtype=torch.int32).expand(3, 1 << 26)), "2\\*\\*29"),
]
SIGHT = [(dict(window=0), "window"), (dict(window=-3), "window"), (dict(window=5, sinks=-1), "sinks")]
OUT = [(dict(out=torch.zeros(3, 4, 9)), "out must"), (dict(out=torch.zeros(3, 4, 8, dtype=torch.float16)), "out must"),
       (dict(out=torch.zeros(1, 4, 8).expand(3, 4, 8)), "expanded"),
       (dict(value_cache=torch.zeros(5, 2, 8, 8)), "match"),
       (dict(value_cache=torch.zeros(5, 2, 8, 16, dtype=torch.float16)), "share one dtype")]
MASKS = [(dict(tree_masks=torch.zeros(3, dtype=torch.int64)), "tree_masks"),
         (dict(tree_masks=torch.zeros(2, 1, dtype=torch.int64)), "tree_masks"),
         (dict(tree_masks=torch.zeros(3, 0, dtype=torch.int64)), "tree_masks"),
         (dict(tree_masks=torch.zeros(3, 1, dtype=torch.int32)), "int64")]
WEIGHTS = [(dict(weights=torch.zeros(3, 2)), "weights must"), (dict(weights=torch.zeros(2, 2, 64)), "weights must"),
           (dict(weights=torch.zeros(3, 4, 64)), "weights must"),
           (dict(weights=torch.zeros(3, 2, 64, dtype=torch.float64)), "float32"),
           (dict(lse=torch.zeros(3, 2)), "lse must"), (dict(lse=torch.zeros(3, 4, dtype=torch.float16)), "float32"),
           (dict(weights=torch.zeros(1, 2, 64).expand(3, 2, 64)), "expanded")]


@pytest.mark.parametrize("op,change,match", [
    *[("kv_paged_attention", *x) for x in COMMON + SIGHT + OUT],
    *[("kv_paged_attention_tree", *x) for x in COMMON + OUT + MASKS],
    *[("kv_accumulate_attention_weights", *x) for x in COMMON + SIGHT + WEIGHTS
      if "value_cache" not in x[0] or "key_cache" in x[0]]])
def test_refusals(op, change, match):
    if op == "kv_accumulate_attention_weights":
        change = {k: v for k, v in change.items() if k != "value_cache"}
    with pytest.raises(ValueError, match=match):
        _attention(op, **change)


@pytest.mark.parametrize("op", NAMES[:3])
def test_cpu_tensors_raise(op):
    with pytest.raises(RuntimeError, match="ROCm"):
        _attention(op)


def _evict(**change):
    a = dict(key_cache=torch.zeros(2, 5, 2, 8, 16), value_cache=torch.zeros(2, 5, 2, 8, 16),
             weights=torch.zeros(2, 3, 2, 64), block_tables=torch.zeros(3, 4, dtype=torch.int32),
             seq_lens=torch.zeros(3, dtype=torch.int32), keep_lens=torch.zeros(3, dtype=torch.int32))
    a.update(change)
    return musa_aiter.kv_evict_paged_tokens(**a)


@pytest.mark.parametrize("change,match", [
    (dict(key_cache=torch.zeros(2, 5, 2, 8, 16, dtype=torch.float64), value_cache=torch.zeros(2, 5, 2, 8, 16, dtype=torch.float64)), "bytes"),
    (dict(value_cache=torch.zeros(2, 5, 2, 8, 16, dtype=torch.float16)), "dtype"),
    (dict(value_cache=torch.zeros(2, 5, 2, 8, 8)), "match"),
    (dict(key_cache=torch.zeros(5, 2, 16)), "4-D"),
    (dict(block_tables=torch.zeros(12, dtype=torch.int32)), "block_tables"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int32)), "seq_lens"),
    (dict(keep_lens=torch.zeros(3, 1, dtype=torch.int32)), "keep_lens"),
    (dict(keep_lens=torch.zeros(3)), "integer"),
    (dict(ref_counts=torch.zeros(4, dtype=torch.int32)), "ref_counts"),
    (dict(weights=torch.zeros(3, 2, 64)), "weights must"),
    (dict(weights=torch.zeros(2, 3, 2, 64, dtype=torch.float16)), "float32"),
    (dict(weights=torch.zeros(1, 3, 2, 64).expand(2, 3, 2, 64)), "expanded"),
    (dict(key_cache=torch.zeros(1, 5, 2, 8, 16).expand(2, 5, 2, 8, 16)), "contiguous"),
    (dict(key_cache=torch.zeros(2, 5, 2, 16, 8).transpose(3, 4)), "contiguous"),
    (dict(sinks=-1), "non-negative"), (dict(recent=-1), "non-negative"),
    (dict(block_tables=torch.zeros(3, 1, dtype=torch.int32).expand(3, 1 << 26)), "2\\*\\*29")])
def test_evict_refusals(change, match):
    with pytest.raises(ValueError, match=match):
        _evict(**change)


def test_evict_takes_two_caches():
    one = torch.zeros(2, 5, 2, 8, 16)
    with pytest.raises(ValueError, match="one tensor"):
        _evict(key_cache=one, value_cache=one)


def test_evict_on_cpu_tensors_raises():
    with pytest.raises(RuntimeError, match="ROCm"):
        _evict()


def test_the_oracle_against_counted_cases():
    """Three tokens, one head: weights by hand."""
    import numpy as np

    from tests import cache_attention_ref as ref

    key = np.zeros((1, 1, 1, 4))
    key[0, 0, 0] = [0.0, np.log(2.0), np.log(3.0), 99.0]
    value = np.asarray([1.0, 2.0, 4.0, 99.0]).reshape(1, 1, 1, 4)
    args = (np.ones((1, 1, 1)), key, value, np.zeros((1, 1), dtype=int), [3])
    out, lse, *_ = ref.attention(*args)
    assert np.allclose(out, (1 + 4 + 12) / 6) and np.allclose(lse, np.log(6))
    out, *_ = ref.attention(*args, window=1, sinks=1)
    assert np.allclose(out, (1 + 12) / 4)
    out, *_ = ref.attention(*args, masks=np.zeros((1, 1), dtype=np.int64))
    assert np.allclose(out, (1 + 4) / 3)
    got, _, terms = ref.gathered(np.ones((1, 1, 2)), *args[:2], *args[3:], np.log(np.full((1, 1), 6.0)))
    assert np.allclose(got, [[[1 + 1 / 6, 1 + 2 / 6]]]) and (terms == 1).all()
    k, v = key.copy(), value.copy()
    w = np.asarray([[[1.0, 5.0, 3.0, 7.0]]], dtype=np.float32)
    assert ref.evict(k, v, w, args[3], [4], [2], recent=1).tolist() == [2]
    assert w.tolist() == [[[5.0, 7.0, 0.0, 0.0]]] and v.ravel().tolist() == [2.0, 99.0, 4.0, 99.0]
