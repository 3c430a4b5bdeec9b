"""Refusals of the calls on Q4_1 caches, cached rows, weights and evictions, on the host:
every call here returns before any HIP call. And their plans and index arithmetic."""
from __future__ import annotations

import ctypes
import pathlib
import subprocess

import pytest

from test_serving_abi import (BAD_BATCHES, BAD_CACHES, INVALID, P, UNSUPPORTED, _sanitized, batch, cache, rope)

ROOT = pathlib.Path(__file__).resolve().parents[1]
Q4_1 = 3
NONE = dict(token_start=None, context=None, page_table=None)


def test_q4_1_caches_need_whole_blocks(qk):
    lib = qk.load()

    def append(c, kind=0):
        return lib.qk_kv_append(c, batch(qk), P, 1024, P, 256, P, 256, 8, rope(qk), 2 * P, kind, None)

    for bad in ({"token_stride": 264}, {"head_stride": 136}, {"page_stride": 4104}, {"head_dim": 96}, {"token_stride": 96}):
        assert append(cache(qk, type=Q4_1, **bad)) == INVALID, bad
    for kind in (30, Q4_1, 12):
        assert append(cache(qk, type=Q4_1), kind) == UNSUPPORTED
    assert lib.qk_paged_attention(cache(qk, type=Q4_1), batch(qk), P, 30, 1024, 8, 0.1, 0, 100, P, None, P, 1 << 40, None) == UNSUPPORTED
    size = lib.qk_paged_attention_workspace_size
    n = size(cache(qk, type=Q4_1), batch(qk, sequences=1, tokens=1), 0, 8, 0, 1 << 20)
    assert n > 0 and size(cache(qk, type=Q4_1), batch(qk), 30, 8, 0, 100) == 0
    assert lib.qk_paged_attention(cache(qk, type=Q4_1), batch(qk, sequences=1, tokens=1), P, 0, 1024, 8, 0.1, 0, 1 << 20, P, None,
                                  P, n - 1, None) == INVALID


def test_append_at_refusals(qk):
    lib = qk.load()

    def call(c=None, b=None, seen=P, k=P, ks=256, v=P, heads=8, kind=0, out=2 * P):
        return lib.qk_kv_append_at(c or cache(qk), b or batch(qk), seen, P, 1024, k, ks, v, 256, heads, rope(qk), out, kind, None)

    for bad, code in BAD_CACHES:
        assert call(cache(qk, **bad)) == code, bad
    for bad in BAD_BATCHES:
        assert call(b=batch(qk, **bad)) == INVALID, bad
    for bad in ({"seen": P + 2}, {"k": None}, {"v": None}, {"ks": 255}, {"heads": 7}, {"out": 2 * P + 4}):
        assert call(**bad) == INVALID, bad
    assert call(b=batch(qk, tokens=0, **NONE), seen=None, k=None, v=None, out=None) == 0


def test_rows_refusals(qk):
    lib = qk.load()

    def call(c=None, b=None, k=P, v=P, kind=0):
        return lib.qk_kv_rows(c or cache(qk), b or batch(qk), k, v, kind, None)

    for bad, code in BAD_CACHES:
        assert call(cache(qk, **bad)) == code, bad
    for bad in BAD_BATCHES:
        assert call(b=batch(qk, **bad)) == INVALID, bad
    for bad in ({"k": None, "v": None}, {"k": P + 8}, {"v": P + 4}):
        assert call(**bad) == INVALID, bad
    for c, kind in ((cache(qk), 30), (cache(qk, type=30), 1), (cache(qk, type=Q4_1), Q4_1), (cache(qk), 12)):
        assert call(c, kind=kind) == UNSUPPORTED
    assert call(b=batch(qk, tokens=0, **NONE), k=None, v=None) == 0
    assert lib.qk_kv_rows(None, batch(qk), P, P, 0, None) == INVALID


def weights(qk, **more):
    return qk.KVWeights(**({"weight": P, "position": P} | more))


def test_weigh_refusals(qk):
    lib = qk.load()

    def call(c=None, b=None, seen=None, q=P, kind=0, stride=1024, heads=8, scale=0.1, lse=P, most=100, w=None, ws=P, n=1 << 40):
        return lib.qk_kv_weigh(c or cache(qk), b or batch(qk), seen, q, kind, stride, heads, scale, lse, most,
                               w or weights(qk), ws, n, None)

    for bad, code in BAD_CACHES:
        assert call(cache(qk, **bad)) == code, bad
    for bad in BAD_BATCHES:
        assert call(b=batch(qk, **bad)) == INVALID, bad
    for bad in ({"q": None}, {"q": P + 8}, {"lse": None}, {"lse": P + 2}, {"seen": P + 1}, {"stride": 1023}, {"stride": 1026},
                {"heads": 9}, {"heads": 0}, {"scale": float("nan")}, {"scale": float("inf")}, {"most": -1}, {"ws": P + 128}):
        assert call(**bad) == INVALID, bad
    for bad in ({"weight": None}, {"position": None}, {"weight": P + 2}, {"position": P + 1}):
        assert call(w=weights(qk, **bad)) == INVALID, bad
    assert call(kind=30) == UNSUPPORTED
    assert call(b=batch(qk, tokens=0, **NONE), q=None, lse=None, ws=None, n=0) == 0
    assert lib.qk_kv_weigh(cache(qk), batch(qk), None, P, 0, 1024, 8, 0.1, P, 100, None, P, 1 << 40, None) == INVALID
    size = lib.qk_kv_weigh_workspace_size
    large = batch(qk, sequences=1, tokens=4000)
    n = size(cache(qk), large, 0, 8, 4000)
    assert n > 0
    assert call(b=large, most=4000, n=n - 1) == INVALID and b"small" in lib.qk_last_error()
    assert call(b=large, most=4000, ws=None) == INVALID
    assert size(cache(qk, head_dim=96), large, 0, 8, 4000) == 0 and size(cache(qk), large, 0, 7, 4000) == 0
    assert size(cache(qk), large, 0, 8, -1) == 0
    # more workgroups than a launch holds
    wide = cache(qk, kv_heads=4096, token_stride=4096 * 128, page_stride=16 * 4096 * 128)
    assert call(wide, batch(qk, sequences=65535, tokens=65535), stride=4096 * 128, heads=4096, most=1 << 20) == INVALID


def test_evict_refusals(qk):
    lib = qk.load()

    def call(c=None, b=None, seen=None, w=None, keep=P, recent=P, most=100, out=2 * P, ws=P, n=1 << 40):
        return lib.qk_kv_evict(c or cache(qk), b or batch(qk), seen, w or weights(qk), keep, recent, most, out, ws, n, None)

    for bad, code in BAD_CACHES:
        assert call(cache(qk, **bad)) == code, bad
    for bad in BAD_BATCHES:
        assert call(b=batch(qk, **bad)) == INVALID, bad
    for bad in ({"keep": None}, {"recent": None}, {"out": None}, {"keep": P + 2}, {"recent": P + 1}, {"out": P + 3},
                {"out": P}, {"seen": P + 2}, {"most": 0}, {"most": -1}, {"most": (1 << 30) + 1}, {"ws": P + 8}, {"ws": None}):
        assert call(**bad) == INVALID, bad
    for bad in ({"weight": None}, {"position": P + 2}):
        assert call(w=weights(qk, **bad)) == INVALID, bad
    size = lib.qk_kv_evict_workspace_size
    n = size(cache(qk), batch(qk), 100)
    assert n > 0 and call(n=n - 1) == INVALID and b"small" in lib.qk_last_error()
    assert size(cache(qk), batch(qk), 0) == 0 and size(cache(qk, pages=0), batch(qk), 100) == 0
    assert call(b=batch(qk, sequences=0, **NONE), keep=None, recent=None, out=None, ws=None, n=0) == 0
    wide = cache(qk, kv_heads=4096, token_stride=4096 * 128, page_stride=16 * 4096 * 128)
    assert call(wide, batch(qk, sequences=65535), most=1000) == INVALID
    assert size(wide, batch(qk, sequences=65535), 1000) == 0


@pytest.mark.parametrize("name", ["seen", "keep", "recent"])
def test_evict_writes_lengths_beside_what_it_reads(qk, name):
    """Other workgroups still read those arrays when the first lengths are written."""
    arrays = {"seen": 4 * P, "keep": 5 * P, "recent": 6 * P}
    status = qk.load().qk_kv_evict(cache(qk), batch(qk), arrays["seen"], weights(qk), arrays["keep"], arrays["recent"], 100,
                                   arrays[name], P, 1 << 40, None)
    assert status == INVALID and b"own" in qk.load().qk_last_error()


@pytest.mark.parametrize("name,entries", [("context", 9), ("seen", 9), ("keep", 9), ("recent", 9), ("page_table", 9 * 4)])
def test_evict_lengths_may_not_overlap_what_it_reads(qk, name, entries):
    """Not by one entry at either end; side by side they may lie (and the workspace is looked at then)."""
    arrays = {"context": 3 * P, "seen": 4 * P, "keep": 5 * P, "recent": 6 * P, "page_table": 7 * P}
    b = batch(qk, sequences=9, context=arrays["context"], page_table=arrays["page_table"], table_stride=4)

    def call(out):
        status = qk.load().qk_kv_evict(cache(qk), b, arrays["seen"], weights(qk), arrays["keep"], arrays["recent"], 100, out,
                                       P, 0, None)
        return status, qk.load().qk_last_error()

    for out in (arrays[name], arrays[name] + 4, arrays[name] - 4, arrays[name] + 4 * (entries - 1), arrays[name] - 4 * 8):
        status, message = call(out)
        assert status == INVALID and b"own" in message, (out - arrays[name], message)
    for out in (arrays[name] + 4 * entries, arrays[name] - 4 * 9):
        status, message = call(out)
        assert status == INVALID and b"small" in message, (out - arrays[name], message)


def test_evict_lengths_beside_tables_of_any_stride(qk):
    """Rows of a table that lie further apart than addresses reach overlap nothing before them."""
    for stride in (1 << 40, (1 << 63) - 1):
        b = batch(qk, sequences=65535, context=1 << 30, page_table=1 << 40, table_stride=stride)
        for out, word in ((1 << 31, b"small"), ((1 << 40) + 8, b"own"), ((1 << 40) + (1 << 20), b"own")):
            status = qk.load().qk_kv_evict(cache(qk), b, None, weights(qk), 1 << 29, 1 << 28, 100, out, P, 0, None)
            assert status == INVALID and word in qk.load().qk_last_error(), (stride, out)


def test_the_weights_structure_matches_the_header(qk, tmp_path):
    lines = [f"_Static_assert(sizeof(qk_kv_weights) == {ctypes.sizeof(qk.KVWeights)}, \"size\");"]
    for field, _ in qk.KVWeights._fields_:
        lines.append(f"_Static_assert(offsetof(qk_kv_weights, {field}) == {getattr(qk.KVWeights, field).offset}, \"{field}\");")
    src = tmp_path / "layout.c"
    src.write_text('#include "qk_abi.h"\n' + "\n".join(lines) + "\nint main(void) { return 0; }\n")
    res = subprocess.run(["gcc", "-std=c11", "-fsyntax-only", "-I", str(ROOT / "include"), str(src)], capture_output=True,
                         text=True, timeout=60)
    assert res.returncode == 0, res.stderr


def test_plans_and_divisions_hold_for_lengths_of_any_size(tmp_path):
    _sanitized(tmp_path, "smaller_cache_check")
