"""Refusals of the cache append, the paged attention and the sampler, on the
host: every call here returns before any HIP call. And the index arithmetic of
a batch, on a CPU build of the header that the kernels use."""
from __future__ import annotations

import ctypes
import os
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
P = 4096  # an aligned address that is never followed
INVALID, UNSUPPORTED = 1, 2


def cache(qk, **more):
    return qk.KVCache(**({"k": P, "v": P, "type": 1, "pages": 10, "page_size": 16, "kv_heads": 2, "head_dim": 128,
                          "page_stride": 4096, "token_stride": 256, "head_stride": 128, "fault": None} | more))


def batch(qk, **more):
    return qk.KVBatch(**({"sequences": 2, "tokens": 3, "token_start": P, "context": P, "page_table": P,
                          "table_stride": 4} | more))


def rope(qk, **more):
    return qk.Rope(**({"q_norm": P, "k_norm": P, "eps": 1e-6, "base": 1e4, "dims": 128, "interleaved": 0} | more))


BAD_CACHES = [({"type": 0}, UNSUPPORTED), ({"type": 12}, UNSUPPORTED), ({"head_dim": 96}, INVALID),
              ({"head_dim": 0}, INVALID), ({"pages": 0}, INVALID), ({"pages": 1 << 31}, INVALID),
              ({"page_size": 0}, INVALID), ({"page_size": 65537}, INVALID), ({"kv_heads": 0}, INVALID),
              ({"token_stride": 132}, INVALID), ({"head_stride": 64}, INVALID), ({"token_stride": 64}, INVALID),
              ({"page_stride": -8}, INVALID), ({"token_stride": 1 << 31}, INVALID), ({"k": None}, INVALID),
              ({"v": P + 8}, INVALID), ({"fault": P + 2}, INVALID)]
BAD_BATCHES = [{"sequences": -1}, {"sequences": 65536}, {"tokens": -1}, {"tokens": (1 << 24) + 1}, {"table_stride": 0},
               {"token_start": None}, {"context": None}, {"page_table": None}, {"context": P + 1}]


def test_append_refusals(qk):
    lib = qk.load()

    def call(c=None, b=None, r=None, q=P, qs=1024, k=P, ks=256, v=P, vs=256, heads=8, out=2 * P, kind=0):
        return lib.qk_kv_append(c or cache(qk), b or batch(qk), q, qs, k, ks, v, vs, heads, r or rope(qk), out, kind, None)

    for bad, code in BAD_CACHES:
        assert call(cache(qk, **bad)) == code, bad
        assert lib.qk_last_error()
    for bad in BAD_BATCHES:
        assert call(b=batch(qk, **bad)) == INVALID, bad
    for bad in ({"dims": 12}, {"dims": 136}, {"dims": -8}, {"base": 0.0}, {"base": float("nan")},
                {"base": float("inf")}, {"eps": 0.0}, {"eps": float("nan")}, {"q_norm": P + 2}):
        assert call(r=rope(qk, **bad)) == INVALID, bad
    for bad in ({"q": None}, {"k": None}, {"v": None}, {"out": None}, {"qs": 1023}, {"ks": 255}, {"vs": -1},
                {"heads": 7}, {"heads": -2}, {"heads": 8192, "qs": 1 << 20}, {"q": P + 2}, {"out": 2 * P + 4},
                {"out": P, "qs": 1032}, {"out": P, "kind": 1}):
        assert call(**bad) == INVALID, bad
    for kind in (30, 12, 99):
        assert call(kind=kind) == UNSUPPORTED
    assert lib.qk_kv_append(None, batch(qk), P, 1024, P, 256, P, 256, 8, None, P, 0, None) == INVALID
    # nothing to do: no pointer is looked at
    none = dict(token_start=None, context=None, page_table=None)
    assert call(cache(qk, k=None, v=None), batch(qk, tokens=0, **none), q=None, k=None, v=None, out=None) == 0
    assert call(cache(qk, k=None, v=None), batch(qk, sequences=0, **none), q=None, k=None, v=None, out=None) == 0


def test_attention_refusals(qk):
    lib = qk.load()

    def call(c=None, b=None, q=P, kind=0, stride=1024, heads=8, scale=0.1, window=0, most=100, out=P, lse=None, ws=P,
             n=1 << 40):
        return lib.qk_paged_attention(c or cache(qk), b or batch(qk), q, kind, stride, heads, scale, window, most, out,
                                      lse, ws, n, None)

    for bad, code in BAD_CACHES:
        assert call(cache(qk, **bad)) == code, bad
    for bad in BAD_BATCHES:
        assert call(b=batch(qk, **bad)) == INVALID, bad
    for bad in ({"q": None}, {"out": None}, {"q": P + 8}, {"out": P + 4}, {"lse": P + 2}, {"stride": 1023},
                {"stride": 1026}, {"heads": 0}, {"heads": 9}, {"window": -1}, {"most": -1}, {"scale": float("nan")},
                {"scale": float("inf")}, {"ws": P + 128}):
        assert call(**bad) == INVALID, bad
    assert call(kind=1, stride=1028) == INVALID  # 16-bit rows 8 bytes off
    assert call(kind=30) == UNSUPPORTED
    assert call(cache(qk, type=30), kind=1) == UNSUPPORTED
    size = lib.qk_paged_attention_workspace_size
    n = size(cache(qk), batch(qk), 0, 8, 0, 1 << 20)
    if n:
        assert call(most=1 << 20, n=n - 1) == INVALID and b"small" in lib.qk_last_error()
        assert call(most=1 << 20, ws=None) == INVALID
    assert size(cache(qk, head_dim=100), batch(qk), 0, 8, 0, 100) == 0
    assert size(cache(qk), batch(qk), 30, 8, 0, 100) == 0
    assert size(cache(qk), batch(qk), 0, 7, 0, 100) == 0
    none = dict(token_start=None, context=None, page_table=None)
    assert call(cache(qk, k=None, v=None), batch(qk, tokens=0, **none), q=None, out=None, ws=None, n=0) == 0
    assert lib.qk_kv_check(None, None) == INVALID
    assert lib.qk_kv_check(cache(qk), None) == 0  # no word to look at


def test_sample_refusals(qk):
    lib = qk.load()

    def call(x=P, rows=2, V=100, stride=100, heat=P, k=None, p=None, m=None, u=P, token=P, share=None, ws=P, n=1 << 40):
        return lib.qk_sample(x, rows, V, stride, heat, k, p, m, u, token, share, ws, n, None)

    for bad in ({"rows": -1}, {"rows": 65536}, {"V": 0}, {"V": (1 << 24) + 1, "stride": 1 << 25}, {"stride": 99},
                {"x": None}, {"heat": None}, {"u": None}, {"token": None}, {"x": P + 2}, {"k": P + 1}, {"p": P + 2},
                {"m": P + 3}, {"share": P + 2}, {"ws": P + 8}):
        assert call(**bad) == INVALID, bad
        assert lib.qk_last_error()
    n = lib.qk_sample_workspace_size(2, 100)
    if n:
        assert call(n=n - 1) == INVALID and call(ws=None) == INVALID
    assert lib.qk_sample_workspace_size(-1, 100) == 0 and lib.qk_sample_workspace_size(1, 1 << 25) == 0
    assert call(x=None, rows=0, heat=None, u=None, token=None, ws=None, n=0) == 0


def test_structures_match_the_header(qk, tmp_path):
    """Sizes and field offsets of the ctypes structures are the C compiler's."""
    lines = []
    for name, kind in (("qk_kv_cache", qk.KVCache), ("qk_kv_batch", qk.KVBatch), ("qk_rope", qk.Rope)):
        lines.append(f"_Static_assert(sizeof({name}) == {ctypes.sizeof(kind)}, \"{name}\");")
        for field, _ in kind._fields_:
            lines.append(f"_Static_assert(offsetof({name}, {field}) == {getattr(kind, field).offset}, \"{field}\");")
    src = tmp_path / "layout.c"
    src.write_text('#include "qk_abi.h"\n' + "\n".join(lines) + "\nint main(void) { return 0; }\n")
    res = subprocess.run(["gcc", "-std=c11", "-fsyntax-only", "-I", str(ROOT / "include"), str(src)],
                         capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stderr


def test_batch_indices_stay_in_bounds(tmp_path):
    """tests/cpp/kv_index_check.cpp under the address and UB sanitizers."""
    exe = tmp_path / "kv_index"
    res = subprocess.run(["g++", "-std=c++20", "-g", "-O1", "-Wall", "-Wextra", "-fsanitize=address,undefined",
                          "-fno-sanitize-recover=undefined", "-I",
                          str(ROOT / "qwen3-4b-q4_k_m-inference-engine_amd" / "csrc"),
                          str(ROOT / "tests" / "cpp" / "kv_index_check.cpp"), "-o", str(exe)],
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1")
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    assert res.returncode == 0 and "all checks passed" in res.stdout, res.stdout + res.stderr


def _sanitized(tmp_path, name):
    """tests/cpp/<name>.cpp under the address and UB sanitizers."""
    exe = tmp_path / name
    res = subprocess.run(["g++", "-std=c++20", "-g", "-O1", "-Wall", "-Wextra", "-fsanitize=address,undefined",
                          "-fno-sanitize-recover=undefined", "-I", str(ROOT / "include"), "-I",
                          str(ROOT / "qwen3-4b-q4_k_m-inference-engine_amd" / "csrc"),
                          str(ROOT / "tests" / "cpp" / f"{name}.cpp"), "-o", str(exe)],
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-3000:]
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1")
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300, env=env)
    assert res.returncode == 0 and "all checks passed" in res.stdout, res.stdout + res.stderr


def test_attention_plans_hold_for_lengths_of_any_size(tmp_path):
    _sanitized(tmp_path, "attention_plan_check")


@pytest.mark.parametrize("tokens", [1, 512])
def test_attention_workspace_of_windows_and_bounds_of_any_size(qk, tokens):
    """INT64_MAX for "no window" takes the workspace of no window, and is refused without it."""
    lib = qk.load()
    most = (1 << 63) - 1
    b = batch(qk, sequences=1, tokens=tokens)
    c = cache(qk, kv_heads=8, token_stride=1024, page_stride=16384)
    size = lambda window, context: lib.qk_paged_attention_workspace_size(c, b, 0, 32, window, context)  # noqa: E731
    for context in (1000, 4096, 131072):
        none = size(0, context)
        assert none > 0 or (tokens, context) == (512, 1000)
        for window in (most, most - 1, most - 255, 1 << 40, (1 << 31) - 1):
            assert size(window, context) == none, (window, context)
            call = lambda ws, n: lib.qk_paged_attention(c, b, P, 0, 4096, 32, 0.1, window, context, P, None, ws, n,  # noqa: E731
                                                        None)
            if none:
                assert call(None, 0) == INVALID and call(P, none - 1) == INVALID
    assert size(0, most) == size(0, (1 << 31) - 1) > 0


def test_attention_keys_stay_in_the_page_table(tmp_path):
    _sanitized(tmp_path, "attention_keys_check")


def test_a_check_refuses_a_word_out_of_place(qk):
    assert qk.load().qk_kv_check(cache(qk, fault=P + 2), None) == INVALID


def test_attention_refuses_more_workgroups_than_a_launch_holds(qk):
    lib = qk.load()
    c = cache(qk, kv_heads=4096, token_stride=4096 * 128, page_stride=16 * 4096 * 128)
    b = batch(qk, sequences=65535, tokens=65535)
    for q_type in (0, 1):
        assert lib.qk_paged_attention(c, b, P, q_type, 4096 * 128, 4096, 0.1, 0, 100, P, None, P, 1 << 40, None) == INVALID
        assert lib.qk_paged_attention_workspace_size(c, b, q_type, 4096, 0, 100) == 0
