"""examples/serve.py: append, attention and sampling together between the
library's projections. A captured decode step, replayed over growing contexts
with host work between the replays, draws the tokens that eager calls draw; a
session at temperature 0 takes the largest logit; sessions served together do
not see one another."""
from __future__ import annotations

import importlib.util
import pathlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location("serve_example", pathlib.Path(__file__).resolve().parents[1] / "examples" / "serve.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)
V = 4096


def test_captured_steps_draw_what_eager_steps_draw(gpu):
    prompts, tokens = [70, 17, 1, 5], 9  # a page of 64 ends within and between the steps
    print("[case] serve eager", flush=True)
    eager, _, server = example.serve(gpu, 2, prompts, tokens, V, captured=False)
    logits = server.logits.download(np.float32).reshape(-1, V)
    print("[case] serve captured", flush=True)
    captured, _, other = example.serve(gpu, 2, prompts, tokens, V, captured=True)
    assert np.array_equal(eager, captured)
    assert eager.max() < V and np.isfinite(logits).all()
    assert np.array_equal(logits.view(np.uint32), other.logits.download(np.float32).reshape(-1, V).view(np.uint32))
    assert eager[-1, 1] == logits[1].argmax()  # the second session's temperature is 0
    assert len({tuple(row) for row in eager}) > 1


def test_a_session_does_not_depend_on_its_neighbours(gpu):
    """The same session beside others of other lengths: attention and append
    give its rows the same bits whatever else the batch holds."""
    qk = gpu
    rng = np.random.default_rng(3)
    D, H, HK, P = 128, 8, 2, 16
    q, kv = rng.standard_normal((1, H, D)).astype(np.float32), rng.standard_normal((2, 41, HK, D)).astype(np.float32)
    results = []
    for others in ([], [5], [30, 1]):
        lengths = others + [41]
        held = [-(-n // P) for n in lengths]
        table = np.zeros((len(lengths), max(held)), np.int32)
        ids = np.random.default_rng(len(others)).permutation(sum(held)).astype(np.int32)
        for s, n in enumerate(held):
            table[s, :n] = ids[sum(held[:s]):][:n]
        dev = qk.DeviceBuffer.from_array
        pools = [dev(rng.standard_normal(sum(held) * P * HK * D).astype(np.float16)) for _ in range(2)]
        d = [dev(table), dev(np.asarray(lengths, np.int32))]
        cache = qk.KVCache(k=pools[0].ptr, v=pools[1].ptr, type=qk.TYPE_F16, pages=sum(held), page_size=P, kv_heads=HK,
                           head_dim=D, page_stride=P * HK * D, token_stride=HK * D, head_stride=D)
        new = [min(n, 2) for n in others] + [41]
        start = dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        batch = qk.KVBatch(sequences=len(lengths), tokens=sum(new), token_start=start.ptr, context=d[1].ptr,
                           page_table=d[0].ptr, table_stride=max(held))
        rows = rng.standard_normal((2, sum(new), HK, D)).astype(np.float32)
        rows[:, sum(new) - 41:] = kv
        k, v = dev(rows[0]), dev(rows[1])
        rope = qk.Rope(eps=1e-6, base=1e4, dims=D)
        qk.kv_append(cache, batch, None, 0, k, HK * D, v, HK * D, 0, rope, None, 0)
        one = dev(np.arange(len(lengths) + 1, dtype=np.int32))
        batch = qk.KVBatch(sequences=len(lengths), tokens=len(lengths), token_start=one.ptr, context=d[1].ptr,
                           page_table=d[0].ptr, table_stride=max(held))
        qs = rng.standard_normal((len(lengths), H, D)).astype(np.float32)
        qs[-1] = q[0]
        qd, out = dev(qs), qk.DeviceBuffer(4 * qs.size)
        n = qk.paged_attention_workspace_size(cache, batch, 0, H, 0, 41)
        ws = dev(np.zeros(max(n, 256), np.uint8))
        qk.paged_attention(cache, batch, qd, 0, H * D, H, D ** -0.5, 0, 41, out, None, ws, ws.nbytes)
        qk.synchronize()
        results.append(out.download(np.uint32).reshape(len(lengths), H, D)[-1])
    assert all(np.array_equal(r, results[0]) for r in results)
