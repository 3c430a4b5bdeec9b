"""The serving example with a smaller cache: Q4_1 blocks, and sessions cut to a budget."""
from __future__ import annotations

import importlib.util
import pathlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = pathlib.Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("serve_example", ROOT / "examples" / "serve.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("cache,keep", [("q4_1", 0), ("f16", 40), ("q4_1", 40), ("bf16", 33)])
def test_captured_steps_draw_what_eager_steps_draw(gpu, example, cache, keep):
    """And lengths, positions and pages fit all along (serve checks the fault word)."""
    print(f"[case] serve {cache} keep={keep}", flush=True)
    runs = [example.serve(gpu, 2, [70, 9, 41], 12, vocabulary=4096, captured=captured, cache=cache, keep=keep, recent=8)
            for captured in (True, False)]
    assert np.array_equal(runs[0][0], runs[1][0])
    server = runs[0][2]
    assert server.counts.tolist() == [70 + 11, 9 + 11, 41 + 11]
    if keep:
        assert server.lengths.tolist() == [keep + 1, 20, keep + 1]
        assert server.cut.download(np.int32).tolist() == [keep, 20, keep]


def test_a_budget_that_is_never_reached_changes_nothing(gpu, example):
    plain = example.serve(gpu, 2, [70, 9], 6, vocabulary=4096)
    kept = example.serve(gpu, 2, [70, 9], 6, vocabulary=4096, keep=1000)
    assert np.array_equal(plain[0], kept[0])
