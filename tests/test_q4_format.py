"""The Q4_1 blocks of a cache, on the host: what the definition promises of them."""
from __future__ import annotations

import numpy as np
import pytest

import q4_ref
import serving_ref as ref


@pytest.mark.parametrize("size,offset", [(1.0, 0.0), (30.0, 1000.0), (1e-6, 0.0), (2e4, 0.0), (1e-3, -500.0), (0.0, 7.3)])
def test_values_are_within_half_a_code_of_what_was_stored(size, offset):
    """m off by half an F16 step, d below the range's 15th by a step of its own, a value by its rounding."""
    rng = np.random.default_rng(int(size) + 5)
    x = (rng.standard_normal((50, 128)) * size + offset).astype(np.float32)
    blocks = q4_ref.blocks_of(x)
    d, m, code = q4_ref.parts(blocks)
    v = ref.decode(q4_ref.values(blocks), ref.F16)
    rows = x.reshape(50, 4, 32).astype(np.float64)
    span = rows.max(-1, keepdims=True) - m
    off = d / 2 + 2.0 ** -11 * (np.abs(m) + np.abs(rows)) + 2.0 ** -10 * np.maximum(span, 0) + 16 * 2.0 ** -24
    beyond = (np.abs(rows) >= 65520).any(-1)  # of F16: NaN as a whole
    v = v.reshape(rows.shape)
    assert np.isnan(v[beyond]).all()
    assert (np.abs(v - rows) <= off)[~beyond].all()
    assert np.isfinite(v[~beyond]).all() and code.max() <= 15


def test_blocks_at_the_ends_of_f16():
    """Ranges of all of F16 stay finite; what rounds to an infinity, or a NaN, takes its block with it."""
    x = np.zeros((1, 128), np.float32)
    x[0, 3], x[0, 9] = 65504, -65504
    x[0, 40] = 65520
    x[0, 70] = np.nan
    x[0, 100] = -np.inf
    v = ref.decode(q4_ref.values(q4_ref.blocks_of(x)), ref.F16)[0]
    assert np.isfinite(v[:32]).all() and v[9] == -65504 and v[3] >= 65504 * (1 - 2.0 ** -9)
    assert np.isnan(v[32:]).all()


def test_codes_lie_as_in_gguf_files():
    x = np.arange(32, dtype=np.float32)[None] / 31 * 15
    b = q4_ref.blocks_of(np.tile(x, 2))[0]
    assert len(b) == 40
    assert b[4] & 15 == 0 and b[4] >> 4 == np.rint(16 / 31 * 15) and b[19] >> 4 == 15
