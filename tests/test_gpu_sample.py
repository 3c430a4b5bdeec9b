"""qk_sample against the definition in 64 bits: the same token for every row
(no tolerance: a draw's border is only met by chance within 2^-40 of the kept
sum, and the rows' seeds are fixed), its probability within one fp32 rounding
and the 2^-30 that fixed-point weights of a large vocabulary may lose."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref

pytestmark = pytest.mark.gpu


class Sample:
    def __init__(self, qk, logits, heat, k=None, p=None, min_p=None, u=0.5, stride=None, seed=1):
        R, V = logits.shape
        self.qk, self.logits, self.stride = qk, logits.astype(np.float32), stride or V
        full = lambda x, t: None if x is None else np.broadcast_to(np.asarray(x, t), (R,)).copy()  # noqa: E731
        self.heat, self.k, self.p, self.min_p, self.u = (full(heat, np.float32), full(k, np.int32), full(p, np.float32),
                                                         full(min_p, np.float32), full(u, np.float32))
        rows = np.full((R, self.stride), np.inf, np.float32)  # what lies between rows is never looked at
        rows[:, :V] = self.logits
        dev = lambda x: None if x is None else qk.DeviceBuffer.from_array(x)  # noqa: E731
        self.x, self.params = dev(rows), [dev(x) for x in (self.heat, self.k, self.p, self.min_p, self.u)]
        self.token, self.share = qk.DeviceBuffer(4 * R), qk.DeviceBuffer(4 * R)
        n = qk.sample_workspace_size(R, V)
        self.ws = qk.DeviceBuffer.from_array(np.zeros(max(n, 256), np.uint8))

    def call(self, stream=None):
        R, V = self.logits.shape
        h, k, p, m, u = self.params
        self.qk.sample(self.x, R, V, self.stride, h, k, p, m, u, self.token, self.share, self.ws, self.ws.nbytes, stream)

    def check(self):
        token, share = self.token.download(np.uint32), self.share.download(np.float32)
        for r in range(self.logits.shape[0]):
            at = lambda x, none: none if x is None else x[r]  # noqa: E731
            want = ref.sample(self.logits[r], self.heat[r], at(self.k, 0), at(self.p, 1.0), at(self.min_p, 0.0), self.u[r])
            assert int(token[r]) == want[0], (r, int(token[r]), want)
            assert abs(share[r] - want[1]) <= 2.0 ** -24 * want[1] + 2.0 ** -30, (r, share[r], want)

    def run(self):
        self.call()
        self.qk.synchronize()
        self.check()


def _logits(rng, R, V, size=2.5):
    x = rng.standard_normal((R, V)).astype(np.float32) * np.float32(size)
    for r in range(R):
        x[r, rng.integers(0, V, 8)] += 8
    return x


@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 1000, 4097, 32003, 151936])
@pytest.mark.parametrize("R", [1, 9])
def test_filters_together_and_alone(gpu, R, V):
    rng = np.random.default_rng(V + R)
    x = _logits(rng, R, V)
    for name, more in {"none": {}, "k": dict(k=20), "p": dict(p=0.9), "min_p": dict(min_p=0.05),
                       "k1": dict(k=1), "p0": dict(p=0.0), "k+p": dict(k=40, p=0.95),
                       "all": dict(k=300, p=0.99, min_p=0.001), "off": dict(k=-1, p=1.0, min_p=0.0),
                       "k=V": dict(k=V), "wide-k": dict(k=2 * V + 5, p=0.7)}.items():
        for heat in (0.7, 1.0, 3.0):
            print(f"[case] sample R={R} V={V} {name} T={heat}", flush=True)
            Sample(gpu, x, heat, u=rng.random(R), stride=V + 3, **more).run()


def test_every_row_has_its_own_parameters(gpu):
    rng = np.random.default_rng(2)
    R, V = 64, 5003
    Sample(gpu, _logits(rng, R, V), rng.choice([0.0, 0.2, 0.8, 1.0, 2.0], R), rng.choice([0, 1, 5, 50, 6000], R),
           rng.choice([0.1, 0.5, 0.9, 1.0], R), rng.choice([0.0, 0.02, 0.5], R), rng.random(R)).run()


def test_many_rows(gpu):
    rng = np.random.default_rng(3)
    R, V = 700, 2000
    Sample(gpu, _logits(rng, R, V), 0.9, 30, 0.9, 0.0, rng.random(R)).run()


@pytest.mark.parametrize("V", [64, 5000, 40000])
def test_equal_logits_rank_by_index(gpu, V):
    """Rows of few distinct values: top-k and top-p cut inside a run of equals."""
    rng = np.random.default_rng(4)
    x = rng.choice(np.float32([0.0, -0.0, 0.5, 1.0, -3.0]), (6, V))
    x[4] = 1.25
    x[5, ::2] = -np.inf
    # uniforms away from the borders of equal weights
    for k, p in ((7, 1.0), (V // 2, 1.0), (0, 0.31), (V // 3, 0.77), (0, 1.0)):
        for u in (0.0, 0.123457, 0.7654321, 0.99999):
            Sample(gpu, x, 1.0, k, p, 0.0, u).run()


def test_large_batches_of_equal_logits(gpu):
    """Chunks whose logits all weigh 1, and rows of few distinct ones, in the layout of large batches."""
    rng = np.random.default_rng(11)
    x = np.full((110, 40001), 0.75, np.float32)
    x[1::2] = rng.choice(np.float32([0.5, 0.25, -1.0]), (55, 40001))
    x[::7, ::3] = -np.inf
    for k, p, min_p in ((0, 1.0, 0.0), (0, 0.63, 0.0), (0, 1.0, 0.9), (3000, 0.71, 0.0)):
        print(f"[case] sample equal logits k={k} p={p}", flush=True)
        Sample(gpu, x, 1.0, k, p, min_p, 0.123 + 0.8 * rng.random(110)).run()


def test_one_workspace_serves_batches_of_all_sizes(gpu):
    """Flat and peaked rows, few and many, in turn on the same bytes, zero-filled once."""
    rng = np.random.default_rng(12)
    calls = [Sample(gpu, _logits(rng, R, V), heat, k, p, 0.0, rng.random(R))
             for R, V, heat, k, p in ((1, 151936, 1.4, 0, 0.9), (130, 9000, 1.2, 0, 0.95), (3, 40000, 1.0, 0, 0.8),
                                      (2, 151936, 0.6, 20, 0.95), (60, 33000, 2.0, 0, 0.97))]
    ws = gpu.DeviceBuffer.from_array(np.zeros(max(s.ws.nbytes for s in calls), np.uint8))
    for s in calls:
        s.ws = ws
    for s in calls + calls[::-1]:
        s.token.fill(0xA5)
        s.run()


@pytest.mark.parametrize("V", [1182, 2054, 11647, 40000, 151936])
def test_kept_sets_of_hundreds(gpu, V):
    """Borders among more listed logits than are ranked one against another,
    at temperatures from low ones, where the k-th lies far below the maximum."""
    rng = np.random.default_rng(V)
    x = _logits(rng, 6, V)
    for k in (0, 100, 129, 360, 1000, 2047):
        for p, min_p, heat in ((1.0, 0.0, 0.8), (0.95, 0.0, 1.4), (0.3, 0.001, 1.0), (0.999, 0.01, 0.2)):
            print(f"[case] sample hundreds V={V} k={k} p={p} T={heat}", flush=True)
            Sample(gpu, x, heat, k, p, min_p, rng.random(6)).run()


@pytest.mark.parametrize("V", [5003, 40000, 151936])
def test_kept_sets_of_thousands(gpu, V):
    """More than the draw ranks at once; rows without a border; nearly flat rows."""
    rng = np.random.default_rng(V + 1)
    x = _logits(rng, 5, V)
    x[3] = np.float32(0.02) * rng.standard_normal(V).astype(np.float32)
    x[4] = np.round(x[4])
    for k in (0, 2500, 4999):
        for p, min_p, heat in ((1.0, 0.0, 1.0), (0.95, 0.0, 1.5), (0.6, 0.001, 0.9)):
            print(f"[case] sample thousands V={V} k={k} p={p} T={heat}", flush=True)
            Sample(gpu, x, heat, k, p, min_p, rng.random(5), stride=V + 1).run()


def test_neighbours_and_equal_logits_among_hundreds(gpu):
    """Kept tokens next to one another, and of one value: all in one part of the
    indices or of the keys."""
    rng = np.random.default_rng(12)
    V, R = 151936, 12
    x = rng.standard_normal((R, V)).astype(np.float32) - 4
    x[:, 1000:1300] = 6 + rng.random((R, 300)).astype(np.float32)
    x[4:8, rng.integers(0, V, 400)] = 8.25
    x[8:, 1000:1300] = 6 + (np.arange(300) // 150).astype(np.float32)
    for k, p in ((250, 1.0), (299, 0.9), (320, 0.6), (700, 0.95), (0, 0.9)):
        Sample(gpu, x, 0.7, k, p, 0.0, rng.random(R)).run()


def test_the_whole_line_of_uniforms(gpu):
    """Uniforms over [0, 1) draw every kept token, in index order."""
    V, R = 130, 400
    x = np.tile(np.random.default_rng(5).standard_normal(V).astype(np.float32), (R, 1))
    s = Sample(gpu, x, 1.0, 11, 1.0, 0.0, (np.arange(R) + 0.37) / R)
    s.run()
    token = s.token.download(np.uint32)
    assert (np.diff(token.astype(np.int64)) >= 0).all() and len(set(token.tolist())) == 11


def test_infinities_and_nan(gpu):
    rng = np.random.default_rng(6)
    x = _logits(rng, 7, 3000)
    x[0] = np.nan
    x[1] = -np.inf
    x[2, ::3] = np.nan
    x[3, 100:] = -np.inf
    x[4, [5, 77, 2999]] = np.inf
    x[5] = np.finfo(np.float32).min
    x[6] = np.float32(3e38)
    x[6, ::2] = np.float32(-3e38)
    for k, p in ((0, 1.0), (50, 0.9), (2, 1.0), (500, 1.0)):
        for heat in (0.0, 1e-30, 0.5, 1e30):
            Sample(gpu, x, heat, k, p, 0.01, rng.random(7)).run()


def test_bounds_of_parameters(gpu):
    """uniform at and beyond 1, and NaN parameters, still give a kept token."""
    x = _logits(np.random.default_rng(7), 6, 900)
    s = Sample(gpu, x, [1, 1, 1, np.nan, 1, -1], 10, [0.9, 0.9, np.nan, 0.9, 0.9, 0.9], 0.0, [1.0, 7.0, 0.5, 0.5, np.nan, 0.5])
    s.call()
    gpu.synchronize()
    token = s.token.download(np.uint32)
    for r in range(6):
        assert token[r] in np.argsort(-x[r], kind="stable")[:10]
    assert token[3] == x[3].argmax() and token[5] == x[5].argmax()


def test_captured_replays_and_another_stream(gpu):
    rng = np.random.default_rng(8)
    for R, V in ((1, 151936), (3, 9001), (40, 3001)):
        s = Sample(gpu, _logits(rng, R, V), 0.8, 40, 0.95, 0.0, rng.random(R))
        stream = gpu.Stream()
        graph = gpu.Graph.capture(stream, lambda: s.call(stream))
        for step in range(4):
            print(f"[case] sample graph R={R} V={V} replay {step}", flush=True)
            s.logits = _logits(rng, R, V)
            s.x.upload(s.logits)
            s.u = rng.random(R).astype(np.float32)
            s.params[4].upload(s.u)
            graph.launch(stream)
            stream.synchronize()
            s.check()
            s.run()
        graph.destroy()
        stream.destroy()
