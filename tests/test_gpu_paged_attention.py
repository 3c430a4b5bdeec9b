"""qk_paged_attention against the definition in 64 bits.

Tolerances: u = 2^-24. A score is a sum of D products in fp32 of parts that
hold q to 2 u; a blocked sum of that length is off by at most D/4 u of
sum |q k|: d = (D/4 + 4) u reach, plus 2 u of the largest |score| for the
scaling and the exponential's argument and 4 u for the exponential. A weight
is so off by e = d + 2 u reach + 4 u relatively, the result by 2 e (weights
and their sum) and the sums' own (64 + sqrt(keys)) u, all of sum p|v|. 16-bit q
adds half a step of the type for the rounded weights, twice (they meet V, and
their sum need not be theirs), and half a step of the result."""
from __future__ import annotations

import math

import numpy as np
import pytest

import serving_ref as ref
from serving_ref import BF16, F16, F32, Paged

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Attend:
    def __init__(self, qk, p: Paged, q_heads, *, q_type=F32, window=0, scale=None, lse=True, pad=0, max_context=None,
                 q_size=1.5):
        self.qk, self.p, self.q_heads, self.q_type, self.window = qk, p, q_heads, q_type, window
        D, T = p.dim, p.tokens
        self.scale = np.float32(D ** -0.5 if scale is None else scale)
        self.stride = q_heads * D + pad
        self.q = ref.encode(p.rng.standard_normal((T, self.stride)) * q_size, q_type)
        p.upload(qk)
        self.qd = qk.DeviceBuffer.from_array(self.q)
        self.out = qk.DeviceBuffer.from_array(np.full(T * q_heads * D, 0xA5A5A5A5 if q_type == F32 else 0xA5A5,
                                                      np.uint32 if q_type == F32 else np.uint16))
        self.lse = qk.DeviceBuffer.from_array(np.full(T * q_heads, 12345.0, np.float32)) if lse else None
        self.max_context = max(p.contexts, default=0) if max_context is None else max_context
        n = qk.paged_attention_workspace_size(p.cache, p.batch, q_type, q_heads, window, self.max_context)
        self.ws = qk.DeviceBuffer.from_array(np.zeros(max(n, 256), np.uint8))

    def call(self, stream=None):
        self.qk.paged_attention(self.p.cache, self.p.batch, self.qd, self.q_type, self.stride, self.q_heads, self.scale,
                                self.window, self.max_context, self.out, self.lse, self.ws, self.ws.nbytes, stream)

    def results(self):
        T, H, D = self.p.tokens, self.q_heads, self.p.dim
        out = self.out.download(np.uint32 if self.q_type == F32 else np.uint16).reshape(T, H, D)
        return out, self.lse.download(np.float32).reshape(T, H) if self.lse else None

    def check(self, sequences=None):
        p, H, D = self.p, self.q_heads, self.p.dim
        bits, lse = self.results()
        got = ref.decode(bits, self.q_type)
        owned = np.zeros(p.tokens, bool)
        step = 0.0 if self.q_type == F32 else ref.HALF_STEP[self.q_type]
        for s, (n, c) in enumerate(zip(p.new, p.contexts)):
            rows = slice(p.start[s], p.start[s] + n)
            owned[rows] = True
            if n == 0 or (sequences is not None and s not in sequences):
                continue
            q = ref.decode(self.q[rows, :H * D].reshape(n, H, D), self.q_type)
            K, V = (ref.decode(p.rows(s, pool), p.kind) for pool in (p.k, p.v))
            out, want_lse, weight, reach = ref.attention(q, K, V, c - n, float(self.scale), self.window)
            e = ((D / 4 + 6) * reach + 4) * U
            off = (2 * e + (64 + math.sqrt(max(c, 1))) * U + 2 * step)[..., None] * weight
            off = off + step * (np.abs(out) + off) + (ref.TINY[self.q_type] if step else 0)
            err = np.abs(got[rows] - out)
            assert (err <= off).all(), (s, np.nanmax(np.where(off > 0, err / np.where(off > 0, off, 1), err * np.inf)))
            if lse is not None:
                none = np.isneginf(want_lse)
                assert np.array_equal(np.isneginf(lse[rows]), none)
                err = np.abs(np.where(none, 0, lse[rows] - want_lse))
                top = np.where(none, 0, np.abs(want_lse))
                assert (err <= 2 * e + (64 + math.sqrt(max(c, 1))) * U + 4 * U * top).all(), s
        assert (bits[~owned] == (0xA5A5A5A5 if self.q_type == F32 else 0xA5A5)).all(), "rows of no sequence"
        if lse is not None:
            assert (lse[~owned] == 12345.0).all()
        assert p.fault() == 0


TYPES = {"f16-f32": (F16, F32), "f16-f16": (F16, F16), "bf16-f32": (BF16, F32), "bf16-bf16": (BF16, BF16)}
CASES = {
    "one-key": dict(new=[1], contexts=[1], q_heads=2),
    "decode": dict(new=[1] * 5, contexts=[1, 15, 16, 17, 200], q_heads=8),
    "decode-long": dict(new=[1, 1], contexts=[3000, 1025], q_heads=8, page=64),
    "drafts": dict(new=[3, 4, 2], contexts=[3, 70, 130], q_heads=8, page=24),
    "ragged": dict(new=[1, 37, 0, 130, 1], contexts=[300, 37, 50, 140, 1], q_heads=4),
    "chunk": dict(new=[150], contexts=[410], q_heads=4, page=7),
    "odd-group": dict(new=[9, 1], contexts=[30, 333], q_heads=14, kv_heads=2),
    "no-group": dict(new=[20, 1], contexts=[31, 90], q_heads=3, kv_heads=3),
    "wide-group": dict(new=[2, 1], contexts=[33, 65], q_heads=40, kv_heads=1),
    "page-1": dict(new=[5], contexts=[77], q_heads=2, page=1),
    "page-256": dict(new=[70, 1], contexts=[300, 257], q_heads=2, page=256),
    "padding-rows": dict(new=[2, 0, 40], contexts=[9, 3, 45], q_heads=4, gaps=(3, 5)),
    "empty-context": dict(new=[0, 2, 0], contexts=[0, 2, 0], q_heads=2),
}


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("name", CASES)
def test_attention_matches_its_definition(gpu, name, types):
    kind, q_type = TYPES[types]
    case = dict(CASES[name])
    q_heads = case.pop("q_heads")
    for dim, head_major in ((128, False), (64, True)):
        print(f"[case] attention {name} {types} dim={dim}", flush=True)
        p = Paged(kind=kind, dim=dim, head_major=head_major, seed=len(name) + dim, **case)
        a = Attend(gpu, p, q_heads, q_type=q_type, pad=8)
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("types", ["f16-f32", "bf16-bf16"])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 5000])
def test_sliding_window(gpu, window, types):
    """Pages wholly before every window may be gone: their table entries are no pages."""
    kind, q_type = TYPES[types]
    p = Paged([1, 90, 3], [400, 300, 3], kind=kind, dim=128, seed=window)
    for s, (n, c) in enumerate(zip(p.new, p.contexts)):
        gone = max(0, c - n - window + 1) // p.page
        K, V = p.seen(p.k), p.seen(p.v)
        for e in range(gone):  # the reference still reads the rows; it masks them
            K[p.table[s, e]], V[p.table[s, e]] = ref.encode(np.nan, kind), ref.encode(np.nan, kind)
    a = Attend(gpu, p, 4, q_type=q_type, window=window)
    spoiled = p.table.copy()
    for s, (n, c) in enumerate(zip(p.new, p.contexts)):
        spoiled[s, :max(0, c - n - window + 1) // p.page] = -1
    p.dev["table"].upload(spoiled)
    a.call()
    gpu.synchronize()
    a.check()


@pytest.mark.parametrize("types", TYPES)
def test_masked_places_may_hold_anything(gpu, types):
    """NaN and infinities in unused slots, unused pages and at positions after
    a row: rows that do not see them are what they were."""
    kind, q_type = TYPES[types]
    for new, contexts in (([1, 1], [50, 131]), ([40, 3], [60, 35]), ([200], [200])):
        p = Paged(new, contexts, kind=kind, dim=128, seed=sum(new))
        used = np.zeros((p.pages, p.page), bool)
        for s, c in enumerate(p.contexts):
            pos = np.arange(c)
            used[p.table[s, pos // p.page], pos % p.page] = True
        for pool, value in ((p.k, np.nan), (p.v, np.inf)):
            p.seen(pool)[~used] = ref.encode(value, kind)
        a = Attend(gpu, p, 4, q_type=q_type)
        a.call()
        gpu.synchronize()
        a.check()
    # the last token's own key and value are not finite: rows before it do not see them
    for value in (np.nan, np.inf, -np.inf):
        p = Paged([40], [60], kind=kind, dim=128, seed=3)
        K, V = p.seen(p.k), p.seen(p.v)
        K[p.table[0, 59 // 16], 59 % 16, :, 3] = ref.encode(value, kind)
        V[p.table[0, 59 // 16], 59 % 16, :, 5] = ref.encode(value, kind)
        a = Attend(gpu, p, 4, q_type=q_type)
        a.call()
        gpu.synchronize()
        bits, _ = a.results()
        before = ref.decode(bits, q_type)[:39]
        assert np.isfinite(before).all()
        with np.errstate(invalid="ignore"):
            K64, V64 = (ref.decode(p.rows(0, pool), kind)[:59] for pool in (p.k, p.v))
        q = ref.decode(a.q[:39].reshape(39, 4, 128), q_type)
        want = ref.attention(q, K64, V64, 20, float(a.scale), 0)[0]
        assert np.abs(before - want).max() <= (1e-4 if q_type == F32 else 8 * ref.HALF_STEP[q_type])


@pytest.mark.parametrize("types", TYPES)
def test_a_value_that_is_infinite_reaches_only_the_rows_that_see_it(gpu, types):
    """+inf in one value of one position: +inf in that column from there on."""
    kind, q_type = TYPES[types]
    p = Paged([30], [30], kind=kind, dim=64, seed=4)
    p.seen(p.v)[p.table[0, 0], 10, :, 7] = ref.encode(np.inf, kind)
    a = Attend(gpu, p, 2, q_type=q_type)
    a.call()
    gpu.synchronize()
    out = ref.decode(a.results()[0], q_type)
    assert np.isfinite(out[:10]).all() and np.isfinite(np.delete(out, 7, axis=2)).all()
    assert (out[10:, :, 7] == np.inf).all()


def test_rows_that_see_nothing_are_zero(gpu):
    """A context shorter than its new tokens: the first of them have no
    position, see nothing, and the misfit is reported."""
    for q_type in (F32, F16):
        p = Paged([5, 2], [2, 40], seed=8)
        a = Attend(gpu, p, 4, q_type=q_type)
        a.call()
        gpu.synchronize()
        bits, lse = a.results()
        assert (bits[:3] == 0).all() and np.isneginf(lse[:3]).all()
        assert p.fault() == gpu.KV_FAULT_LENGTH
        with pytest.raises(gpu.QKError):
            gpu.kv_check(p.cache)
        a.check()


def test_large_scores_do_not_overflow(gpu):
    for types in TYPES:
        kind, q_type = TYPES[types]
        p = Paged([3, 1], [90, 300], kind=kind, dim=128, seed=13)
        p.k = ref.encode(ref.decode(p.k, kind) * 30, kind)
        a = Attend(gpu, p, 4, q_type=q_type, q_size=100.0, scale=1.0)
        a.call()
        gpu.synchronize()
        out, lse = a.results()
        assert np.isfinite(ref.decode(out, q_type)).all() and np.isfinite(lse).all()
        q = ref.decode(a.q[:3].reshape(3, 4, 128), q_type)
        K, V = (ref.decode(p.rows(0, pool), kind) for pool in (p.k, p.v))
        want = ref.attention(q, K, V, 87, 1.0, 0)
        assert np.abs(lse[:3] / want[1] - 1).max() <= 1e-5


def test_q_of_any_size_keeps_its_precision(gpu):
    """fp32 queries far outside fp16's range, their scale the inverse."""
    for size in (1e-12, 1e9):
        p = Paged([2, 1], [40, 77], dim=64, seed=14)
        a = Attend(gpu, p, 4, q_size=size, scale=0.1 / size)
        a.call()
        gpu.synchronize()
        a.check()


def test_max_context_is_only_a_bound_for_the_split(gpu):
    p = Paged([1, 2], [2500, 1700], dim=128, kv_heads=2, seed=15)
    for bound in (0, 1, 100, 2500, 1 << 20):
        a = Attend(gpu, p, 8, max_context=bound)
        a.call()
        a.call()  # the workspace is ready again
        gpu.synchronize()
        a.check()


def test_one_workspace_serves_batches_of_all_sizes(gpu):
    """Batches of few and many tiles in turn on the same bytes, zero-filled once."""
    calls = []
    for i, (new, context, q_type) in enumerate((([1], [3000], F32), ([1] * 40, [700] * 40, F16), ([150], [1800], F32),
                                                ([1] * 9, [1500] * 9, F32), ([300, 290], [2000, 1000], F16))):
        calls.append(Attend(gpu, Paged(new, context, dim=128, kv_heads=2, seed=30 + i), 8, q_type=q_type))
    ws = gpu.DeviceBuffer.from_array(np.zeros(max(a.ws.nbytes for a in calls), np.uint8))
    for a in calls:
        a.ws = ws
    for a in calls + calls[::-1]:
        a.out.fill(0x5A)
        a.call()
        gpu.synchronize()
        a.check()


# Layouts that large calls take, at sizes that can be checked: the bound on the
# context and the number of heads decide on tiles and parts.
LAYOUTS = {"wide": dict(max_context=4000), "wide-whole": dict(max_context=2100, kv_heads=96),
           "pairs": dict(max_context=400, kv_heads=80)}


def _layout(name, new, contexts, seed, **more):
    """A batch in that layout: group 1 where it takes many heads, else 4."""
    layout = dict(LAYOUTS[name])
    bound = layout.pop("max_context")
    heads = layout.pop("kv_heads", 2)
    q_heads = heads if heads > 2 else 8
    return Paged(new, contexts, kv_heads=heads, seed=seed, **more), q_heads, bound


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dim", [64, 128])
def test_layouts_of_large_calls(gpu, layout, types, dim):
    kind, q_type = TYPES[types]
    for new, contexts, window in (([100, 33, 0, 1], [700, 40, 9, 300], 0), ([90, 60], [400, 130], 70)):
        print(f"[case] attention {layout} {types} dim={dim} window={window}", flush=True)
        p, q_heads, bound = _layout(layout, new, contexts, dim, kind=kind, dim=dim, page=24, gaps=(1, 2))
        a = Attend(gpu, p, q_heads, q_type=q_type, max_context=bound, window=window)
        a.call()
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_masked_places_in_layouts_of_large_calls(gpu, layout, types):
    """NaN and infinities in unused slots, in later positions and in one value that some rows see."""
    kind, q_type = TYPES[types]
    p, q_heads, bound = _layout(layout, [120, 80], [120, 333], 5, kind=kind, dim=64)
    used = np.zeros((p.pages, p.page), bool)
    for s, c in enumerate(p.contexts):
        used[p.table[s, np.arange(c) // p.page], np.arange(c) % p.page] = True
    for pool, value in ((p.k, np.nan), (p.v, np.inf)):
        p.seen(pool)[~used] = ref.encode(value, kind)
    a = Attend(gpu, p, q_heads, q_type=q_type, max_context=bound)
    a.call()
    gpu.synchronize()
    a.check()
    p.seen(p.v)[p.table[0, 3], 2, :, 7] = ref.encode(np.inf, kind)  # position 50
    p.seen(p.k)[p.table[0, 119 // 16], 119 % 16, :, 3] = ref.encode(np.nan, kind)
    p.dev["k"].upload(p.k)
    p.dev["v"].upload(p.v)
    a.call()
    gpu.synchronize()
    out = ref.decode(a.results()[0], q_type)[:119]
    assert np.isfinite(out[:50]).all() and np.isfinite(np.delete(out, 7, axis=2)).all()
    assert (out[50:, :, 7] == np.inf).all()
    a.check(sequences=(1,))


@pytest.mark.parametrize("types", TYPES)
def test_scales_of_either_sign_and_zero(gpu, types):
    kind, q_type = TYPES[types]
    for new, contexts, bound in (([1, 2], [300, 70], 300), ([70], [130], 130), ([70], [130], 4000)):
        for scale in (-0.11, 0.0):
            p = Paged(new, contexts, kind=kind, dim=64, seed=6)
            a = Attend(gpu, p, 4, q_type=q_type, scale=scale, max_context=bound)
            a.call()
            gpu.synchronize()
            a.check()


# Between them every size of tile (256, 128 or 64 rows; 128, 64 or 32 with F32 q
# over BF16), with its keys whole and in parts, in each pair of types.
TILES = {
    "few-keys": dict(new=[100], contexts=[180], kv_heads=1, group=4, bound=200),
    "parts": dict(new=[100], contexts=[700], kv_heads=1, group=4, bound=1000),
    "long-bound": dict(new=[100], contexts=[500], kv_heads=1, group=4, bound=6000),
    "longer-bound": dict(new=[190], contexts=[600], kv_heads=2, group=4, bound=8000),
    "heads": dict(new=[150], contexts=[300], kv_heads=96, group=1, bound=700),
    "heads-parts": dict(new=[150], contexts=[600], kv_heads=40, group=1, bound=6000),
    "two-prompts": dict(new=[170, 130], contexts=[200, 150], kv_heads=96, group=1, bound=700),
    "more-heads": dict(new=[300], contexts=[330], kv_heads=128, group=1, bound=1000),
}


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("name", TILES)
@pytest.mark.parametrize("dim", [64, 128])
def test_tiles_and_parts(gpu, name, types, dim):
    kind, q_type = TYPES[types]
    case = TILES[name]
    print(f"[case] attention tiles {name} {types} dim={dim}", flush=True)
    p = Paged(case["new"], case["contexts"], kv_heads=case["kv_heads"], kind=kind, dim=dim, seed=dim + len(name))
    used = np.zeros((p.pages, p.page), bool)
    for s, c in enumerate(p.contexts):
        used[p.table[s, np.arange(c) // p.page], np.arange(c) % p.page] = True
    for pool, value in ((p.k, np.inf), (p.v, np.nan)):
        p.seen(pool)[~used] = ref.encode(value, kind)
    a = Attend(gpu, p, case["kv_heads"] * case["group"], q_type=q_type, max_context=case["bound"])
    a.call()
    a.call()
    gpu.synchronize()
    a.check()


# Few rows over many keys: 4, 7, 8, 12 and 16 rows of a tile, two to five tiles, from
# nine parts to more than a hundred.
MANY_PARTS = {
    "four-rows": dict(new=[1], contexts=[5000], kv_heads=2, group=4),
    "seven-rows": dict(new=[1, 1], contexts=[3000, 1300], kv_heads=2, group=7),
    "eight-rows": dict(new=[1, 2], contexts=[2500, 2050], kv_heads=2, group=8),
    "twelve-rows": dict(new=[3], contexts=[9000], kv_heads=1, group=4),
    "sixteen-rows": dict(new=[4, 4, 1], contexts=[3000, 40, 1500], kv_heads=2, group=4),
    "tiles": dict(new=[16, 5], contexts=[2600, 700], kv_heads=2, group=4),
    "uneven-tiles": dict(new=[17, 9, 0, 1], contexts=[4500, 130, 0, 2200], kv_heads=2, group=4),
    "hundred-parts": dict(new=[1], contexts=[20000], kv_heads=1, group=3),
}


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("name", MANY_PARTS)
def test_few_rows_in_many_parts(gpu, name, types):
    kind, q_type = TYPES[types]
    case = MANY_PARTS[name]
    for dim in (64, 128):
        print(f"[case] attention parts {name} {types} dim={dim}", flush=True)
        p = Paged(case["new"], case["contexts"], kv_heads=case["kv_heads"], kind=kind, dim=dim, page=64, seed=dim + 1)
        a = Attend(gpu, p, case["kv_heads"] * case["group"], q_type=q_type)
        a.call()
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("types", ["f16-f32", "bf16-bf16"])
def test_batches_of_several_tiles_in_parts(gpu, types):
    """More (tile, head) units than compute units, too many tiles a sequence to take contexts by length."""
    kind, q_type = TYPES[types]
    rng = np.random.default_rng(33)
    new = [int(n) for n in rng.integers(1, 11, 20)]
    contexts = [int(c) + n for c, n in zip(rng.integers(1, 500, 20), new)]
    contexts[3], contexts[11] = 4400, 2300
    p = Paged(new, contexts, kv_heads=6, kind=kind, dim=64, seed=34, gaps=(1, 2))
    for window in (0, 2500):
        a = Attend(gpu, p, 24, q_type=q_type, window=window)
        a.call()
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("types", ["f16-f32", "bf16-bf16"])
@pytest.mark.parametrize("case", ["singles", "drafts", "window", "misfit"])
def test_batches_that_are_taken_by_length(gpu, case, types):
    """Many sequences of uneven contexts, some without a new token; drafts of
    two tiles (then in their own order); a context shorter than its new tokens."""
    kind, q_type = TYPES[types]
    rng = np.random.default_rng(21)
    new = [0 if i % 9 == 4 else 1 for i in range(70)]
    contexts = [int(c) for c in rng.integers(1, 260, 70)]
    contexts[5] = contexts[33] = 1300  # equal lengths rank by their order
    q_heads = 8
    if case == "drafts":
        new = [3 * n for n in new]
        new[2], q_heads = 9, 8  # 18 rows: two tiles
    contexts = [max(c, n) for c, n in zip(contexts, new)]
    if case == "misfit":
        new[7], contexts[7] = 2, 1
    p = Paged(new, contexts, kv_heads=4, dim=64, kind=kind, seed=22, gaps=(2, 1))
    a = Attend(gpu, p, q_heads, q_type=q_type, window=90 if case == "window" else 0, max_context=1300)
    print(f"[case] attention by length {case} {types}", flush=True)
    a.call()
    gpu.synchronize()
    if case == "misfit":
        assert p.fault() == gpu.KV_FAULT_LENGTH
        p.dev["fault"].upload(np.zeros(1, np.uint32))
    a.check()


def test_bad_pages_are_reported_and_reach_no_other_sequence(gpu):
    for new, contexts in (([1, 1, 1], [40, 40, 40]), ([30, 30, 30], [40, 40, 40])):
        p = Paged(new, contexts, page=8, dim=128, seed=16)
        p.table[1, 3] = p.pages + 5
        a = Attend(gpu, p, 4)
        a.call()
        gpu.synchronize()
        out, _ = a.results()
        last = out[p.start[2] - 1].view(np.float32)
        assert np.isnan(last).all()
        assert p.fault() == gpu.KV_FAULT_PAGE
        with pytest.raises(gpu.QKError, match="page"):
            gpu.kv_check(p.cache)
        a.check(sequences=(0, 2))


def test_another_stream_and_captured_replays(gpu):
    """A captured step over lengths that change between replays, eager calls and
    synchronizations between them: every replay is the eager result, bit for bit."""
    p = Paged([1, 1, 1], [600, 40, 1300], dim=128, kv_heads=2, spare=4, seed=17)
    a = Attend(gpu, p, 8, max_context=1300)
    stream = gpu.Stream()
    graph = gpu.Graph.capture(stream, lambda: a.call(stream))
    for step, contexts in enumerate(([600, 40, 1300], [601, 41, 1], [17, 33, 1299], [600, 40, 1300])):
        print(f"[case] attention graph replay {step}", flush=True)
        p.contexts = list(contexts)
        p.dev["context"].upload(np.asarray(contexts, np.int32))
        graph.launch(stream)
        stream.synchronize()
        replay = [x.copy() for x in a.results()]
        a.check()
        a.out.fill(0x5A)
        a.call()
        gpu.synchronize()
        assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(replay, a.results()))
    graph.destroy()
    stream.destroy()


def test_a_page_far_into_a_large_pool(gpu):
    """Offsets past 2^32 bytes: a pool of 4.5 GB, pages at its end."""
    P, H, D = 64, 8, 128
    pages = (9 << 28) // (P * H * D * 2) + 3
    p = Paged([2], [130], kv_heads=H, dim=D, page=P, seed=18)
    big = {n: gpu.DeviceBuffer(pages * P * H * D * 2) for n in "kv"}
    a = Attend(gpu, p, 16)
    far = np.array([[pages - 1, pages - 3, pages - 2]], np.int32)
    for n, pool in (("k", p.k), ("v", p.v)):
        for e in range(3):
            big[n].upload(pool[p.table[0, e]], offset=int(far[0, e]) * P * H * D * 2)
    p.dev["table"].upload(far)
    p.cache.k, p.cache.v, p.cache.pages = big["k"].ptr, big["v"].ptr, pages
    a.call()
    gpu.synchronize()
    a.check()
    for b in big.values():
        b.free()


@pytest.mark.parametrize("length", [0x7FFFFFFF, 1500000000, (1 << 30) + 1000, 5 * 8 + 1])
def test_a_context_beyond_its_page_table_is_reported(gpu, length):
    """No key of it is walked: its rows are NaN, the others what they are."""
    for new, contexts, bound in (([1, 1, 1], [40, 40, 40], 40), ([1, 2, 1], [40, 40, 40], 1 << 20),
                                 ([30, 30, 30], [40, 40, 40], 40), ([90, 30, 30], [90, 40, 40], 1 << 20)):
        print(f"[case] attention context {length} new={new} bound={bound}", flush=True)
        p = Paged(new, contexts, page=8, dim=128, seed=23)
        if max(contexts) > 40:
            length = max(length, 12 * 8 + 1)
        a = Attend(gpu, p, 4, max_context=bound)
        lengths = np.asarray(contexts, np.int32)
        lengths[1] = length
        p.dev["context"].upload(lengths)
        for window in (0, 7):
            a.window = window
            a.call()
            gpu.synchronize()
            out, lse = a.results()
            rows = slice(p.start[1], p.start[2])
            assert np.isnan(out[rows].view(np.float32)).all() and np.isnan(lse[rows]).all()
            assert p.fault() == gpu.KV_FAULT_PAGE
            with pytest.raises(gpu.QKError, match="page"):
                gpu.kv_check(p.cache)
            a.check(sequences=(0, 2))


def test_a_context_beyond_its_page_table_among_many(gpu):
    """Sequences taken by length."""
    rng = np.random.default_rng(24)
    contexts = [int(c) for c in rng.integers(1, 260, 70)]
    contexts[5] = 1300
    p = Paged([1] * 70, contexts, kv_heads=4, dim=64, seed=25)
    a = Attend(gpu, p, 8, max_context=1300)
    lengths = np.asarray(contexts, np.int32)
    lengths[9] = 0x7FFFFFFF
    p.dev["context"].upload(lengths)
    a.call()
    gpu.synchronize()
    assert np.isnan(a.results()[0][9].view(np.float32)).all()
    assert p.fault() == gpu.KV_FAULT_PAGE
    p.dev["fault"].upload(np.zeros(1, np.uint32))
    a.check(sequences=[s for s in range(70) if s != 9])


def _misfits(layout):
    """(sequence, new, contexts, contexts with a negative one there) of batches in that layout."""
    if layout == "long":
        new, contexts = [90, 30, 30], [300, 200, 31]
    elif layout == "by-length":
        new, contexts = [1] * 70, [20 + 3 * i for i in range(69)] + [1300]
    else:
        new, contexts = [1, 2, 1], [40, 300, 7]
    last = len(new) - 1
    for s in (0, last // 2, last):
        yield s, new, contexts, np.asarray(contexts[:s] + [-1 - s] + contexts[s + 1:], np.int32)
        yield s, new, contexts, np.asarray(contexts[:s] + [-(1 << 31)] + contexts[s + 1:], np.int32)


@pytest.mark.parametrize("layout", ["few", "long", "by-length"])
def test_negative_contexts_see_nothing_and_are_reported(gpu, layout):
    for s, new, contexts, lengths in _misfits(layout):
        print(f"[case] attention {layout} sequence {s} context {lengths[s]}", flush=True)
        p = Paged(new, contexts, kv_heads=4, dim=64, seed=26)
        a = Attend(gpu, p, 8)
        p.dev["context"].upload(lengths)
        a.call()
        gpu.synchronize()
        bits, lse = a.results()
        rows = slice(p.start[s], p.start[s + 1])
        assert (bits[rows] == 0).all() and np.isneginf(lse[rows]).all()
        assert p.fault() == gpu.KV_FAULT_LENGTH
        with pytest.raises(gpu.QKError, match="token_start"):
            gpu.kv_check(p.cache)
        a.check(sequences=[i for i in range(len(new)) if i != s])


@pytest.mark.parametrize("layout", ["few", "long", "by-length"])
def test_starts_that_descend_or_pass_the_rows_are_reported(gpu, layout):
    """Sequences that so own no row have no tile; the word is set all the same."""
    for s, new, contexts, _ in _misfits(layout):
        for start_of in ("descends", "passes", "negative"):
            if s + (start_of != "negative") >= len(new):
                continue
            print(f"[case] attention {layout} sequence {s} {start_of}", flush=True)
            p = Paged(new, contexts, kv_heads=4, dim=64, seed=27)
            a = Attend(gpu, p, 8)
            starts = p.start.copy()
            if start_of == "descends":  # sequence s + 1 ends before it begins
                starts[s + 1:] = starts[-1]
                starts[s + 2:] = starts[s]
            elif start_of == "passes":
                starts[s + 1:] = p.tokens + 5
            else:
                starts[:s + 1] = -1
            p.dev["start"].upload(starts)
            a.call()
            gpu.synchronize()
            assert p.fault() & gpu.KV_FAULT_LENGTH
            with pytest.raises(gpu.QKError):
                gpu.kv_check(p.cache)


def test_a_last_sequence_without_rows_is_reported(gpu):
    """Only its own lengths are wrong: no row of the batch is its."""
    for new, contexts in (([1, 1, 0], [40, 300, 9]), ([90, 30, 0], [300, 200, 9]), ([1] * 70 + [0], [1300] * 71)):
        p = Paged(new, contexts, kv_heads=4, dim=64, seed=28)
        a = Attend(gpu, p, 8)
        lengths = np.asarray(contexts, np.int32)
        lengths[-1] = -5
        p.dev["context"].upload(lengths)
        a.call()
        gpu.synchronize()
        assert p.fault() == gpu.KV_FAULT_LENGTH
        p.dev["fault"].upload(np.zeros(1, np.uint32))
        a.check()


class Sinks(Attend):
    """Attend, with keys that the queries prefer by about `gaps` nats each and whose values are nothing."""

    def __init__(self, qk, p, q_heads, gaps, at, *, noise=0.12, value=0.0, **more):
        kind, D = p.kind, p.dim
        u = np.sign(p.rng.standard_normal(D)) / math.sqrt(D)
        p.k = ref.encode(ref.decode(p.k, kind) * noise, kind)
        K, V = p.seen(p.k), p.seen(p.v)
        for s, c in enumerate(p.contexts):
            for gap, pos in zip(gaps, at):
                if pos < c:
                    place = p.table[s, pos // p.page], pos % p.page
                    K[place] = ref.encode(u * (gap / 8), kind)
                    V[place] = ref.encode(ref.decode(V[place], kind) * value, kind)
        super().__init__(qk, p, q_heads, scale=1.0, q_size=1.0, **more)
        q = ref.decode(self.q, self.q_type)
        q[:, :q_heads * D] += np.tile(8 * u, q_heads)
        self.q = ref.encode(q, self.q_type)
        self.qd.upload(self.q)


# where the kernels differ: single tokens, drafts, prompts whose keys lie in one
# workgroup, in waves of it, in several workgroups
SINKS = {
    "single": dict(new=[1, 1], contexts=[300, 47], q_heads=8),
    "single-parts": dict(new=[1], contexts=[5000], q_heads=8, page=64),
    "drafts": dict(new=[4, 3], contexts=[700, 33], q_heads=8),
    "window": dict(new=[3, 90], contexts=[700, 300], q_heads=8, window=250),
    "prompt": dict(new=[150], contexts=[400], q_heads=8),
    "prompt-parts": dict(new=[100, 40], contexts=[900, 90], q_heads=8, max_context=6000),
    "prompt-wide": dict(new=[60], contexts=[330], q_heads=96, kv_heads=96, max_context=700),
    "prompt-pairs": dict(new=[60], contexts=[330], q_heads=80, kv_heads=80, max_context=400),
}


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("name", SINKS)
def test_weights_beside_much_larger_ones_keep_their_precision(gpu, name, types):
    """Keys that take nearly all of the mass and have values of nothing: the rest
    of the row, down to 2^-90 of the mass, is all of the result."""
    kind, q_type = TYPES[types]
    case = dict(SINKS[name])
    q_heads, window, bound = case.pop("q_heads"), case.pop("window", 0), case.pop("max_context", None)
    for i, (gaps, at, value) in enumerate((([10], [0], 0.0), ([14], [0], 1e-6), ([18], [0], 0.0), ([25, 12], [0, 5], 0.0),
                                           ([12, 30, 45, 20], [2, 130, 61, 64], 0.0), ([55], [33], 0.0),
                                           ([60, 38, 18], [0, 1, 2], 0.0))):
        dim = 128 if i % 2 == 0 else 64
        print(f"[case] attention sinks {name} {types} {gaps} at {at} dim={dim}", flush=True)
        p = Paged(kind=kind, dim=dim, seed=40 + i, **case)
        a = Sinks(gpu, p, q_heads, gaps, at, value=value, q_type=q_type, window=window, max_context=bound)
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("name", ["single", "drafts", "prompt", "prompt-parts"])
def test_large_weights_of_small_values_and_the_rest(gpu, name, types):
    """Values between nothing and those of the rest: what the rest adds is a part
    of the result, of any size."""
    kind, q_type = TYPES[types]
    case = dict(SINKS[name])
    q_heads, bound = case.pop("q_heads"), case.pop("max_context", None)
    for i, (gap, at, value) in enumerate(((14, 0, 0.3), (14, 40, 0.05), (14, 0, 2.0 ** -8), (25, 0, 0.05), (25, 33, 2.0 ** -10),
                                          (40, 0, 2.0 ** -14))):
        print(f"[case] attention small values {name} {types} {gap} at {at} value={value}", flush=True)
        p = Paged(kind=kind, dim=128 if i % 2 == 0 else 64, seed=70 + i, **case)
        a = Sinks(gpu, p, q_heads, [gap], [at], value=value, q_type=q_type, max_context=bound)
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("new", [1, 4, 100])
def test_scores_of_any_spread_keep_their_precision(gpu, new, types):
    """Weights over tens of powers of two in every block of keys."""
    kind, q_type = TYPES[types]
    for i, (size, bound) in enumerate(((4.0, None), (9.0, None), (9.0, 6000), (25.0, None))):
        print(f"[case] attention spread {size} {types} new={new} bound={bound}", flush=True)
        p = Paged([new], [new + 400], kind=kind, dim=128 if i % 2 == 0 else 64, seed=50 + i)
        a = Attend(gpu, p, 8, q_type=q_type, q_size=size, max_context=bound)
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("types", TYPES)
def test_an_infinite_value_of_a_tiny_weight(gpu, types):
    """Infinity times any weight is infinity, in blocks of keys that all rows see too."""
    kind, q_type = TYPES[types]
    for new, contexts, bound in (([1], [600], None), ([100], [600], None), ([100], [600], 6000)):
        for gap, at in ((0, 0), (14, 0), (20, 33), (30, 0), (35, 33)):  # 33: in the same 32 keys
            print(f"[case] attention infinite value {types} new={new} gap={gap} at {at} bound={bound}", flush=True)
            p = Paged(new, contexts, kind=kind, dim=128, seed=60)
            p.seen(p.v)[p.table[0, 40 // p.page], 40 % p.page, :, 7] = ref.encode(np.inf, kind)
            a = Sinks(gpu, p, 8, [gap], [at], q_type=q_type, max_context=bound)
            a.call()
            gpu.synchronize()
            out = ref.decode(a.results()[0], q_type)
            assert (out[:, :, 7] == np.inf).all() and np.isfinite(np.delete(out, 7, axis=2)).all()


@pytest.mark.parametrize("types", ["f16-f16", "bf16-bf16"])
@pytest.mark.parametrize("name", ["decode", "decode-long", "drafts"])
def test_single_tokens_round_once(gpu, name, types):
    """Few new tokens, 16-bit q: the result is within half a step of the type, and
    what weights of two parts (2^-16 of BF16, 2^-20 of F16) and the sums are off by."""
    kind, q_type = TYPES[types]
    case = dict(CASES[name])
    q_heads = case.pop("q_heads")
    for dim in (64, 128):
        p = Paged(kind=kind, dim=dim, seed=80 + dim, **case)
        a = Attend(gpu, p, q_heads, q_type=q_type)
        a.call()
        gpu.synchronize()
        got, step = ref.decode(a.results()[0], q_type), ref.HALF_STEP[q_type]
        for s, (n, c) in enumerate(zip(p.new, p.contexts)):
            rows = slice(p.start[s], p.start[s] + n)
            q = ref.decode(a.q[rows].reshape(n, q_heads, dim), q_type)
            K, V = (ref.decode(p.rows(s, pool), kind) for pool in (p.k, p.v))
            out, _, weight, reach = ref.attention(q, K, V, c - n, float(a.scale), 0)
            e = ((dim / 4 + 6) * reach + 4) * U + (2.0 ** -16 if kind == BF16 else 2.0 ** -20)
            off = (2 * e + (64 + math.sqrt(c)) * U)[..., None] * weight
            off = off + step * (np.abs(out) + off) + ref.TINY[q_type]
            assert (np.abs(got[rows] - out) <= off).all(), s


@pytest.mark.parametrize("types", TYPES)
def test_single_tokens_beside_a_long_chunk(gpu, types):
    """A chunk of a prompt among decode rows in one call: one kernel takes both."""
    kind, q_type = TYPES[types]
    for new, contexts, bound in (([1] * 40 + [300] + [1] * 23, [5 + 31 * i for i in range(40)] + [700] + [400] * 23, 1300),
                                 ([200] + [1] * 9, [260] + [3000] + [90] * 8, 4000)):
        print(f"[case] attention singles and a chunk {types} {len(new)} sequences", flush=True)
        p = Paged(new, contexts, kv_heads=2, kind=kind, dim=64, seed=90 + len(new))
        a = Attend(gpu, p, 8, q_type=q_type, max_context=bound)
        a.call()
        a.call()
        gpu.synchronize()
        a.check()
