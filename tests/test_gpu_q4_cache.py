"""Caches of Q4_1 blocks: what qk_kv_append writes, qk_kv_rows reads back and
qk_paged_attention makes of them, against the definitions in 64 bits.

Attention: the definition over the F16 values that the blocks stand for, with
the tolerances of an F16 cache (test_gpu_paged_attention). Keys: a stored value is
off by half a code, by half a step of m where m lies above the least value, by
what d lacks of a fifteenth of the range (an F16 step of it, 15 times), by the
rounding of the value, and by the row's own error before (24 u of the rotated
pair, test_gpu_kv_append); the codes' arithmetic in fp32 adds 3 u of 15 codes.
Values pass through no arithmetic before: their bytes are the definition's."""
from __future__ import annotations

import numpy as np
import pytest

import q4_ref
import serving_ref as ref
import test_gpu_paged_attention as f16
from q4_ref import Paged4
from serving_ref import BF16, F16, F32, Paged
from test_gpu_paged_attention import Attend

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6
Q_TYPES = {"f32": F32, "f16": F16}

APPENDS = {
    "one-token": dict(new=[1], contexts=[1], q_heads=4),
    "decode-far": dict(new=[1, 1, 1], contexts=[100001, 17, 131072], q_heads=4, page=256, kv_heads=1),
    "ragged": dict(new=[5, 1, 33, 16], contexts=[5, 40, 50, 16], q_heads=6, page=24),
    "empty-sequences": dict(new=[0, 3, 0, 0, 2, 0], contexts=[0, 3, 9, 0, 20, 4], q_heads=2),
    "padding-rows": dict(new=[2, 3], contexts=[2, 7], q_heads=2, gaps=(3, 2)),
    "odd-page": dict(new=[40], contexts=[41], q_heads=6, page=7, kv_heads=3),
    "many-heads": dict(new=[2, 1], contexts=[70, 3], q_heads=32, kv_heads=8),
}
FORMS = {"plain": dict(dim=128), "pairs-partial": dict(dim=64, interleaved=True, dims=32, base=1e4),
         "partial": dict(dim=128, dims=40), "same-head-major": dict(dim=64, q_type=F16, head_major=True),
         "no-norm": dict(dim=128, norm=False), "nothing": dict(dim=64, norm=False, dims=0)}


def append(gpu, p, q_heads, *, q_type=F32, dims=None, interleaved=False, norm=True, base=1e6, seen=None, stream=None,
           spoil=None):
    """One call; everything it went by."""
    D, H, T, rng = p.dim, p.kv_heads, p.tokens, p.rng
    dims = D if dims is None else dims
    width = (q_heads + 2 * H) * D + 3
    x = (rng.standard_normal((T, width)) * 2).astype(np.float32)
    if spoil:
        spoil(x)
    norms = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in range(2)]
    p.upload(gpu)
    xd = gpu.DeviceBuffer.from_array(x)
    nd = [gpu.DeviceBuffer.from_array(n) if norm else None for n in norms]
    q_out = gpu.DeviceBuffer.from_array(np.full(max(1, T * q_heads * D * (4 if q_type == F32 else 2)), 0xA5, np.uint8))
    rope = gpu.Rope(q_norm=nd[0].ptr if norm else None, k_norm=nd[1].ptr if norm else None, eps=EPS, base=base, dims=dims,
                    interleaved=interleaved)
    seen_d = gpu.DeviceBuffer.from_array(np.asarray(seen, np.int32)) if seen is not None else None
    k_at, v_at = q_heads * D * 4, (q_heads + H) * D * 4
    gpu.kv_append_at(p.cache, p.batch, seen_d, xd, width, xd.ptr + k_at, width, xd.ptr + v_at, width, q_heads, rope, q_out,
                     q_type, stream)
    gpu.synchronize(stream)
    return x, norms, q_out, dims, seen


def check_append(p, q_heads, made, *, q_type=F32, interleaved=False, base=1e6, **_):
    x, norms, q_out, dims, seen = made
    D, H, T = p.dim, p.kv_heads, p.tokens
    got = {n: p.downloaded(n) for n in "kv"}
    want = {"k": p.k4.copy(), "v": p.v4.copy()}
    size = np.uint32 if q_type == F32 else np.uint16
    got_q = q_out.download(size)[:T * q_heads * D].reshape(T, q_heads, D)
    owned = np.zeros(T, bool)
    for s, (n, c) in enumerate(zip(p.new, p.contexts)):
        rows = slice(p.start[s], p.start[s] + n)
        owned[rows] = True
        at = np.arange(c - n, c)
        pos = at if seen is None else at + (seen[s] - c)
        q, k, v = np.split(x[rows, :(q_heads + 2 * H) * D].reshape(n, q_heads + 2 * H, D), [q_heads, q_heads + H], 1)

        def rotated(part, weight):
            out = ref.rotate(part, pos, weight, EPS, base, dims, interleaved)
            plain = ref.rotate(part, pos, weight, EPS, base, 0, False)
            return out, 24 * U * ref.pair_size(plain, dims, interleaved)

        out, off = rotated(q, norms[0])
        off = off + ref.HALF_STEP[q_type] * (np.abs(out) + off) + ref.TINY[q_type]
        assert (np.abs(ref.decode(got_q[rows], q_type) - out) <= off).all(), ("q", s)
        out, off = rotated(k, norms[1])
        for i in range(n):
            page, slot = p.table[s, at[i] // p.page], at[i] % p.page
            row = p.seen(got["k"])[page, slot]  # [heads, bytes]
            d, m, _ = q4_ref.parts(row)
            y, delta = out[i].reshape(H, -1, 32), off[i].reshape(H, -1, 32).max(-1, keepdims=True)
            low, high = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
            step = 2.0 ** -11 * np.abs(low) + 2.0 ** -25 + 2 * delta
            assert (np.abs(m - low) <= step).all(), ("m", s, i)
            span = np.maximum(high - m, 0) / 15
            assert (np.abs(d - span) <= 2.0 ** -10 * span + 2.0 ** -24 + 2 * delta).all(), ("d", s, i)
            values = ref.decode(q4_ref.values(row), F16).reshape(y.shape)
            most = d / 2 + 45 * U * d + step + 2.0 ** -10 * 15 * span + 16 * 2.0 ** -24 + 2.0 ** -11 * (np.abs(y) + d)
            assert (np.abs(values - y) <= most).all(), ("k", s, i)
            p.seen(want["k"])[page, slot] = row
            p.seen(want["v"])[page, slot] = q4_ref.blocks_of(v[i])
    assert (got_q[~owned] == (0xA5A5A5A5 if q_type == F32 else 0xA5A5)).all(), "rows of no sequence"
    for n in "kv":
        assert np.array_equal(got[n], want[n]), n


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("name", APPENDS)
def test_append_matches_its_definition(gpu, name, form):
    case, more = dict(APPENDS[name]), dict(FORMS[form])
    q_heads = case.pop("q_heads")
    print(f"[case] append q4_1 {name} {form}", flush=True)
    p = Paged4(dim=more.pop("dim"), head_major=more.pop("head_major", False), seed=len(name), **case)
    made = append(gpu, p, q_heads, **more)
    check_append(p, q_heads, made, **more)
    assert p.fault() == 0


def test_positions_of_their_own(gpu):
    """Angles by the tokens that the sequences have had, places by the contexts; in every type of cache."""
    seen = [131000, 40, 9]
    p = Paged4([3, 1, 2], [50, 40, 2], dim=128, seed=3)
    check_append(p, 4, append(gpu, p, 4, seen=seen))
    for kind in (F16, BF16):  # as the same tokens at those positions of a longer context
        rows = []
        for contexts, more in (([50, 40, 2], seen), (seen, None)):
            p = Paged([3, 1, 2], contexts, dim=64, kind=kind, kv_heads=2, page=256, seed=4)
            x = np.random.default_rng(8).standard_normal((6, 4 * 64)).astype(np.float32)
            p.upload(gpu)
            xd, out = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer(6 * 2 * 64 * 4)
            k_out, v_out = gpu.DeviceBuffer(6 * 2 * 64 * 4), gpu.DeviceBuffer(6 * 2 * 64 * 4)
            rope = gpu.Rope(eps=EPS, base=1e6, dims=64)
            sd = gpu.DeviceBuffer.from_array(np.asarray(more, np.int32)) if more else None
            gpu.kv_append_at(p.cache, p.batch, sd, xd, 256, xd, 256, xd.ptr + 512, 256, 2, rope, out, F32)
            gpu.kv_rows(p.cache, p.batch, k_out, v_out, F32)
            gpu.synchronize()
            rows.append([b.download(np.uint32) for b in (out, k_out, v_out)])
        # (position 9 - 2 .. of the last sequence is not -1 .. of a context of 2)
        assert all(np.array_equal(a, b) for a, b in zip(*rows))


def test_broken_blocks(gpu):
    """A NaN, an infinity or a value beyond F16 makes its block NaN and no other."""
    p = Paged4([2], [2], dim=128, kv_heads=1, seed=5)

    def spoil(x):
        x[0, 128 + 3], x[0, 128 + 40], x[0, 128 + 70] = np.nan, np.inf, -65520.0  # values of token 0: blocks 0, 1, 2
        x[1, 128:128 + 32] = 0.25

    append(gpu, p, 0, dims=0, norm=False, spoil=spoil)
    k_out, v_out = (gpu.DeviceBuffer(2 * 128 * 4) for _ in range(2))
    gpu.kv_rows(p.cache, p.batch, k_out, v_out, F32)
    gpu.synchronize()
    v = v_out.download(np.float32).reshape(2, 4, 32)
    assert np.isnan(v[0, :3]).all() and np.isfinite(v[0, 3]).all()
    assert (v[1, 0] == 0.25).all() and np.isfinite(v[1]).all()
    assert np.isfinite(k_out.download(np.float32)).all()


def test_a_bad_page_stores_nothing(gpu):
    p = Paged4([4, 4], [20, 20], page=8, seed=9)
    p.table[0, 2] = p.pages
    p.table[1, 2] = -1
    append(gpu, p, 2)
    assert p.fault() == gpu.KV_FAULT_PAGE
    for n, before in (("k", p.k4), ("v", p.v4)):
        assert np.array_equal(p.downloaded(n), before)


# -------------------------------------------------------------------- rows --

@pytest.mark.parametrize("out_type", ["same", "f32"])
@pytest.mark.parametrize("kind", ["f16", "bf16", "q4_1"])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_come_out_as_they_are(gpu, dim, kind, out_type):
    make = Paged4 if kind == "q4_1" else Paged
    bits = BF16 if kind == "bf16" else F16
    for case in (dict(new=[1], contexts=[1]), dict(new=[7, 0, 40, 1], contexts=[7, 5, 61, 300], gaps=(2, 3), page=24),
                 dict(new=[33], contexts=[33], kv_heads=9, head_major=True)):
        p = make(kind=bits, dim=dim, seed=dim, **case)
        p.upload(gpu)
        T, H = p.tokens, p.kv_heads
        size = np.uint32 if out_type == "f32" else np.uint16
        outs = [gpu.DeviceBuffer.from_array(np.full((T, H, dim), 0x5A5A, size)) for _ in range(2)]
        gpu.kv_rows(p.cache, p.batch, *outs, F32 if out_type == "f32" else bits)
        gpu.synchronize()
        for out, pool in zip(outs, (p.k, p.v)):
            want = np.full((T, H, dim), 0x5A5A, size)
            for s, (n, c) in enumerate(zip(p.new, p.contexts)):
                rows = p.rows(s, pool)[c - n:]
                want[p.start[s]:p.start[s] + n] = (ref.decode(rows, bits).astype(np.float32).view(np.uint32)
                                                   if out_type == "f32" else rows)
            assert np.array_equal(out.download(size).reshape(want.shape), want)
        assert p.fault() == 0
        only = gpu.DeviceBuffer.from_array(np.zeros((T, H, dim), size))
        gpu.kv_rows(p.cache, p.batch, None, only, F32 if out_type == "f32" else bits)
        gpu.synchronize()
        owned = np.concatenate([np.arange(p.start[s], p.start[s] + n) for s, n in enumerate(p.new)]).astype(int)
        assert np.array_equal(only.download(size).reshape(T, H, dim)[owned], outs[1].download(size).reshape(T, H, dim)[owned])


def test_rows_of_bad_pages_are_nan(gpu):
    for make in (Paged, Paged4):
        p = make([3, 2], [20, 9], page=8, seed=3)
        p.table[0, 2] = p.pages + 4
        p.upload(gpu)
        outs = [gpu.DeviceBuffer(5 * 2 * 64 * 4) for _ in range(2)]
        gpu.kv_rows(p.cache, p.batch, *outs, F32)
        gpu.synchronize()
        for out, pool in zip(outs, (p.k, p.v)):
            got = out.download(np.float32).reshape(5, 2, 64)
            assert np.isnan(got[:3]).all()  # positions 17 .. 19 all lie on that page
            assert np.array_equal(got[3:], ref.decode(p.rows(1, pool), F16)[7:].astype(np.float32))
        assert p.fault() == gpu.KV_FAULT_PAGE


# --------------------------------------------------------------- attention --

def attend(gpu, p, q_heads, **more):
    a = Attend(gpu, p, q_heads, **more)
    a.call()
    a.call()
    gpu.synchronize()
    a.check()
    return a


@pytest.mark.parametrize("q_type", Q_TYPES)
@pytest.mark.parametrize("name", f16.CASES)
def test_attention_matches_its_definition(gpu, name, q_type):
    case = dict(f16.CASES[name])
    q_heads = case.pop("q_heads")
    for dim, head_major in ((128, False), (64, True)):
        print(f"[case] attention q4_1 {name} {q_type} dim={dim}", flush=True)
        attend(gpu, Paged4(dim=dim, head_major=head_major, seed=len(name) + dim, **case), q_heads, q_type=Q_TYPES[q_type], pad=8)


@pytest.mark.parametrize("q_type", Q_TYPES)
@pytest.mark.parametrize("window", [1, 64, 100, 5000])
def test_sliding_window(gpu, window, q_type):
    p = Paged4([1, 90, 3], [400, 300, 3], dim=128, seed=window)
    attend(gpu, p, 4, q_type=Q_TYPES[q_type], window=window)


@pytest.mark.parametrize("q_type", Q_TYPES)
@pytest.mark.parametrize("layout", f16.LAYOUTS)
@pytest.mark.parametrize("dim", [64, 128])
def test_layouts_of_large_calls(gpu, layout, q_type, dim):
    for new, contexts, window in (([100, 33, 0, 1], [700, 40, 9, 300], 0), ([90, 60], [400, 130], 70)):
        print(f"[case] attention q4_1 {layout} {q_type} dim={dim} window={window}", flush=True)
        more = dict(f16.LAYOUTS[layout])
        bound, heads = more.pop("max_context"), more.pop("kv_heads", 2)
        p = Paged4(new, contexts, kv_heads=heads, seed=dim, dim=dim, page=24, gaps=(1, 2))
        attend(gpu, p, heads if heads > 2 else 8, q_type=Q_TYPES[q_type], max_context=bound, window=window)


@pytest.mark.parametrize("q_type", Q_TYPES)
@pytest.mark.parametrize("name", f16.TILES)
@pytest.mark.parametrize("dim", [64, 128])
def test_tiles_and_parts(gpu, name, q_type, dim):
    """NaN blocks in every place that no row sees."""
    case = f16.TILES[name]
    print(f"[case] attention q4_1 tiles {name} {q_type} dim={dim}", flush=True)
    p = Paged4(case["new"], case["contexts"], kv_heads=case["kv_heads"], dim=dim, seed=dim + len(name))
    used = np.zeros((p.pages, p.page), bool)
    for s, c in enumerate(p.contexts):
        used[p.table[s, np.arange(c) // p.page], np.arange(c) % p.page] = True
    p.spoil(p.k4, ~used)
    p.spoil(p.v4, ~used)
    attend(gpu, p.settle(), case["kv_heads"] * case["group"], q_type=Q_TYPES[q_type], max_context=case["bound"])


@pytest.mark.parametrize("q_type", Q_TYPES)
@pytest.mark.parametrize("name", f16.MANY_PARTS)
def test_few_rows_in_many_parts(gpu, name, q_type):
    case = f16.MANY_PARTS[name]
    for dim in (64, 128):
        print(f"[case] attention q4_1 parts {name} {q_type} dim={dim}", flush=True)
        p = Paged4(case["new"], case["contexts"], kv_heads=case["kv_heads"], dim=dim, page=64, seed=dim + 1)
        attend(gpu, p, case["kv_heads"] * case["group"], q_type=Q_TYPES[q_type])


@pytest.mark.parametrize("q_type", Q_TYPES)
def test_batches_of_many_sequences(gpu, q_type):
    """Single tokens of uneven contexts, taken by length, and drafts of several tiles in parts."""
    rng = np.random.default_rng(21)
    new = [0 if i % 9 == 4 else 1 for i in range(70)]
    contexts = [max(int(c), n) for c, n in zip(rng.integers(1, 260, 70), new)]
    contexts[5] = contexts[33] = 1300
    print("[case] attention q4_1 by length", flush=True)
    attend(gpu, Paged4(new, contexts, kv_heads=4, dim=64, seed=22, gaps=(2, 1)), 8, q_type=Q_TYPES[q_type], max_context=1300)
    new = [int(n) for n in rng.integers(1, 11, 20)]
    contexts = [int(c) + n for c, n in zip(rng.integers(1, 500, 20), new)]
    contexts[3], contexts[11] = 4400, 2300
    print("[case] attention q4_1 several tiles", flush=True)
    attend(gpu, Paged4(new, contexts, kv_heads=6, dim=128, seed=34, gaps=(1, 2)), 24, q_type=Q_TYPES[q_type])


@pytest.mark.parametrize("q_type", Q_TYPES)
def test_nan_blocks_reach_only_the_rows_that_see_them(gpu, q_type):
    """A value's block of NaN: NaN in its columns from that position on, all else finite."""
    for new, contexts, bound in (([30], [30], 30), ([3], [60], 60), ([120, 80], [120, 333], 4000)):
        p = Paged4(new, contexts, dim=64, seed=4)
        at = contexts[0] - new[0] + 1
        rows = p.seen(p.v4)[p.table[0, at // p.page], at % p.page]
        rows[:, 20:24] = np.array([0x7E00, 0x7E00], np.uint16).view(np.uint8)  # block 1
        a = Attend(gpu, p.settle(), 2, q_type=Q_TYPES[q_type], max_context=bound)
        a.call()
        gpu.synchronize()
        out = ref.decode(a.results()[0], Q_TYPES[q_type])[:new[0]]
        assert np.isfinite(out[:1]).all() and np.isfinite(out[..., :32]).all()
        assert np.isnan(out[1:, :, 32:]).all()


@pytest.mark.parametrize("q_type", Q_TYPES)
def test_infinite_codes_reach_only_the_rows_that_see_them(gpu, q_type):
    """Blocks whose code 15 stands for an infinity: infinities and NaN where the definition has them, beside finite columns."""
    for new, contexts, bound in (([30], [30], 30), ([3], [60], 60), ([5, 1], [300, 90], 300), ([120, 80], [120, 333], 4000)):
        for dim in (64, 128):
            print(f"[case] attention q4_1 infinite codes {contexts} {q_type} dim={dim}", flush=True)
            p = Paged4(new, contexts, dim=dim, seed=14)
            first = contexts[0] - new[0]
            for at, d, codes in ((first + 1, 6000, {3: 15, 20: 15}), (first + 2, -6000, {3: 15, 7: 10})):  # block 1 of two tokens
                row = p.seen(p.v4)[p.table[0, at // p.page], at % p.page]
                row[:, 20:40] = 0
                row[:, 20:22] = np.array([d], np.float16).view(np.uint8)
                for i, code in codes.items():
                    row[:, 24 + i % 16] |= code << (4 if i >= 16 else 0)
            p.settle()
            a = Attend(gpu, p, 4, q_type=Q_TYPES[q_type], max_context=bound)
            a.call()
            gpu.synchronize()
            out = ref.decode(a.results()[0], Q_TYPES[q_type])[p.start[0]:p.start[1]]
            assert np.isfinite(out[:1]).all()
            assert np.isposinf(out[1:, :, 52]).all() and np.isposinf(out[1, :, 35]).all() and np.isnan(out[2:, :, 35]).all()
            others = np.delete(out, [35, 52], axis=-1)
            assert np.isfinite(others).all()
            V = ref.decode(p.rows(0, p.v), F16)[:, :, 39]
            assert V[first + 2, 0] == -60000 and p.fault() == 0


@pytest.mark.parametrize("q_type", Q_TYPES)
def test_weights_beside_much_larger_ones_keep_their_precision(gpu, q_type):
    """A first token of near-zero value that takes nearly all of the mass."""
    for new, contexts in (([1, 1], [1000, 333]), ([40], [700])):
        p = Paged4(new, contexts, dim=128, seed=6)
        a = Attend(gpu, p, 4, q_type=Q_TYPES[q_type])
        first = p.seen(p.v4)
        for s in range(len(new)):
            first[p.table[s, 0], 0] = q4_ref.blocks_of(np.full((2, 128), 2.0 ** -12, np.float32))
            q = ref.decode(a.q, a.q_type)[p.start[s], :4 * 128].reshape(4, 128)
            for h in range(2):  # a key along the first of the head's queries
                k = q[2 * h] / np.linalg.norm(q[2 * h]) * 14.0 / abs(float(a.scale)) / np.linalg.norm(q[2 * h])
                p.seen(p.k4)[p.table[s, 0], 0, h] = q4_ref.blocks_of(k.astype(np.float32)[None])[0]
        p.settle()
        p.dev["k"].upload(p.k4)
        p.dev["v"].upload(p.v4)
        a.call()
        gpu.synchronize()
        a.check()


@pytest.mark.parametrize("q_type", Q_TYPES)
def test_weights_keep_their_precision_over_blocks_whose_largest_code_leaves_f16(gpu, q_type):
    """The same where the other tokens' blocks are not the append's: code 15, which none of them
    holds, would stand for an infinity, and what they do hold is near F16's largest value."""
    for new, contexts in (([1, 1], [1000, 333]), ([3, 2], [400, 90]), ([40], [700])):
        for dim in (64, 128):
            print(f"[case] attention q4_1 large blocks {contexts} {q_type} dim={dim}", flush=True)
            p = Paged4(new, contexts, dim=dim, seed=7)
            blocks = p.v4.reshape(-1, 20)
            blocks[:, 4:] = p.rng.integers(0, 11, (len(blocks), 16)) | p.rng.integers(0, 11, (len(blocks), 16)) << 4
            d = np.where(p.rng.random(len(blocks)) < 0.5, 6000.0, -6000.0).astype(np.float16)
            blocks[:, :4] = np.stack([d, np.zeros_like(d)], -1).view(np.uint8)
            a = Attend(gpu, p, 4, q_type=Q_TYPES[q_type])
            for s in range(len(new)):
                p.seen(p.v4)[p.table[s, 0], 0] = 0
                q = ref.decode(a.q, a.q_type)[p.start[s], :4 * dim].reshape(4, dim)
                for h in range(2):  # a key along the first of the head's queries, 25 nats ahead
                    k = q[2 * h] / (q[2 * h] @ q[2 * h]) * 25.0 / abs(float(a.scale))
                    p.seen(p.k4)[p.table[s, 0], 0, h] = q4_ref.blocks_of(k.astype(np.float32)[None])[0]
            p.settle()
            assert np.isfinite(ref.decode(p.v, F16)).all()
            p.dev["k"].upload(p.k4)
            p.dev["v"].upload(p.v4)
            a.call()
            gpu.synchronize()
            a.check()


def test_bad_pages_are_reported_and_reach_no_other_sequence(gpu):
    for new, contexts in (([1, 1, 1], [40, 40, 40]), ([30, 30, 30], [40, 40, 40])):
        p = Paged4(new, contexts, page=8, dim=128, seed=16)
        p.table[1, 3] = p.pages + 5
        a = Attend(gpu, p, 4)
        a.call()
        gpu.synchronize()
        assert np.isnan(a.results()[0][p.start[2] - 1].view(np.float32)).all()
        assert p.fault() == gpu.KV_FAULT_PAGE
        with pytest.raises(gpu.QKError, match="page"):
            gpu.kv_check(p.cache)
        a.check(sequences=(0, 2))


def test_another_stream_and_captured_replays(gpu):
    """Append, attention and rows captured together, replayed on changed lengths with eager work in between."""
    p = Paged4([1, 1, 1], [600, 40, 1300], dim=128, kv_heads=2, spare=4, seed=17)
    a = Attend(gpu, p, 8, max_context=1300)
    x = np.random.default_rng(3).standard_normal((3, 2 * 2 * 128)).astype(np.float32)
    xd, k_out, v_out = gpu.DeviceBuffer.from_array(x), gpu.DeviceBuffer(3 * 256 * 2), gpu.DeviceBuffer(3 * 256 * 2)
    rope = gpu.Rope(eps=EPS, base=1e4, dims=128)

    def step(stream=None):
        gpu.kv_append(p.cache, p.batch, None, 0, xd, 512, xd.ptr + 1024, 512, 0, rope, None, F32, stream)
        a.call(stream)
        gpu.kv_rows(p.cache, p.batch, k_out, v_out, F16, stream)

    stream = gpu.Stream()
    graph = gpu.Graph.capture(stream, lambda: step(stream))
    for i, contexts in enumerate(([600, 40, 1300], [601, 41, 1], [17, 33, 1299], [600, 40, 1300])):
        print(f"[case] q4_1 graph replay {i}", flush=True)
        p.contexts = list(contexts)
        p.dev["context"].upload(np.asarray(contexts, np.int32))
        graph.launch(stream)
        stream.synchronize()
        replay = [y.copy() for y in a.results()] + [k_out.download(np.uint16), v_out.download(np.uint16)]
        p.k4, p.v4 = p.downloaded("k"), p.downloaded("v")
        p.settle()
        a.check()
        a.out.fill(0x5A)
        step()
        gpu.synchronize()
        eager = [*a.results(), k_out.download(np.uint16), v_out.download(np.uint16)]
        assert all(np.array_equal(y.view(np.uint8), z.view(np.uint8)) for y, z in zip(replay, eager))
        got = v_out.download(np.uint16).reshape(3, 2, 128)
        assert np.array_equal(got, q4_ref.values(q4_ref.blocks_of(x[:, 256:].reshape(3, 2, 128))))
    graph.destroy()
    stream.destroy()


def test_a_page_far_into_a_large_pool(gpu):
    """Offsets past 2^32 bytes: a pool of 4.5 GB, pages at its end."""
    P, H, D = 64, 8, 128
    page_bytes = P * H * D // 32 * 20
    pages = (9 << 29) // page_bytes + 3
    p = Paged4([2], [130], kv_heads=H, dim=D, page=P, seed=18)
    big = {n: gpu.DeviceBuffer(pages * page_bytes) for n in "kv"}
    a = Attend(gpu, p, 16)
    far = np.array([[pages - 1, pages - 3, pages - 2]], np.int32)
    for n, pool in (("k", p.k4), ("v", p.v4)):
        for e in range(3):
            big[n].upload(pool[p.table[0, e]], offset=int(far[0, e]) * page_bytes)
    p.dev["table"].upload(far)
    p.cache.k, p.cache.v, p.cache.pages = big["k"].ptr, big["v"].ptr, pages
    a.call()
    rows = [gpu.DeviceBuffer(2 * H * D * 2) for _ in range(2)]
    gpu.kv_rows(p.cache, p.batch, *rows, F16)
    gpu.synchronize()
    a.check()
    for out, pool in zip(rows, (p.k, p.v)):
        assert np.array_equal(out.download(np.uint16).reshape(2, H, D), p.rows(0, pool)[-2:])
    for b in big.values():
        b.free()


@pytest.mark.parametrize("bound", [0, 1, 300, 1 << 62])
@pytest.mark.parametrize("q_type", Q_TYPES)
def test_contexts_beyond_the_bound(gpu, bound, q_type):
    """max_context shares the work out; results do not depend on it."""
    for new, contexts, window in (([1], [2500], 0), ([1, 1, 1], [3000, 40, 1300], 0), ([2, 5], [1500, 700], 600)):
        print(f"[case] attention q4_1 bound={bound} {q_type} {contexts} window={window}", flush=True)
        p = Paged4(new, contexts, kv_heads=2, dim=128, seed=len(contexts))
        attend(gpu, p, 8, q_type=Q_TYPES[q_type], max_context=bound, window=window)
