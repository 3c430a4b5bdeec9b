"""qk_kv_append against the definition in 64 bits.

Tolerances, in units u = 2^-24 of the length of the rotated pair: the norm's
sum of squares is 4 + 8 additions deep (8 values a lane, then 4 or 3 lane
exchanges; half of it after the root), its root and reciprocal 2, the two
products 2: 10 u; the angle, a fraction of a turn rounded to fp32, is off by
at most 2 pi u / 2, sine and cosine by 2 u each: 6 u; the rotation's products
and sum 2 u. 24 u covers them; a 16-bit output adds half of its step."""
from __future__ import annotations

import numpy as np
import pytest

import serving_ref as ref
from serving_ref import BF16, F16, F32, Paged

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


class Append:
    def __init__(self, qk, p: Paged, q_heads, *, q_type=F32, dims=None, interleaved=False, norm=True, base=1e6, pad=0,
                 in_place=False):
        D, H, T, rng = p.dim, p.kv_heads, p.tokens, p.rng
        self.p, self.q_heads, self.q_type = p, q_heads, q_type
        self.dims, self.interleaved, self.base = D if dims is None else dims, interleaved, base
        # rows of one fused projection: q, k and v of a token side by side, `pad` floats between tokens
        self.width = (q_heads + 2 * H) * D + pad
        self.x = (rng.standard_normal((T, self.width)) * 2).astype(np.float32)
        self.norms = [(1 + 0.2 * rng.standard_normal(D)).astype(np.float32) if norm else None for _ in range(2)]
        p.upload(qk)
        self.xd = qk.DeviceBuffer.from_array(self.x)
        self.nd = [qk.DeviceBuffer.from_array(n) if n is not None else None for n in self.norms]
        size = 4 if q_type == F32 else 2
        self.q_out = qk.DeviceBuffer.from_array(np.full(max(1, T * q_heads * D * size), 0xA5, np.uint8))
        self.rope = qk.Rope(q_norm=self.nd[0].ptr if norm else None, k_norm=self.nd[1].ptr if norm else None, eps=EPS,
                            base=base, dims=self.dims, interleaved=interleaved)
        self.qk = qk

    def call(self, stream=None):
        p, D = self.p, self.p.dim
        k_at, v_at = self.q_heads * D * 4, (self.q_heads + p.kv_heads) * D * 4
        self.qk.kv_append(p.cache, p.batch, self.xd.ptr if self.q_heads else None, self.width, self.xd.ptr + k_at,
                          self.width, self.xd.ptr + v_at, self.width, self.q_heads, self.rope,
                          self.q_out.ptr if self.q_heads else None, self.q_type, stream)

    def check(self, skip=()):
        """Every value of q_out and of both pools; `skip`: (sequence, position) whose rows are not stored."""
        p, D, H = self.p, self.p.dim, self.p.kv_heads
        want = {"k": ref.decode(p.k, p.kind).copy(), "v": ref.decode(p.v, p.kind).copy()}
        tol = {n: np.zeros_like(a) for n, a in want.items()}
        size = np.uint32 if self.q_type == F32 else np.uint16
        T = p.tokens
        got_q = self.q_out.download(size)[:T * self.q_heads * D].reshape(T, self.q_heads, D)
        owned = np.zeros(T, bool)
        for s, (n, c) in enumerate(zip(p.new, p.contexts)):
            rows = slice(p.start[s], p.start[s] + n)
            owned[rows] = True
            pos = np.arange(c - n, c)
            x = self.x[rows]
            parts = np.split(x[:, :(self.q_heads + 2 * H) * D].reshape(n, self.q_heads + 2 * H, D), [self.q_heads, self.q_heads + H], 1)
            for name, part, weight, kind in (("q", parts[0], self.norms[0], self.q_type),
                                             ("k", parts[1], self.norms[1], p.kind)):
                out = ref.rotate(part, pos, weight, EPS, self.base, self.dims, self.interleaved)
                plain = ref.rotate(part, pos, weight, EPS, self.base, 0, False)
                off = 24 * U * ref.pair_size(plain, self.dims, self.interleaved)
                off = off + ref.HALF_STEP[kind] * (np.abs(out) + off) + ref.TINY[kind]
                if name == "q":
                    if self.q_heads:
                        err = np.abs(ref.decode(got_q[rows], kind) - out)
                        assert (err <= off).all(), ("q", s, (err / off).max())
                    continue
                for i in range(n):
                    if (s, pos[i]) in skip or pos[i] < 0:
                        continue
                    page, slot = p.table[s, pos[i] // p.page], pos[i] % p.page
                    p.seen(want["k"])[page, slot], p.seen(tol["k"])[page, slot] = out[i], off[i]
                    p.seen(want["v"])[page, slot] = ref.decode(ref.encode(parts[2][i], p.kind), p.kind)
        if self.q_heads:
            untouched = got_q[~owned]
            assert (untouched == (0xA5A5A5A5 if self.q_type == F32 else 0xA5A5)).all(), "rows of no sequence"
        for name in ("k", "v"):
            got = ref.decode(p.dev[name].download(np.uint16).reshape(p.k.shape), p.kind)
            err = np.abs(got - want[name])
            assert (err <= tol[name]).all(), (name, err.max())  # tolerance 0: old values stay, v is one rounding


CASES = {
    "one-token": dict(new=[1], contexts=[1], q_heads=4),
    "decode-far": dict(new=[1, 1, 1], contexts=[100001, 17, 131072], q_heads=4, page=256, kv_heads=1),
    "ragged": dict(new=[5, 1, 33, 16], contexts=[5, 40, 50, 16], q_heads=6, page=24, dim=64),
    "empty-sequences": dict(new=[0, 3, 0, 0, 2, 0], contexts=[0, 3, 9, 0, 20, 4], q_heads=2),
    "padding-rows": dict(new=[2, 3], contexts=[2, 7], q_heads=2, gaps=(3, 2)),
    "page-1": dict(new=[7, 2], contexts=[9, 2], q_heads=2, page=1),
    "odd-page": dict(new=[40], contexts=[41], q_heads=2, page=7, dim=128),
    "qwen3-heads": dict(new=[2, 1], contexts=[70, 3], q_heads=32, kv_heads=8, dim=128),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("form", ["f16", "bf16-same-head-major", "f16-pairs-partial", "bf16-no-norm", "plain-same"])
def test_append_matches_its_definition(gpu, name, form):
    case = dict(CASES[name])
    q_heads = case.pop("q_heads")
    kind = BF16 if "bf16" in form else F16
    case.setdefault("dim", 128 if form == "f16" else 64)
    print(f"[case] append {name} {form}", flush=True)
    p = Paged(kind=kind, head_major="major" in form, seed=len(name), **case)
    a = Append(gpu, p, q_heads, q_type=kind if "same" in form else F32, interleaved="pairs" in form,
               dims=0 if form == "plain-same" else p.dim // 2 if "partial" in form else None,
               norm=form not in ("bf16-no-norm", "plain-same"), base=1e4 if "pairs" in form else 1e6, pad=3)
    a.call()
    gpu.synchronize()
    a.check()
    assert p.fault() == 0
    gpu.kv_check(p.cache)


def test_append_without_queries_and_without_rope(gpu):
    p = Paged([3, 2], [10, 2], seed=5)
    a = Append(gpu, p, 0, dims=0, norm=False)
    a.rope = None
    a.call()
    gpu.synchronize()
    a.check()


def test_queries_may_be_rotated_in_place(gpu):
    p = Paged([3, 9], [10, 9], kv_heads=2, dim=128, seed=6).upload(gpu)
    T, H, D = p.tokens, 4, 128
    q = p.rng.standard_normal((T, H, D)).astype(np.float32)
    kv = gpu.DeviceBuffer.from_array(p.rng.standard_normal((T, 2, D)).astype(np.float32))
    d, out = gpu.DeviceBuffer.from_array(q), gpu.DeviceBuffer(4 * q.size)
    rope = gpu.Rope(eps=EPS, base=1e4, dims=D)
    gpu.kv_append(p.cache, p.batch, d, H * D, kv, 2 * D, kv, 2 * D, H, rope, out, F32)
    gpu.kv_append(p.cache, p.batch, d, H * D, kv, 2 * D, kv, 2 * D, H, rope, d, F32)
    gpu.synchronize()
    assert np.array_equal(d.download(np.uint32), out.download(np.uint32))


def test_values_beyond_the_cache_type_saturate_as_the_type_does(gpu):
    p = Paged([1], [1], kv_heads=1, kind=F16, seed=7).upload(gpu)
    x = np.zeros((1, 1, 64), np.float32)
    x[0, 0, :6] = [1e6, -1e6, np.inf, np.nan, 65519.9, 1e-9]
    d = gpu.DeviceBuffer.from_array(x)
    gpu.kv_append(p.cache, p.batch, None, 0, d, 64, d, 64, 0, None, None, F32)
    gpu.synchronize()
    got = ref.decode(p.seen(p.dev["v"].download(np.uint16).reshape(p.k.shape))[p.table[0, 0], 0, 0], F16)
    assert got[0] == np.inf and got[1] == -np.inf and got[2] == np.inf and np.isnan(got[3])
    assert got[4] == 65504 and got[5] == 0


def test_bad_pages_and_lengths_store_nothing_and_are_reported(gpu):
    """Page ids outside the pool, positions past the table, contexts shorter
    than their new tokens: those rows are not stored, the rest is, and
    kv_check says so once."""
    p = Paged([4, 4, 2], [20, 20, 2], page=8, seed=9)
    p.table[0, 2] = p.pages        # positions 16 .. 19 of sequence 0
    p.table[1, 2] = -1
    a = Append(gpu, p, 2)
    a.call()
    gpu.synchronize()
    a.check(skip={(s, t) for s in (0, 1) for t in range(16, 20)})
    assert p.fault() == gpu.KV_FAULT_PAGE
    with pytest.raises(gpu.QKError, match="page"):
        gpu.kv_check(p.cache)
    gpu.kv_check(p.cache)  # cleared

    p = Paged([3], [40], page=8, seed=10)
    a = Append(gpu, p, 2)
    p.batch.table_stride = 4  # position 32 and on have no entry
    a.call()
    gpu.synchronize()
    assert p.fault() == gpu.KV_FAULT_PAGE
    a.check(skip={(0, t) for t in range(37, 40)})

    p = Paged([5], [2], page=8, seed=11)  # positions -3 .. 1
    a = Append(gpu, p, 2)
    a.call()
    gpu.synchronize()
    a.check()
    assert p.fault() == gpu.KV_FAULT_LENGTH
    with pytest.raises(gpu.QKError, match="token_start"):
        gpu.kv_check(p.cache)


def test_captured_append_serves_new_lengths(gpu):
    """One captured step, replayed on changed lengths, tables and inputs with
    eager work between the replays."""
    p = Paged([1, 1, 1], [5, 40, 17], page=8, extra_entries=2, spare=12, seed=12)  # 21 pages, 7 entries a row
    a = Append(gpu, p, 4)
    stream = gpu.Stream()
    graph = gpu.Graph.capture(stream, lambda: a.call(stream))
    for step in range(4):
        print(f"[case] append graph replay {step}", flush=True)
        contexts = p.contexts = [5 + step, 41 - 9 * step, 17 + step]
        p.table = ((np.arange(21) * 5 + step) % 21).astype(np.int32).reshape(3, 7)
        p.dev["context"].upload(np.asarray(contexts, np.int32))
        p.dev["table"].upload(p.table)
        p.k, p.v = p.dev["k"].download(np.uint16).reshape(p.k.shape), p.dev["v"].download(np.uint16).reshape(p.k.shape)
        graph.launch(stream)
        stream.synchronize()
        a.check()
    graph.destroy()
    stream.destroy()


def test_lengths_that_do_not_fit_are_reported_whoever_owns_the_rows(gpu):
    """A sequence that owns no row, and a negative context, store nothing and are reported."""
    p = Paged([3, 0], [20, 9], page=8, seed=14)
    a = Append(gpu, p, 2)
    p.dev["context"].upload(np.asarray([20, -1], np.int32))
    a.call()
    gpu.synchronize()
    assert p.fault() == gpu.KV_FAULT_LENGTH
    p.dev["fault"].upload(np.zeros(1, np.uint32))
    a.check()
    for context in (-1, -(1 << 31)):
        p = Paged([2, 3], [20, 9], page=8, seed=15)
        a = Append(gpu, p, 2)
        p.dev["context"].upload(np.asarray([20, context], np.int32))
        before = [p.dev[n].download(np.uint16).reshape(p.k.shape) for n in "kv"]
        a.call()
        gpu.synchronize()
        assert p.fault() == gpu.KV_FAULT_LENGTH
        for n, pool in zip("kv", before):
            after = p.dev[n].download(np.uint16).reshape(p.k.shape)
            held = p.table[1, :2]
            assert np.array_equal(p.seen(after)[held], p.seen(pool)[held])
    p = Paged([2, 3, 1], [20, 9, 5], page=8, seed=16)
    a = Append(gpu, p, 2)
    p.dev["start"].upload(np.asarray([0, 5, 2, 6], np.int32))
    a.call()
    gpu.synchronize()
    assert p.fault() & gpu.KV_FAULT_LENGTH


def test_a_check_names_and_clears_what_it_read(gpu):
    p = Paged([1], [5], page=8, seed=17).upload(gpu)
    page, length = gpu.KV_FAULT_PAGE, gpu.KV_FAULT_LENGTH
    for word, named in ((page, ["page"]), (length, ["token_start"]), (page | length, ["page", "token_start"])):
        p.dev["fault"].upload(np.asarray([word], np.uint32))
        with pytest.raises(gpu.QKError) as error:
            gpu.kv_check(p.cache)
        for name in ("page", "token_start"):
            assert (name in str(error.value)) == (name in named)
        assert p.fault() == 0
        gpu.kv_check(p.cache)


def test_checks_beside_calls_on_another_stream_lose_no_fault(gpu):
    """Every faulty call is followed by a check on its own stream while checks on
    another stream run: one of the two reports it."""
    import threading

    p = Paged([2], [20], page=8, seed=18)
    p.table[0, 2] = -1
    a = Append(gpu, p, 2)
    mine, theirs = gpu.Stream(), gpu.Stream()
    reports, done = [0], threading.Event()

    def check(stream):
        try:
            gpu.kv_check(p.cache, stream)
        except gpu.QKError:
            return 1
        return 0

    def others():
        while not done.is_set():
            reports[0] += check(theirs)

    thread = threading.Thread(target=others)
    thread.start()
    try:
        for _ in range(50):
            before = reports[0]
            a.call(mine)
            found = check(mine)
            mine.synchronize()
            if not found:  # the other's, on its way at most
                for _ in range(2000):
                    if reports[0] > before:
                        break
                    done.wait(0.001)
                assert reports[0] > before
    finally:
        done.set()
        thread.join()
    for stream in (mine, theirs):
        stream.synchronize()
        stream.destroy()
