"""qk_kv_weigh and qk_kv_evict against their definitions in 64 bits, and a session
that lives with both.

Weights, u = 2^-24: a score is off by d = (D/4 + 6) u reach (reach = |scale| sum |q k|,
as in test_gpu_paged_attention), the row's log by its rounding in base 2 and the sum
with it, 3 u |lse|, the exponential by 4 u and its argument's rounding 2 u (|score| +
|lse|): a weight is so off by (d + (2 reach + 5 |lse| + 6) u) of itself. Sums of n
positive weights in one register are off by n u at most: rows / 2 of them a lane, joined
in up to 40 parts. What was there is added with one rounding more.
An eviction moves bits: everything is equal."""
from __future__ import annotations

import numpy as np
import pytest

import q4_ref
import serving_ref as ref
from q4_ref import Paged4
from serving_ref import BF16, F16, F32, Paged

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
KINDS = {"f16": (Paged, F16), "bf16": (Paged, BF16), "q4_1": (Paged4, F16)}


def make(kind, new, contexts, **more):
    cls, bits = KINDS[kind]
    return cls(new, contexts, kind=bits, **more)


def add_weights(gpu, p, seed=1):
    """weight and position of every slot, random, on the host and the device."""
    rng = np.random.default_rng(seed)
    shape = (p.pages, p.kv_heads, p.page)
    p.weight = np.exp(rng.standard_normal(shape)).astype(np.float32)
    p.position = rng.integers(0, 1000, shape).astype(np.int32)
    p.dev["weight"], p.dev["position"] = (gpu.DeviceBuffer.from_array(x) for x in (p.weight, p.position))
    p.weights = gpu.KVWeights(weight=p.dev["weight"].ptr, position=p.dev["position"].ptr)


def slots(p, s, n):
    """(pages, slots) of a sequence's first n places."""
    j = np.arange(n)
    return p.table[s, j // p.page], j % p.page


class Weigh:
    def __init__(self, gpu, p, q_heads, *, q_type=F32, seen=None, max_context=None, pad=0, scale=None, q_size=1.5):
        self.gpu, self.p, self.q_heads, self.q_type, self.seen = gpu, p, q_heads, q_type, seen
        D, T = p.dim, p.tokens
        self.scale = np.float32(D ** -0.5 if scale is None else scale)
        self.stride = q_heads * D + pad
        self.q = ref.encode(p.rng.standard_normal((T, self.stride)) * q_size, q_type)
        p.upload(gpu)
        add_weights(gpu, p)
        self.lse = np.full((T, q_heads), np.nan, np.float32)
        G = q_heads // p.kv_heads
        self.want, self.off, self.want_position = p.weight.astype(np.float64), np.zeros(p.weight.shape), p.position.copy()
        q64 = ref.decode(self.q, q_type)
        for s, (n, c) in enumerate(zip(p.new, p.contexts)):
            if n == 0:
                continue
            K = ref.decode(p.rows(s, p.k), p.kind)
            pg, sl = slots(p, s, c)
            rows = np.arange(p.start[s], p.start[s] + n)
            seen_here = np.arange(c)[None] <= np.arange(c - n, c)[:, None]
            self.want[pg[c - n:], :, sl[c - n:]] = 0
            self.want_position[pg[c - n:], :, sl[c - n:]] = (np.arange(c - n, c) + (0 if seen is None else seen[s] - c))[:, None]
            for h in range(q_heads):
                qh = q64[rows, h * D:(h + 1) * D]
                with np.errstate(invalid="ignore"):
                    x = np.where(seen_here, float(self.scale) * (qh @ K[:, h // G].T), -np.inf)
                    reach = abs(float(self.scale)) * (np.abs(qh) @ np.abs(K[:, h // G]).T)
                top = x.max(1)
                self.lse[rows, h] = top + np.log(np.exp(x - top[:, None]).sum(1))
                lse = self.lse[rows, h].astype(np.float64)[:, None]
                w = np.exp(x - lse)
                e = ((D / 4 + 8) * reach + 5 * np.abs(lse) + 6) * U
                self.want[pg, h // G, sl] += w.sum(0)
                self.off[pg, h // G, sl] += (w * e).sum(0) + (n * G / 2 + 40) * U * w.sum(0)
        self.off += U * np.abs(self.want)
        self.off[self.want == p.weight] = 0
        self.qd, self.lsed = gpu.DeviceBuffer.from_array(self.q), gpu.DeviceBuffer.from_array(self.lse)
        self.seend = gpu.DeviceBuffer.from_array(np.asarray(seen, np.int32)) if seen is not None else None
        self.max_context = max(p.contexts, default=0) if max_context is None else max_context
        n = gpu.kv_weigh_workspace_size(p.cache, p.batch, q_type, q_heads, self.max_context)
        self.ws = gpu.DeviceBuffer.from_array(np.full(max(n, 256), 0x5A, np.uint8))

    def call(self, stream=None):
        p = self.p
        self.gpu.kv_weigh(p.cache, p.batch, self.seend, self.qd, self.q_type, self.stride, self.q_heads, self.scale,
                          self.lsed, self.max_context, p.weights, self.ws, self.ws.nbytes, stream)

    def got(self):
        p = self.p
        return (p.dev["weight"].download(np.float32).reshape(p.weight.shape),
                p.dev["position"].download(np.int32).reshape(p.position.shape))

    def check(self):
        weight, position = self.got()
        assert np.array_equal(position, self.want_position)
        err = np.abs(weight - self.want)
        assert (err <= self.off).all(), (np.argwhere(~(err <= self.off))[:4], (err / np.where(self.off > 0, self.off, 1)).max())


WEIGH = {
    "one-key": dict(new=[1], contexts=[1], q_heads=2),
    "decode": dict(new=[1] * 5, contexts=[1, 31, 32, 33, 200], q_heads=8),
    "decode-long": dict(new=[1, 1], contexts=[3000, 1025], q_heads=8, page=64),
    "drafts": dict(new=[3, 4, 2], contexts=[3, 70, 130], q_heads=8, page=24),
    "two-row-tiles": dict(new=[9, 1, 0, 7], contexts=[200, 90, 40, 7], q_heads=8),
    "ragged": dict(new=[1, 37, 0, 130, 1], contexts=[300, 37, 50, 140, 1], q_heads=4),
    "chunk": dict(new=[150], contexts=[410], q_heads=4, page=7),
    "prompt": dict(new=[300], contexts=[300], q_heads=8, page=256),
    "prompts-parts": dict(new=[400, 350], contexts=[900, 351], q_heads=8, page=24),
    "odd-group": dict(new=[9, 1], contexts=[30, 333], q_heads=14),
    "odd-group-chunk": dict(new=[90, 70], contexts=[290, 70], q_heads=14),
    "no-group": dict(new=[20, 1], contexts=[31, 90], q_heads=3, kv_heads=3),
    "wide-group": dict(new=[2, 1], contexts=[33, 65], q_heads=40, kv_heads=1),
    "page-1": dict(new=[5], contexts=[77], q_heads=2, page=1),
    "padding-rows": dict(new=[2, 0, 40], contexts=[9, 3, 45], q_heads=4, gaps=(3, 5)),
    "empty-context": dict(new=[0, 2, 0], contexts=[0, 2, 0], q_heads=2),
}


@pytest.mark.parametrize("q", ["f32", "same"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", WEIGH)
def test_weights_match_their_definition(gpu, name, kind, q):
    case = dict(WEIGH[name])
    q_heads = case.pop("q_heads")
    for dim, head_major in ((128, False), (64, True)):
        print(f"[case] weigh {name} {kind} {q} dim={dim}", flush=True)
        p = make(kind, dim=dim, head_major=head_major, seed=len(name) + dim, **case)
        seen = [c + 17 * s for s, c in enumerate(p.contexts)] if dim == 64 else None
        w = Weigh(gpu, p, q_heads, q_type=F32 if q == "f32" else KINDS[kind][1], pad=8, seen=seen)
        w.call()
        gpu.synchronize()
        w.check()
        assert p.fault() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_weights_add_up_in_the_same_order_every_time(gpu, kind):
    """Twice on the same start: the same bits; and twice in a row: old tokens' weights grow."""
    for new, contexts in (([1, 2], [90, 700]), ([200], [600]), ([500, 3], [500, 90])):
        p = make(kind, new, contexts, dim=128, seed=9)
        w = Weigh(gpu, p, 4)
        w.call()
        gpu.synchronize()
        first = w.got()
        p.dev["weight"].upload(p.weight)
        w.call()
        gpu.synchronize()
        assert np.array_equal(w.got()[0].view(np.uint32), first[0].view(np.uint32))
        w.call()
        gpu.synchronize()
        for s, (n, c) in enumerate(zip(new, contexts)):
            pg, sl = slots(p, s, c)
            again, once = w.got()[0][pg, :, sl], first[0][pg, :, sl]
            assert np.array_equal(again[c - n:], once[c - n:])
            assert (again[:c - n] >= once[:c - n]).all() and (c == n or (again[:c - n] > once[:c - n]).any())


@pytest.mark.parametrize("kind", KINDS)
def test_rows_without_a_log_give_nothing(gpu, kind):
    """lse of -inf and NaN, and keys that are NaN: nothing, and no harm to others."""
    for new, contexts in (([2], [60]), ([90], [150])):
        p = make(kind, new, contexts, dim=64, seed=5)
        w = Weigh(gpu, p, 4)
        lse = w.lse.copy()
        lse[:, 1], lse[:, 3] = -np.inf, np.nan
        w.lsed.upload(lse)
        w.call()
        gpu.synchronize()
        half = w.got()[0]
        lse = w.lse.copy()
        lse[:, 1] = lse[:, 3] = 1e30  # weights of nothing
        w.lsed.upload(lse)
        p.dev["weight"].upload(p.weight)
        w.call()
        gpu.synchronize()
        assert np.array_equal(w.got()[0], half)
        # a key of NaN
        if kind == "q4_1":
            p.spoil(p.k4, (p.table[0, 0], 3))
            p.dev["k"].upload(p.k4)
        else:
            p.seen(p.k)[p.table[0, 0], 3, :, 5] = ref.encode(np.nan, p.kind)
            p.dev["k"].upload(p.k)
        p.dev["weight"].upload(p.weight)
        w.call()
        gpu.synchronize()
        got = w.got()[0]
        half[p.table[0, 0], :, 3] = p.weight[p.table[0, 0], :, 3]
        assert np.array_equal(got, half)


def test_weights_of_bad_pages_and_lengths(gpu):
    for new, contexts in (([1, 1, 1], [40, 40, 40]), ([50, 50, 50], [60, 60, 60])):
        p = Paged(new, contexts, page=8, dim=128, seed=16)
        page = p.table[1, 3]
        p.table[1, 3] = p.pages + 5
        p.table = p.table.copy()
        good = p.table.copy()
        good[1, 3] = page
        p.table = good
        w = Weigh(gpu, p, 4)
        bad = good.copy()
        bad[1, 3] = p.pages + 5
        p.dev["table"].upload(bad)
        w.call()
        gpu.synchronize()
        assert p.fault() == gpu.KV_FAULT_PAGE
        p.dev["fault"].upload(np.zeros(1, np.uint32))
        w.want[page], w.want_position[page], w.off[page] = p.weight[page], p.position[page], 0  # untouched
        w.check()
        # a context past its table, one past the bound, one shorter than its new tokens
        for context, fault in ((8 * p.table.shape[1] + 1, "page"), (-1, "length")):
            p.dev["table"].upload(good)
            lengths = np.asarray(contexts, np.int32)
            lengths[1] = context
            p.dev["context"].upload(lengths)
            p.dev["weight"].upload(p.weight)
            p.dev["position"].upload(p.position)
            w.call()
            gpu.synchronize()
            assert p.fault() & (gpu.KV_FAULT_PAGE if fault == "page" else gpu.KV_FAULT_LENGTH)
            p.dev["fault"].upload(np.zeros(1, np.uint32))
            got = w.got()[0]
            held = p.table[1]
            assert np.array_equal(got[held], p.weight[held])
        # longer than max_context by more than a share
        p.dev["context"].upload(np.asarray(contexts, np.int32))
        p.dev["weight"].upload(p.weight)
        p.dev["position"].upload(p.position)
    p = Paged([1], [2000], dim=64, seed=17)
    w = Weigh(gpu, p, 4, max_context=100)
    w.call()
    gpu.synchronize()
    assert p.fault() == gpu.KV_FAULT_LENGTH
    assert np.array_equal(w.got()[0], p.weight)


@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("kind", ["q4_1", "f16"])
def test_weights_of_many_contexts(gpu, kind, head_major):
    """More (context, head) units than compute units, and parts of contexts that eight do not divide."""
    print(f"[case] weigh many contexts {kind} head_major={head_major}", flush=True)
    rng = np.random.default_rng(31)
    new = [0 if i % 11 == 5 else 3 if i % 7 == 2 else 1 for i in range(35)]
    contexts = [max(int(c), n) for c, n in zip(rng.integers(1, 701, 35), new)]
    contexts[20] = 700
    p = make(kind, new, contexts, kv_heads=9, dim=64, page=24, head_major=head_major, seed=32, gaps=(2, 1))
    w = Weigh(gpu, p, 18, seen=[c + 5 * s for s, c in enumerate(contexts)])
    w.call()
    gpu.synchronize()
    w.check()
    assert p.fault() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_weights_of_a_chunk_beside_single_tokens(gpu, kind):
    """A sequence of many rows among ones of few, in the kernel for few: its rows' tiles add to a weight one
    after another, each with a rounding of its own (the others have one tile, as the class says of all)."""
    print(f"[case] weigh chunk beside tokens {kind}", flush=True)
    rng = np.random.default_rng(33)
    new, chunk, G = [1] * 20, 170, 4
    contexts = [int(c) for c in rng.integers(1, 300, 20)]
    new.insert(7, chunk)
    contexts.insert(7, 400)
    p = make(kind, new, contexts, dim=128, seed=34)
    w = Weigh(gpu, p, 2 * G)
    pg, sl = slots(p, 7, 400)
    w.off[pg, :, sl] += (chunk * G / 16) * U * np.abs(w.want[pg, :, sl])
    w.call()
    gpu.synchronize()
    w.check()
    assert p.fault() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_weights_of_contexts_shorter_than_their_new_tokens(gpu, kind):
    """Reported, and no harm to other sequences or to slots past that context."""
    for new, contexts, short in (([1, 5, 2], [40, 40, 30], 2), ([50, 50, 50], [60, 90, 75], 30)):
        print(f"[case] weigh short context {new} {kind}", flush=True)
        p = make(kind, new, contexts, page=8, dim=64, seed=35)
        w = Weigh(gpu, p, 4)
        lengths = np.asarray(contexts, np.int32)
        lengths[1] = short
        p.dev["context"].upload(lengths)
        w.call()
        gpu.synchronize()
        assert p.fault() == gpu.KV_FAULT_LENGTH
        weight, position = w.got()
        pg, sl = slots(p, 1, contexts[1])
        assert np.array_equal(weight[pg[short:], :, sl[short:]], p.weight[pg[short:], :, sl[short:]])
        assert np.array_equal(position[pg[short:], :, sl[short:]], p.position[pg[short:], :, sl[short:]])
        # new token i of n has position short - n + i: the slots before `short` are all of new tokens
        assert (position[pg[:short], :, sl[:short]] == np.arange(short)[:, None]).all()
        q, K = ref.decode(w.q, F32)[p.start[1]:p.start[2]], ref.decode(p.rows(1, p.k), p.kind)
        got, want, off = (np.zeros((short, 2)) for _ in range(3))
        got[:] = weight[pg[:short], :, sl[:short]]
        at = np.arange(short - new[1], short)[:, None]
        for h in range(4):
            qh, k, lse = q[:, h * 64:(h + 1) * 64], K[:short, h // 2], w.lse[p.start[1]:p.start[2], h].astype(np.float64)[:, None]
            x, reach = float(w.scale) * (qh @ k.T), float(w.scale) * (np.abs(qh) @ np.abs(k).T)
            g = np.where(np.arange(short) <= at, np.exp(x - lse), 0)
            want[:, h // 2] += g.sum(0)
            off[:, h // 2] += (g * ((64 / 4 + 8) * reach + 5 * np.abs(lse) + 6) * U).sum(0) + (new[1] + 41) * U * g.sum(0)
        assert (np.abs(got - want) <= off).all()
        for x, y, e in ((weight, w.want, w.off), (position, w.want_position, 0)):
            for s in (0, 2):
                pg, sl = slots(p, s, contexts[s])
                assert (np.abs(x[pg, :, sl] - y[pg, :, sl]) <= (e if np.isscalar(e) else e[pg, :, sl])).all()


# ------------------------------------------------------------------- evict --

def rank_key(weight):
    """Ascending sort key of what is wanted least first: NaN, then the weights."""
    w = weight.astype(np.float64) + 0.0
    return np.where(np.isnan(w), -np.inf, np.where(np.isneginf(w), -1e300, w))


def evicted(p, seen, keep, recent):
    """What qk_kv_evict leaves: pools (as stored), weight, position, contexts."""
    stored = {"k": (p.k4 if isinstance(p, Paged4) else p.k).copy(), "v": (p.v4 if isinstance(p, Paged4) else p.v).copy()}
    weight, position, contexts, moved = p.weight.copy(), p.position.copy(), list(p.contexts), 0
    for s, c in enumerate(p.contexts):
        if keep[s] <= 0 or keep[s] >= c:
            continue
        contexts[s] = keep[s]
        pg, sl = slots(p, s, c)
        for h in range(p.kv_heads):
            late = position[pg, h, sl] >= seen[s] - max(recent[s], 0)
            key = np.where(late, np.inf, rank_key(weight[pg, h, sl]))
            key = np.where(~late & np.isposinf(weight[pg, h, sl]), 1e300, key)
            order = np.argsort(-key, kind="stable")
            stays = np.zeros(c, bool)
            stays[order[:keep[s]]] = True
            free = np.flatnonzero(~stays[:keep[s]])
            source = keep[s] + np.flatnonzero(stays[keep[s]:])
            assert len(free) == len(source)
            moved += len(free)
            for to, at in zip(free, source):
                for x in stored.values():
                    y = p.seen(x)
                    y[pg[to], sl[to], h] = y[pg[at], sl[at], h]
                for x in (weight, position):
                    x[pg[to], h, sl[to]] = x[pg[at], h, sl[at]]
    return stored, weight, position, contexts, moved


class Evict:
    def __init__(self, gpu, p, keep, recent, seen=None, max_context=None, weight=None):
        self.gpu, self.p, self.keep, self.recent = gpu, p, keep, recent
        self.seen = list(p.contexts) if seen is None else seen
        p.upload(gpu)
        add_weights(gpu, p, seed=len(keep) + p.dim)
        if weight is not None:
            p.weight = weight(p).astype(np.float32)
        for s, c in enumerate(p.contexts):  # each slot its own position, the last ones in order
            pg, sl = slots(p, s, c)
            older = max(0, c - 20)
            for h in range(p.kv_heads):
                early = p.rng.permutation(max(self.seen[s] - 20, older))[:older]
                p.position[pg, h, sl] = np.concatenate([early, np.arange(self.seen[s] - (c - older), self.seen[s])])
        p.dev["weight"].upload(p.weight)
        p.dev["position"].upload(p.position)
        array = lambda x: gpu.DeviceBuffer.from_array(np.asarray(x, np.int32))  # noqa: E731
        self.d = {"keep": array(keep), "recent": array(recent), "out": array([-5] * len(keep)),
                  "seen": array(seen) if seen is not None else None}
        self.max_context = max(max(p.contexts, default=1), 1) if max_context is None else max_context
        n = gpu.kv_evict_workspace_size(p.cache, p.batch, self.max_context)
        assert n > 0
        self.ws = gpu.DeviceBuffer.from_array(np.full(n, 0x5A, np.uint8))

    def call(self, stream=None):
        p, d = self.p, self.d
        self.gpu.kv_evict(p.cache, p.batch, d["seen"], p.weights, d["keep"], d["recent"], self.max_context, d["out"], self.ws,
                          self.ws.nbytes, stream)

    def stored(self, name):
        p = self.p
        if isinstance(p, Paged4):
            return p.downloaded(name)
        return p.dev[name].download(np.uint16).reshape(p.k.shape)

    def check(self, want=None):
        p = self.p
        stored, weight, position, contexts, moved = want or evicted(p, self.seen, self.keep, self.recent)
        assert self.d["out"].download(np.int32).tolist() == contexts
        for n in "kv":
            assert np.array_equal(self.stored(n), stored[n]), n
        assert np.array_equal(p.dev["weight"].download(np.uint32).reshape(weight.shape), weight.view(np.uint32))
        assert np.array_equal(p.dev["position"].download(np.int32).reshape(position.shape), position)
        return moved


EVICT = {
    "one-over": dict(contexts=[33, 5, 1], keep=[32, 5, 1], recent=[4, 2, 0]),
    "half": dict(contexts=[200, 64, 130], keep=[100, 32, 65], recent=[10, 0, 20], page=24),
    "uneven": dict(contexts=[500, 0, 77, 1500], keep=[20, 8, 0, 1499], recent=[20, 3, 5, 100], page=64),
    "no-budget": dict(contexts=[50, 60], keep=[0, -3], recent=[1, 1]),
    "to-one": dict(contexts=[100, 40], keep=[1, 1], recent=[0, 1], page=7),
    "all-latest": dict(contexts=[64, 30], keep=[10, 10], recent=[50, 1000]),
    "page-1": dict(contexts=[90], keep=[31], recent=[6], page=1),
    "long": dict(contexts=[5000, 3001], keep=[700, 2900], recent=[64, 64], page=256),
    "dropped-before": dict(contexts=[300, 90], keep=[128, 60], recent=[16, 30], seen=[9000, 95]),
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", EVICT)
def test_evictions_move_what_their_definition_says(gpu, name, kind):
    case = dict(EVICT[name])
    keep, recent, seen = case.pop("keep"), case.pop("recent"), case.pop("seen", None)
    for dim, head_major, heads in ((128, False, 2), (64, True, 3)):
        print(f"[case] evict {name} {kind} dim={dim}", flush=True)
        p = make(kind, [0] * len(keep), dim=dim, head_major=head_major, kv_heads=heads, seed=len(name), **case)
        p.batch_tokens = 0
        e = Evict(gpu, p, keep, recent, seen)
        e.call()
        gpu.synchronize()
        moved = e.check()
        assert p.fault() == 0
        assert (moved > 0) == (name not in ("no-budget",)) or name == "one-over"


WEIGHTS = {
    "ties": lambda p: np.round(p.weight),
    "all-alike": lambda p: np.full(p.weight.shape, 0.5),
    "zeros-of-both-signs": lambda p: np.where(p.weight > 1, 0.0, -0.0),
    "negative": lambda p: p.weight - 1,
    "infinite-and-nan": lambda p: np.where(p.weight > 2, np.inf, np.where(p.weight < 0.4, np.nan, np.where(p.weight < 0.6, -np.inf, p.weight))),
    "tiny": lambda p: p.weight * 1e-44,
    "alike-in-their-high-bits": lambda p: (np.float32(1.0).view(np.uint32) + (p.weight * 1000).astype(np.uint32)).view(np.float32),
}


@pytest.mark.parametrize("name", WEIGHTS)
def test_ties_and_odd_weights(gpu, name):
    p = Paged([0, 0], [700, 90], dim=64, page=24, kv_heads=3, seed=4)
    e = Evict(gpu, p, [300, 41], [9, 5], weight=WEIGHTS[name])
    e.call()
    gpu.synchronize()
    e.check()


def test_sequences_that_cannot_be_cut_stay_and_are_reported(gpu):
    def fresh():
        p = Paged([0, 0, 0], [90, 80, 70], page=8, dim=64, seed=6)
        return p, Evict(gpu, p, [40, 40, 40], [4, 4, 4])

    p, e = fresh()
    want = evicted(p, e.seen, [40, 0, 40], e.recent)
    bad = p.table.copy()
    bad[1, 9] = p.pages
    p.dev["table"].upload(bad)
    e.call()
    gpu.synchronize()
    assert p.fault() == gpu.KV_FAULT_PAGE
    e.check(want)
    for context, fault in ((-3, "LENGTH"), (91, "LENGTH"), (1 << 30, "LENGTH")):
        p, e = fresh()
        want = evicted(p, e.seen, [40, 0, 40], e.recent)
        p.dev["context"].upload(np.asarray([90, context, 70], np.int32))
        want = (*want[:3], [40, context, 40], want[4])
        e.call()
        gpu.synchronize()
        assert p.fault() & getattr(gpu, "KV_FAULT_" + fault)
        e.check(want)
    p, e = fresh()
    e.max_context = 500
    e.ws = gpu.DeviceBuffer(gpu.kv_evict_workspace_size(p.cache, p.batch, 500))
    want = evicted(p, e.seen, [40, 0, 40], e.recent)
    p.dev["context"].upload(np.asarray([90, 200, 70], np.int32))  # past its table
    e.call()
    gpu.synchronize()
    assert p.fault() == gpu.KV_FAULT_PAGE
    e.check((*want[:3], [40, 200, 40], want[4]))


LONG = {"as-they-come": None, "all-alike": WEIGHTS["all-alike"], "ties": WEIGHTS["ties"]}


@pytest.mark.parametrize("name", LONG)
def test_evictions_of_long_contexts(gpu, name):
    """Every loop over a head's slots takes several turns, and ties are counted on from one to the next."""
    print(f"[case] evict long {name}", flush=True)
    p = Paged([0, 0, 0], [40000, 16385, 70001], dim=64, page=256, kv_heads=2, seed=41)
    e = Evict(gpu, p, [30000, 8000, 11], [500, 20, 3], weight=LONG[name])
    e.call()
    gpu.synchronize()
    assert e.check() > 0
    assert p.fault() == 0


@pytest.mark.parametrize("kind", ["f16", "q4_1"])
def test_evictions_of_many_heads(gpu, kind):
    """A few hundred (sequence, head) units, each of more moves than its workgroups take in a turn."""
    print(f"[case] evict many heads {kind}", flush=True)
    p = make(kind, [0] * 32, [1300 - 2 * s for s in range(32)], dim=64, page=64, kv_heads=8, seed=42)
    e = Evict(gpu, p, [650] * 32, [40] * 32)
    e.call()
    gpu.synchronize()
    assert e.check() > 32 * 8 * 256
    assert p.fault() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_a_prompt_of_which_only_the_last_rows_count(gpu, kind):
    """Slots begin with the call whose new tokens they hold: with -inf for the other rows' logs all of a prompt's
    do, whatever they held, and an eviction goes by what its last rows looked at."""
    for n, count in ((300, 20), (14, 3)):
        print(f"[case] weigh last rows of {n} {kind}", flush=True)
        p = make(kind, [n], [n], dim=64, page=24, seed=43)
        w = Weigh(gpu, p, 4)
        lse = w.lse.copy()
        lse[:n - count] = -np.inf
        w.lsed.upload(lse)
        p.dev["weight"].upload(np.full(p.weight.shape, np.nan, np.float32))
        p.dev["position"].upload(np.full(p.position.shape, 1 << 30, np.int32))
        w.call()
        gpu.synchronize()
        weight, position = w.got()
        pg, sl = slots(p, 0, n)
        assert (position[pg, :, sl] == np.arange(n)[:, None]).all()
        q, K = ref.decode(w.q, F32), ref.decode(p.rows(0, p.k), p.kind)
        want, off = np.zeros((n, 2)), np.zeros((n, 2))
        for h in range(4):
            qh, l = q[n - count:, h * 64:(h + 1) * 64], lse[n - count:, h].astype(np.float64)[:, None]
            reach = float(w.scale) * (np.abs(qh) @ np.abs(K[:, h // 2]).T)
            g = np.where(np.arange(n) <= np.arange(n - count, n)[:, None], np.exp(float(w.scale) * (qh @ K[:, h // 2].T) - l), 0)
            want[:, h // 2] += g.sum(0)
            off[:, h // 2] += (g * ((64 / 4 + 8) * reach + 5 * np.abs(l) + 6) * U).sum(0) + (count + 41) * U * g.sum(0)
        assert (np.abs(weight[pg, :, sl] - want) <= off).all()
        e = Evict(gpu, p, [n // 2], [2])
        e.p.weight, e.p.position = np.nan_to_num(weight), position
        p.dev["weight"].upload(e.p.weight)
        p.dev["position"].upload(e.p.position)
        e.call()
        gpu.synchronize()
        e.check()


def test_captured_weighing_and_eviction(gpu):
    """One captured pair of calls, replayed on changed lengths with eager work in between."""
    p = Paged4([1, 1], [150, 700], dim=128, seed=8)
    w = Weigh(gpu, p, 8, max_context=700)
    array = lambda x: gpu.DeviceBuffer.from_array(np.asarray(x, np.int32))  # noqa: E731
    keep, recent, out = array([64, 600]), array([8, 8]), array([0, 0])
    n = gpu.kv_evict_workspace_size(p.cache, p.batch, 700)
    ws = gpu.DeviceBuffer(n)

    def both(stream=None):
        w.call(stream)
        gpu.kv_evict(p.cache, p.batch, None, p.weights, keep, recent, 700, out, ws, n, stream)

    def state():
        return [p.downloaded("k"), p.downloaded("v"), *w.got(), out.download(np.int32)]

    def reset(contexts):
        p.dev["k"].upload(p.k4), p.dev["v"].upload(p.v4)
        p.dev["weight"].upload(p.weight), p.dev["position"].upload(p.position)
        p.dev["context"].upload(np.asarray(contexts, np.int32))

    stream = gpu.Stream()
    graph = gpu.Graph.capture(stream, lambda: both(stream))
    for i, contexts in enumerate(([150, 700], [70, 20], [64, 601], [150, 700])):
        print(f"[case] weigh and evict replay {i}", flush=True)
        reset(contexts)
        graph.launch(stream)
        stream.synchronize()
        replay = state()
        reset(contexts)
        both()
        gpu.synchronize()
        assert all(np.array_equal(x, y) for x, y in zip(replay, state()))
        assert out.download(np.int32).tolist() == [min(contexts[0], 64), min(contexts[1], 600)]
    graph.destroy()
    stream.destroy()


@pytest.mark.parametrize("kind", KINDS)
def test_a_session_that_is_cut_while_it_goes_on(gpu, kind):
    """Append, attend, weigh and evict step by step: every attention result is that over
    the tokens which the cache holds, and those are the ones that the weights name."""
    H, G, D, P, steps = 2, 4, 64, 16, 40
    p = make(kind, [1, 1], [100, 60], kv_heads=H, dim=D, page=P, seed=11, extra_entries=1)
    p.upload(gpu)
    add_weights(gpu, p)
    rng = np.random.default_rng(3)
    array = lambda x: gpu.DeviceBuffer.from_array(np.asarray(x, np.int32))  # noqa: E731
    floats = lambda n: gpu.DeviceBuffer(4 * n)  # noqa: E731
    keep, recent, out = array([48, 48]), array([8, 8]), array([0, 0])
    seen, context = np.array([100, 60]), np.array([100, 60])
    seen_d = array(seen)
    for s, c in enumerate(context):
        pg, sl = slots(p, s, c)
        p.position[pg, :, sl] = np.arange(c)[:, None]
    p.dev["position"].upload(p.position)
    width = (H * G + 2 * H) * D
    q_out, o, lse = floats(2 * H * G * D), floats(2 * H * G * D), floats(2 * H * G)
    rope = gpu.Rope(eps=1e-6, base=1e4, dims=D)
    attn_ws = gpu.DeviceBuffer.from_array(np.zeros(max(256, gpu.paged_attention_workspace_size(p.cache, p.batch, F32, H * G, 0, 110)), np.uint8))
    weigh_ws = gpu.DeviceBuffer(max(256, gpu.kv_weigh_workspace_size(p.cache, p.batch, F32, H * G, 110)))
    evict_ws = gpu.DeviceBuffer(gpu.kv_evict_workspace_size(p.cache, p.batch, 110))
    keys = {}  # rotated keys by (sequence, position), as they come out of the cache
    for step in range(steps):
        x = gpu.DeviceBuffer.from_array(rng.standard_normal((2, width)).astype(np.float32))
        k_at, v_at = x.ptr + 4 * H * G * D, x.ptr + 4 * (H * G + H) * D
        gpu.kv_append_at(p.cache, p.batch, seen_d, x, width, k_at, width, v_at, width, H * G, rope, q_out, F32)
        gpu.paged_attention(p.cache, p.batch, q_out, F32, H * G * D, H * G, D ** -0.5, 0, 110, o, lse, attn_ws, attn_ws.nbytes)
        gpu.kv_weigh(p.cache, p.batch, seen_d, q_out, F32, H * G * D, H * G, D ** -0.5, lse, 110, p.weights, weigh_ws, weigh_ws.nbytes)
        gpu.synchronize()
        if isinstance(p, Paged4):
            p.k4, p.v4 = p.downloaded("k"), p.downloaded("v")
            p.settle()
        else:
            p.k, p.v = (p.dev[n].download(np.uint16).reshape(p.k.shape) for n in "kv")
        p.contexts = context.tolist()
        q = q_out.download(np.float32).reshape(2, H * G, D).astype(np.float64)
        got = o.download(np.float32).reshape(2, H * G, D)
        position = p.dev["position"].download(np.int32).reshape(p.position.shape)
        weight = p.dev["weight"].download(np.float32).reshape(p.weight.shape)
        for s in range(2):
            K, V = (ref.decode(p.rows(s, pool), p.kind) for pool in (p.k, p.v))
            want = ref.attention(q[s:s + 1], K, V, int(context[s]) - 1, D ** -0.5, 0)[0]
            assert np.abs(got[s] - want[0]).max() <= 1e-4 * np.abs(V).max()
            pg, sl = slots(p, s, int(context[s]))
            at = position[pg, :, sl]
            for h in range(H):  # every slot holds the token that its position names
                assert len(set(at[:, h])) == len(at) and at[:, h].max() == seen[s] - 1
                for j, t in enumerate(at[:, h]):
                    row = K[j, h]
                    assert np.array_equal(keys.setdefault((s, h, int(t)), row), row)
            assert np.isfinite(weight[pg, :, sl]).all()
        gpu.kv_evict(p.cache, p.batch, seen_d, p.weights, keep, recent, 110, out, evict_ws, evict_ws.nbytes)
        gpu.synchronize()
        assert out.download(np.int32).tolist() == [min(int(c), 48) for c in context]
        # (the largest contexts need no more than the pages that they began with)
        context = np.minimum(context, 48) + 1
        seen += 1
        p.dev["context"].upload(context.astype(np.int32))
        seen_d.upload(seen.astype(np.int32))
    assert p.fault() == 0
