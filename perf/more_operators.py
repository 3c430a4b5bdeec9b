"""A smaller key/value cache, as measurable cases: a cache held in 4 bits with the
attention over it, and the eviction of cached tokens by the attention weight that
they have gathered. The operators' plain forms in elementary torch operations, the
library's calls for the same work, and their definitions in 64 bits.

A case's "op" is one of
  append  new tokens' keys and values into a paged cache of Q4_1 blocks (head
          RMSNorm and rotary positions on the way, q rotated too), and their rows
          back out as the values that they stand for: qk_kv_append_at, qk_kv_rows
  attend  attention of the new tokens over such a cache: qk_paged_attention
  weigh   the attention weight that cached tokens get from the new tokens, added
          up a key/value head: qk_kv_weigh
  evict   every sequence cut to the tokens with the most weight and the latest
          ones, in place: qk_kv_evict
Sizes are those of the Qwen3-4B layers (32 query heads, 8 key/value heads of 128,
rotary base 1e6) and generic smaller ones. The lengths of a ragged batch follow from
its case alone.
"""
from __future__ import annotations

import importlib.util
import math
import pathlib
import random
import sys

import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]
DEVICE = "cuda"
own = False
EPS = 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "q4_1": 3, "bf16": 30}
BLOCK, BLOCK_BYTES = 32, 20


def _package():
    """The package, whose folder's name is not a Python identifier."""
    if "qk_amd" not in sys.modules:
        path = ROOT / "qwen3-4b-q4_k_m-inference-engine_amd" / "__init__.py"
        spec = importlib.util.spec_from_file_location("qk_amd", path)
        module = importlib.util.module_from_spec(spec)
        sys.modules["qk_amd"] = module
        spec.loader.exec_module(module)
        module.load()
    return sys.modules["qk_amd"]


def _case(name, op, sequences, new, context, **more):
    return {"name": name, "op": op, "sequences": sequences, "new": new, "context": context, "mix": 1, "q_heads": 32,
            "kv_heads": 8, "dim": 128, "page": 16, "cache": "q4_1", "q": "f32", "head_major": False} | more


def _append(name, sequences, new, context, **more):
    return _case(name, "append", sequences, new, context, dropped=0, rotary=128, interleaved=False, norm=True,
                 base=1e6) | more


def _attend(name, sequences, new, context, **more):
    return _case(name, "attend", sequences, new, context, window=0, lse=False) | more


def _weigh(name, sequences, new, context, **more):
    return _case(name, "weigh", sequences, new, context, dropped=0) | more


def _evict(name, sequences, keep, recent, context, **more):
    return _case(name, "evict", sequences, 1, context, keep=keep, recent=recent, fresh=context // 8, dropped=1000) | more


def listed():
    return [
        # one token of a chat session that has had tokens evicted: the smallest call, one for each layer of every token
        _append("append-1", 1, 1, 1000, dropped=3000),
        # a long prompt in one chunk, behind a long context
        _append("append-4096", 1, 4096, 100000, page=64),
        # one token of a chat session over what was said before
        _attend("attend-1", 1, 1, 1000),
        # a decode step of sixty-four sequences of very different lengths
        _attend("attend-64", 64, 1, 8192),
        # a few sequences of very long contexts, 16-bit queries
        _attend("attend-long", 3, 1, 131072, q="f16", page=64, head_major=True),
        # a chunk of a prompt behind a context, with the log-sums that the weights are formed from
        _attend("attend-chunk", 1, 512, 4096, lse=True),
        # the weights of one chat session's decode step
        _weigh("weigh-1", 1, 1, 1000, dropped=3000),
        # of a decode step of sixty-four sequences
        _weigh("weigh-64", 64, 1, 8192),
        # what the last tokens of a long prompt look at, before it is cut; a 16-bit cache
        _weigh("weigh-last", 1, 63, 32768, cache="f16", page=64),
        # whole prompts of two requests, odd and ragged, of another head layout
        _weigh("weigh-prompts", 2, 2047, 2047, q_heads=28, kv_heads=4, cache="bf16", q="bf16", page=24),
        # a server's sequences cut back to their budget after some hundred steps
        _evict("evict-32", 32, 2048, 128, 2304, cache="f16", page=64),
        # a long prompt cut to an eighth
        _evict("evict-long", 1, 8192, 256, 65536, head_major=True, dropped=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "weigh", "weigh", "weigh", "evict", "evict"])
    most = [work(c) for c in listed() if c["op"] == op]
    most = {m: max(w[m] for w in most) for m in ("bytes", "flops")}
    while True:
        case = _drawn(rng, op)
        if all(work(case)[m] <= most[m] for m in most):
            case.pop("name")
            return case


def _drawn(rng, op):
    q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (28, 4), (14, 2), (8, 8), (9, 3)])
    more = {"q_heads": q_heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128]), "mix": rng.randrange(1000),
            "page": rng.choice([8, 16, 24, 64, 256]), "q": rng.choice(["f32", "f32", "f16"]),
            "head_major": rng.random() < 0.3}
    if op == "append":
        new = rng.choice([1, _log(rng, 2, 4096)])
        sequences = _log(rng, 1, 64 if new == 1 else 8)
        return _append("", sequences, new, new + _log(rng, 1, 100000 // sequences),
                       **more | {"rotary": rng.choice([more["dim"], more["dim"], more["dim"] // 2]), "norm": rng.random() < 0.6,
                                 "interleaved": rng.random() < 0.3, "base": rng.choice([1e4, 5e5, 1e6]),
                                 "dropped": rng.choice([0, 0, _log(rng, 1, 10000)])})
    if op == "evict":
        sequences = _log(rng, 1, 32)
        context = _log(rng, 100, min(65536, 73728 // sequences))
        keep = rng.choice([int(context * rng.uniform(0.05, 0.95)) + 1, max(1, context - rng.randint(1, 300))])
        return _evict("", sequences, keep, rng.randint(0, keep // 2), context,
                      **more | {"cache": rng.choice(["q4_1", "f16", "bf16"]), "q": "f32", "fresh": rng.randint(1, context),
                                "dropped": rng.choice([0, _log(rng, 1, 10000)])})
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "long"])
    if op == "weigh":
        cache = rng.choice(["q4_1", "q4_1", "f16", "bf16"])
        more |= {"cache": cache, "q": "f32" if more["q"] == "f32" else "bf16" if cache == "bf16" else "f16",
                 "dropped": rng.choice([0, 0, _log(rng, 1, 10000)])}
        make = _weigh
    else:
        more |= {"lse": rng.random() < 0.3, "window": rng.choice([0, 0, 0, _log(rng, 10, 4000)])}
        make = _attend
    if kind == "decode":
        sequences = _log(rng, 1, 128)
        return make("", sequences, 1, _log(rng, 1, min(32768, (1 << 19) // sequences)), **more)
    if kind == "long":
        return make("", rng.randint(1, 3), 1, _log(rng, 20000, 131072), **more)
    sequences = _log(rng, 1, 8)
    new = _log(rng, 2, 2047 // sequences)
    return make("", sequences, new, new + _log(rng, 1, 8192 // sequences), **more)


def _lengths(case):
    """New tokens and context (these included) of each sequence; the first has the most."""
    rng, B = random.Random(case["mix"]), case["sequences"]
    new = [case["new"]] + [_log(rng, 1, case["new"]) for _ in range(B - 1)]
    if case["op"] == "evict":  # all near the length at which they are cut, some not there yet
        return new, [case["context"]] + [rng.randint(case["context"] * 3 // 4, case["context"]) for _ in range(B - 1)]
    before = [case["context"] - case["new"]] + [rng.randint(0, case["context"] - case["new"]) for _ in range(B - 1)]
    return new, [n + b for n, b in zip(new, before)]


def _seen(case):
    """(keys that any new token of a sequence sees, pairs of new token and key) summed over the sequences."""
    keys = pairs = 0
    for n, c in zip(*_lengths(case)):
        w = case.get("window") or c
        keys += min(c, w + n - 1)
        full = max(0, min(n, w - (c - n)))  # tokens whose window reaches the first key
        pairs += full * (c - n) + full * (full + 1) // 2 + (n - full) * w
    return keys, pairs


def _row_bytes(case):
    return case["dim"] // BLOCK * BLOCK_BYTES if case["cache"] == "q4_1" else 2 * case["dim"]


def work(case):
    D, Hq, Hkv, row = case["dim"], case["q_heads"], case["kv_heads"], _row_bytes(case)
    new, contexts = _lengths(case)
    tokens = sum(new)
    q_size = 4 if case["q"] == "f32" else 2
    if case["op"] == "append":
        # fp32 q, k, v in; q and the blocks out; the blocks in again and their values out
        return {"bytes": tokens * (D * (4 * (Hq + 2 * Hkv) + q_size * Hq) + 2 * Hkv * (2 * row + 2 * D)),
                "flops": tokens * D * ((Hq + Hkv) * (7 if case["norm"] else 3) + 2 * Hkv * 5)}
    if case["op"] == "evict":
        moved = slots = 0
        for c in contexts:
            keep = min(c, case["keep"])
            late = min(case["recent"], keep, c - keep)  # latest tokens, which stay, behind the budget
            moved += late + (keep - late) * (c - keep - late) / max(1, c - late)
            slots += c
        return {"bytes": Hkv * (8 * slots + moved * (4 * row + 16)), "flops": 2 * Hkv * slots}
    keys, pairs = _seen(case)
    if case["op"] == "weigh":
        return {"bytes": keys * Hkv * (row + 8) + tokens * Hq * (D * q_size + 4) + tokens * Hkv * 4,
                "flops": pairs * Hq * (2 * D + 3)}
    return {"bytes": keys * Hkv * 2 * row + tokens * Hq * D * 2 * q_size + (4 * tokens * Hq if case["lse"] else 0),
            "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------ Q4_1 blocks --

def _to_blocks(x):
    """[.., D] in 32 bits -> the blocks' bytes [.., D / 32 * 20]: 16-bit scale and lowest value, then 16 bytes
    of codes, byte j with value j in its low half and value j + 16 in its high half."""
    x = x.unflatten(-1, (-1, BLOCK))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = low.half()
    span = (high - m.float()).clamp(min=0) / 15
    d = span.half()
    d = (d.view(torch.int16) - (d.float() > span).to(torch.int16)).view(torch.float16)  # rounded towards zero
    inverse = torch.where(d == 0, 0, 1 / d.float())
    code = torch.round((x - m.float()) * inverse).clamp(0, 15)
    broken = ~(low.half().isfinite() & high.half().isfinite() & ~x.isnan().any(-1, keepdim=True))
    code = torch.where(broken, 0, code).to(torch.uint8)
    d, m = torch.where(broken, math.nan, d), torch.where(broken, math.nan, m)
    return torch.cat([d.view(torch.uint8), m.view(torch.uint8), code[..., :16] | code[..., 16:] << 4], -1).flatten(-2)


def _values(blocks):
    """The values that blocks [.., n] stand for: d * code + m, rounded once to F16; in 32 bits."""
    b = blocks.unflatten(-1, (-1, BLOCK_BYTES))
    d, m = b[..., :2].contiguous().view(torch.float16), b[..., 2:4].contiguous().view(torch.float16)
    code = torch.cat([b[..., 4:] & 15, b[..., 4:] >> 4], -1)
    return (d.double() * code + m.double()).half().float().flatten(-2)  # 64 bits: rounded to F16 once


def _read(case, rows):
    """Cached rows as numbers in 32 bits."""
    return _values(rows) if case["cache"] == "q4_1" else rows.float()


# ------------------------------------------------------------------ inputs --

def _randn(rng, *shape):
    return torch.randn(*shape, device=DEVICE, generator=rng)


def _pool(case, pages, rng):
    """One of the cache's two arrays: what is seen as [page, slot, head, dim or a row's bytes]."""
    H, P, D = case["kv_heads"], case["page"], case["dim"]
    x = _randn(rng, *((pages, H, P, D) if case["head_major"] else (pages, P, H, D)))
    x = _to_blocks(x) if case["cache"] == "q4_1" else x.to(DTYPES[case["cache"]])
    return x.permute(0, 2, 1, 3) if case["head_major"] else x


def prepare(case, seed):
    rng = torch.Generator(device=DEVICE)
    rng.manual_seed(seed)
    D, Hq, Hkv, P = case["dim"], case["q_heads"], case["kv_heads"], case["page"]
    new, context = _lengths(case)
    B, T = len(new), sum(new)
    held = [-(-c // P) for c in context]
    pages = sum(held) + 3
    shuffled = torch.randperm(pages, device=DEVICE, generator=rng).to(torch.int32)
    table = torch.zeros(B, max(held), dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = shuffled[at:at + n]
        at += n
    whole = lambda of: torch.tensor(of, dtype=torch.int32, device=DEVICE)  # noqa: E731
    starts = lambda of: whole([sum(of[:b]) for b in range(len(of) + 1)])  # noqa: E731
    s = {"case": case, "table": table, "new": new, "contexts": context, "start": starts(new), "context": whole(context),
         "k_pool": _pool(case, pages, rng), "v_pool": _pool(case, pages, rng),
         "fault": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    q_type = DTYPES[case["q"]]
    if "dropped" in case:  # tokens that the sequences have had, evicted ones among them
        s["seen"] = s["context"] + case["dropped"]
    if case["op"] == "append":
        s |= {"q": _randn(rng, T, Hq, D) * 2, "k": _randn(rng, T, Hkv, D) * 2, "v": _randn(rng, T, Hkv, D),
              "out": torch.empty(T, Hq, D, dtype=q_type, device=DEVICE)}
        for name in ("q_norm", "k_norm"):
            s[name] = 1 + 0.2 * _randn(rng, D) if case["norm"] else None
        for name in ("k_out", "v_out"):
            s[name] = torch.empty(T, Hkv, D, dtype=torch.float16, device=DEVICE)
        return s
    if case["op"] in ("attend", "weigh"):
        s["q"] = (_randn(rng, T, Hq, D) * 1.5).to(q_type)
    if case["op"] == "attend":
        s["out"] = torch.empty(T, Hq, D, dtype=q_type, device=DEVICE)
        s["lse"] = torch.empty(T, Hq, dtype=torch.float32, device=DEVICE) if case["lse"] else None
        return s
    # what the slots' tokens have gathered, a few of them nearly all of it; and the tokens' positions
    weight = (1.5 * _randn(rng, pages, Hkv, P)).exp()
    position = torch.zeros(pages, Hkv, P, dtype=torch.int32, device=DEVICE)
    if case["op"] == "weigh":
        # about what the attention of these rows gives: scores have a spread of 1.5
        visible = torch.cat([torch.arange(c - n + 1, c + 1, device=DEVICE) for n, c in zip(new, context)])
        s["lse"] = (visible[:, None].float().log() + 1.125 + 0.2 * _randn(rng, T, Hq)).contiguous()
        return s | {"weight": weight, "position": position}
    weight = torch.where(weight < 0.3, 0, weight)  # tokens that nothing ever looks at: equal weights
    for b, c in enumerate(context):
        # slots behind `older` hold the latest tokens as they came, the others those of earlier evictions
        older = max(0, c - case["fresh"]) if case["dropped"] else 0
        slot = torch.arange(c, device=DEVICE)
        for h in range(Hkv):
            earlier = torch.randperm(older + case["dropped"], device=DEVICE, generator=rng)[:older]
            at = torch.cat([earlier, torch.arange(older + case["dropped"], c + case["dropped"], device=DEVICE)])
            position[table[b, slot // P].long(), h, slot % P] = at.to(torch.int32)
    s["fresh"] = torch.stack([weight.view(torch.int32), position])
    s["state"] = s["fresh"].clone()
    s["weight"], s["position"] = s["state"][0].view(torch.float32), s["state"][1]
    # half of a larger batch has a larger budget of its own
    budget = [case["keep"] + (case["keep"] // 8 if b % 2 else 0) for b in range(B)]
    kept = [min(c, k) for c, k in zip(context, budget)]
    s |= {"keep": whole(budget), "recent": whole([case["recent"]] * B), "context_out": torch.zeros_like(s["context"]),
          "kept": kept, "kept_start": starts(kept)}
    if case["cache"] == "q4_1":
        for name in ("k_out", "v_out"):
            s[name] = torch.empty(sum(kept), Hkv, D, dtype=torch.float16, device=DEVICE)
    return s


# ------------------------------------------------------------- plain forms --

def _places(start, context, T):
    """Sequence and place in the cache of every new token."""
    t = torch.arange(T, device=DEVICE)
    seq = torch.searchsorted(start, t.to(torch.int32), right=True) - 1
    return seq, t - start[seq + 1] + context[seq]


def _plain_rows(s, pool, start, context, T):
    seq, at = _places(start, context, T)
    P = s["case"]["page"]
    return _values(pool[s["table"][seq, at // P].long(), at % P]).half()


def _plain_append(s):
    case = s["case"]
    r, P = case["rotary"], case["page"]
    T = s["k"].shape[0]
    seq, at = _places(s["start"], s["context"], T)
    position = at + (s["seen"] - s["context"])[seq]
    turn = position.double()[:, None] * case["base"] ** (-torch.arange(0, r, 2, device=DEVICE, dtype=torch.float64) / r)
    cos, sin = turn.cos().float()[:, None], turn.sin().float()[:, None]

    def rotated(x, weight):
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        a, b = a * cos - b * sin, b * cos + a * sin
        out = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([out, x[..., r:]], -1)

    page, slot = s["table"][seq, at // P].long(), at % P
    s["k_pool"][page, slot] = _to_blocks(rotated(s["k"], s["k_norm"]))
    s["v_pool"][page, slot] = _to_blocks(s["v"])
    return {"q": rotated(s["q"], s["q_norm"]).to(s["out"].dtype),
            "k": _plain_rows(s, s["k_pool"], s["start"], s["context"], T),
            "v": _plain_rows(s, s["v_pool"], s["start"], s["context"], T)}


def _plain_scores(s):
    """Scores [sequence, kv head, head of the group, new token, key], -inf where the token does not see the key;
    sequence and number within it of every new token; pages and slots of the keys."""
    case = s["case"]
    D, Hq, Hkv, P = case["dim"], case["q_heads"], case["kv_heads"], case["page"]
    B, N, C, T, G = len(s["new"]), max(s["new"]), max(s["contexts"]), s["q"].shape[0], Hq // Hkv
    j = torch.arange(C, device=DEVICE)
    page, slot = s["table"][:, j // P].long(), (j % P).expand(B, C)
    keys = _read(case, s["k_pool"][page, slot]).permute(0, 2, 3, 1)  # [B, Hkv, D, C]
    seq, at = _places(s["start"], s["context"], T)
    i = torch.arange(T, device=DEVICE) - s["start"][seq]
    q = torch.zeros(B, N, Hq, D, device=DEVICE)
    q[seq, i] = s["q"].float()
    places = torch.full((B, N), -1, dtype=torch.long, device=DEVICE)
    places[seq, i] = at
    hidden = j > places[:, :, None]
    if case.get("window"):
        hidden |= j <= places[:, :, None] - case["window"]
    q = q.view(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, D)
    score = (q @ keys.contiguous()).view(B, Hkv, G, N, C)
    score *= D ** -0.5
    score.masked_fill_(hidden[:, None, None], -math.inf)
    return score, seq, i, page, slot


def _plain_attend(s):
    case = s["case"]
    score, seq, i, page, slot = _plain_scores(s)
    B, Hkv, G, N, C = score.shape
    D = case["dim"]
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    values = _read(case, s["v_pool"][page, slot]).permute(0, 2, 1, 3)  # [B, Hkv, C, D]
    out = (p.view(B, Hkv, G * N, C) @ values.contiguous()).view(B, Hkv, G, N, D) / torch.where(total == 0, 1, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, N, Hkv * G, D)[seq, i].to(s["out"].dtype)
    if not case["lse"]:
        return {"out": out}
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(B, N, Hkv * G)[seq, i]
    return {"out": out, "lse": lse}


def _plain_weigh(s):
    score, seq, i, page, slot = _plain_scores(s)
    B, Hkv, G, N, C = score.shape
    lse = torch.zeros(B, N, Hkv * G, device=DEVICE)
    lse[seq, i] = s["lse"]
    lse = lse.view(B, N, Hkv, G).permute(0, 2, 3, 1)
    got = score.sub_(lse[..., None]).exp_().sum((2, 3))  # [B, Hkv, C]
    j = torch.arange(C, device=DEVICE)
    first = s["context"] - (s["start"][1:] - s["start"][:-1])
    old = (j < first[:, None])[:, None]
    b, h, j = (j < s["context"][:, None])[:, None].expand(B, Hkv, C).nonzero(as_tuple=True)
    at = page[b, j], h, slot[b, j]
    s["weight"][at] = torch.where(old.expand(B, Hkv, C)[b, h, j], s["weight"][at], 0) + got[b, h, j]
    late = j >= first[b]
    at = tuple(x[late] for x in at)
    s["position"][at] = (j + s["seen"][b] - s["context"][b])[late].to(torch.int32)
    return {"weight": s["weight"], "position": s["position"]}


def _plain_evict(s):
    case = s["case"]
    P, Hkv, B, C = case["page"], case["kv_heads"], len(s["contexts"]), max(s["contexts"])
    s["state"].copy_(s["fresh"])
    j = torch.arange(C, device=DEVICE)
    page, slot = s["table"][:, j // P].long(), (j % P).expand(B, C)
    weight = s["weight"][page, :, slot].permute(0, 2, 1)  # [B, Hkv, C]
    position = s["position"][page, :, slot].permute(0, 2, 1)
    rank = torch.where(position >= (s["seen"] - s["recent"])[:, None, None], math.inf, weight)
    rank = torch.where(j < s["context"][:, None, None], rank, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices  # equal ones: the first slot first
    count = torch.minimum(s["keep"], s["context"])[:, None, None]
    stays = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, order, (j < count).expand_as(rank))
    b, h, to = (~stays & (j < count)).nonzero(as_tuple=True)  # free places, and as many tokens behind the budget
    _, _, source = (stays & (j >= count)).nonzero(as_tuple=True)
    for name in ("k_pool", "v_pool"):
        s[name][page[b, to], slot[b, to], h] = s[name][page[b, source], slot[b, source], h]
    for name in ("weight", "position"):
        s[name][page[b, to], h, slot[b, to]] = s[name][page[b, source], h, slot[b, source]]
    context = count[:, 0, 0].to(torch.int32)
    out = {"weight": s["weight"], "position": s["position"], "context": context}
    if case["cache"] != "q4_1":
        return out | {"k": s["k_pool"], "v": s["v_pool"]}
    return out | {n: _plain_rows(s, s[n + "_pool"], s["kept_start"], context, sum(s["kept"])) for n in "kv"}


# ------------------------------------------------------ the library's calls --

def _handles(s):
    """What a program makes once and keeps: the descriptions of its cache and batch, and the workspace."""
    if "handles" in s:
        return s["handles"]
    qk, case = _package(), s["case"]
    pool = s["k_pool"]
    # strides are counted in values: of 4-bit blocks, 32 to 20 bytes
    stride = lambda i: pool.stride(i) * BLOCK // BLOCK_BYTES if case["cache"] == "q4_1" else pool.stride(i)  # noqa: E731
    cache = qk.KVCache(k=pool.data_ptr(), v=s["v_pool"].data_ptr(), type=TYPE_IDS[case["cache"]], pages=pool.shape[0],
                       page_size=case["page"], kv_heads=case["kv_heads"], head_dim=case["dim"], page_stride=stride(0),
                       token_stride=stride(1), head_stride=stride(2), fault=s["fault"].data_ptr())

    def batch(tokens, start, context):
        return qk.KVBatch(sequences=case["sequences"], tokens=tokens, token_start=start.data_ptr(),
                          context=context.data_ptr(), page_table=s["table"].data_ptr(), table_stride=s["table"].stride(0))

    h = {"qk": qk, "cache": cache, "batch": batch(sum(s["new"]), s["start"], s["context"])}
    need, longest = 0, max(s["contexts"])
    if case["op"] == "append":
        h["rope"] = qk.Rope(q_norm=s["q_norm"].data_ptr() if case["norm"] else None,
                            k_norm=s["k_norm"].data_ptr() if case["norm"] else None, eps=EPS, base=case["base"],
                            dims=case["rotary"], interleaved=case["interleaved"])
    elif case["op"] == "attend":
        need = qk.paged_attention_workspace_size(cache, h["batch"], TYPE_IDS[case["q"]], case["q_heads"], case["window"], longest)
    else:
        h["weights"] = qk.KVWeights(weight=s["weight"].data_ptr(), position=s["position"].data_ptr())
        if case["op"] == "weigh":
            need = qk.kv_weigh_workspace_size(cache, h["batch"], TYPE_IDS[case["q"]], case["q_heads"], longest)
        else:
            need = qk.kv_evict_workspace_size(cache, h["batch"], longest)
            h["kept"] = batch(sum(s["kept"]), s["kept_start"], s["context_out"])
    h["workspace"] = torch.zeros(max(need, 256), dtype=torch.uint8, device=DEVICE)
    s["handles"] = h
    return h


def _run_own(s):
    case, stream, h = s["case"], torch.cuda.current_stream().cuda_stream, _handles(s)
    qk, cache, batch, workspace = h["qk"], h["cache"], h["batch"], h["workspace"]
    D, Hq, Hkv, longest, q_type = case["dim"], case["q_heads"], case["kv_heads"], max(s["contexts"]), TYPE_IDS[case["q"]]
    if case["op"] == "append":
        qk.kv_append_at(cache, batch, s["seen"].data_ptr(), s["q"].data_ptr(), Hq * D, s["k"].data_ptr(), Hkv * D,
                        s["v"].data_ptr(), Hkv * D, Hq, h["rope"], s["out"].data_ptr(), q_type, stream)
        qk.kv_rows(cache, batch, s["k_out"].data_ptr(), s["v_out"].data_ptr(), TYPE_IDS["f16"], stream)
        return {"q": s["out"], "k": s["k_out"], "v": s["v_out"]}
    if case["op"] == "attend":
        qk.paged_attention(cache, batch, s["q"].data_ptr(), q_type, Hq * D, Hq, D ** -0.5, case["window"], longest,
                           s["out"].data_ptr(), s["lse"].data_ptr() if case["lse"] else None, workspace.data_ptr(),
                           workspace.numel(), stream)
        return {"out": s["out"], "lse": s["lse"]} if case["lse"] else {"out": s["out"]}
    if case["op"] == "weigh":
        qk.kv_weigh(cache, batch, s["seen"].data_ptr(), s["q"].data_ptr(), q_type, Hq * D, Hq, D ** -0.5,
                    s["lse"].data_ptr(), longest, h["weights"], workspace.data_ptr(), workspace.numel(), stream)
        return {"weight": s["weight"], "position": s["position"]}
    s["state"].copy_(s["fresh"])  # evicted in place: every pass begins with the same weights
    qk.kv_evict(cache, batch, s["seen"].data_ptr(), h["weights"], s["keep"].data_ptr(), s["recent"].data_ptr(), longest,
                s["context_out"].data_ptr(), workspace.data_ptr(), workspace.numel(), stream)
    out = {"weight": s["weight"], "position": s["position"], "context": s["context_out"]}
    if case["cache"] != "q4_1":
        return out | {"k": s["k_pool"], "v": s["v_pool"]}
    qk.kv_rows(cache, h["kept"], s["k_out"].data_ptr(), s["v_out"].data_ptr(), TYPE_IDS["f16"], stream)
    return out | {"k": s["k_out"], "v": s["v_out"]}


def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_weigh, "evict": _plain_evict}[s["case"]["op"]](s)


# ---------------------------------------------- the definitions in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "weigh": _exact_weigh, "evict": _exact_evict}[case["op"]](s, case)


def _exact_quantised(x):
    """x [.., D] in 64 bits -> the values that its blocks stand for, in 64 bits."""
    x = x.reshape(*x.shape[:-1], -1, BLOCK)
    m = x.min(-1, keepdim=True).values.half().double()
    span = torch.relu(x.max(-1, keepdim=True).values - m) / 15
    d = span.half()
    below = (d.view(torch.int16) - 1).view(torch.float16)
    d = torch.where(d.double() > span, below, d).double()
    code = torch.where(d > 0, ((x - m) / torch.where(d > 0, d, 1)).round(), 0).clamp(0, 15)
    return (code * d + m).half().double().reshape(*x.shape[:-2], -1)


def _exact_cached(s, case, name, b):
    """Sequence b's cached rows [context, kv head, dim] in 64 bits."""
    c, P = s["contexts"][b], case["page"]
    rows = s[name][s["table"][b, :-(-c // P)].long()].reshape(-1, case["kv_heads"], s[name].shape[-1])[:c]
    if case["cache"] != "q4_1":
        return rows.double()
    blocks = rows.reshape(-1, BLOCK_BYTES)
    scale = blocks[:, :4].contiguous().view(torch.float16).double()
    bits = blocks[:, 4:].to(torch.int64)
    out = torch.empty(len(blocks), BLOCK, dtype=torch.float64, device=DEVICE)
    out[:, :16], out[:, 16:] = (bits % 16).double(), (bits // 16).double()
    return (out * scale[:, :1] + scale[:, 1:]).half().double().reshape(c, case["kv_heads"], case["dim"])


def _exact_append(s, case):
    D, r = case["dim"], case["rotary"]
    speed = torch.exp(torch.arange(r // 2, device=DEVICE, dtype=torch.float64) * (-2 * math.log(case["base"]) / r))
    pos = torch.cat([torch.arange(c - n, c, device=DEVICE) + case["dropped"] for n, c in zip(s["new"], s["contexts"])])
    spin = torch.polar(torch.ones(len(pos), r // 2, dtype=torch.float64, device=DEVICE), pos[:, None] * speed)[:, None]

    def turned(x, weight):
        y = x.double()
        if weight is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * weight.double()
        out = y.clone()
        first = slice(0, r, 2) if case["interleaved"] else slice(0, r // 2)
        second = slice(1, r, 2) if case["interleaved"] else slice(r // 2, r)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * spin
        out[..., first], out[..., second] = z.real, z.imag
        return out

    return {"q": turned(s["q"], s["q_norm"]), "k": _exact_quantised(turned(s["k"], s["k_norm"])),
            "v": _exact_quantised(s["v"].double())}


def _exact_scores(s, case, b, at, h, K):
    """Scores [new token, key] of query head h of sequence b, whose new tokens begin at row `at`."""
    n, c = s["new"][b], s["contexts"][b]
    pos, key = torch.arange(c - n, c, device=DEVICE)[:, None], torch.arange(c, device=DEVICE)
    seen = (key <= pos) & ((key > pos - case["window"]) if case.get("window") else (key >= 0))
    x = s["q"][at:at + n, h].double() @ K[:, h // (case["q_heads"] // case["kv_heads"])].T.contiguous()
    return torch.where(seen, x / math.sqrt(case["dim"]), -math.inf)


def _exact_attend(s, case):
    G = case["q_heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    lse, at = torch.empty(out.shape[:2], dtype=torch.float64, device=DEVICE), 0
    for b, n in enumerate(s["new"]):
        K, V = (_exact_cached(s, case, name, b) for name in ("k_pool", "v_pool"))
        for h in range(case["q_heads"]):
            x = _exact_scores(s, case, b, at, h, K)
            lse[at:at + n, h] = torch.logsumexp(x, -1)
            out[at:at + n, h] = torch.exp(x - lse[at:at + n, h, None]) @ V[:, h // G].contiguous()
        at += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_weigh(s, case):
    P, G, at = case["page"], case["q_heads"] // case["kv_heads"], 0
    weight, position = s["weight"].double(), s["position"].clone()
    for b, (n, c) in enumerate(zip(s["new"], s["contexts"])):
        K = _exact_cached(s, case, "k_pool", b)
        slot = torch.arange(c, device=DEVICE)
        page = s["table"][b].long()[slot // P]
        position[page[c - n:], :, slot[c - n:] % P] = (slot[c - n:, None] + case["dropped"]).to(torch.int32)
        weight[page[c - n:], :, slot[c - n:] % P] = 0.0
        for h in range(case["q_heads"]):
            x = _exact_scores(s, case, b, at, h, K)
            weight[page, h // G, slot % P] += torch.exp(x - s["lse"][at:at + n, h, None].double()).sum(0)
        at += n
    return {"weight": weight, "position": position}


def _exact_evict(s, case):
    """A head of a sequence at a time: its tokens listed from the most wanted one on, those that stay set apart."""
    P = case["page"]
    weight, position = s["weight"].double(), s["position"].clone()
    pools = {n: (torch.stack([x for x in s[n + "_pool"]]) if case["cache"] == "q4_1" else s[n + "_pool"].double()) for n in "kv"}
    for b, c in enumerate(s["contexts"]):
        slot = torch.arange(c, device=DEVICE)
        page, keep = s["table"][b].long()[slot // P], s["kept"][b]
        slot = slot % P
        for h in range(case["kv_heads"]):
            late = position[page, h, slot] >= int(s["seen"][b]) - int(s["recent"][b])
            wanted = torch.argsort(-weight[page, h, slot], stable=True)
            wanted = torch.cat([late.nonzero()[:, 0], wanted[~late[wanted]]])[:keep].sort().values
            source = wanted[wanted >= keep]
            free = torch.ones(keep, dtype=torch.bool, device=DEVICE)
            free[wanted[wanted < keep]] = False
            to = free.nonzero()[:, 0]
            for x in (weight, position):
                x[page[to], h, slot[to]] = x[page[source], h, slot[source]]
            for x in pools.values():
                x[page[to], slot[to], h] = x[page[source], slot[source], h]
    out = {"weight": weight, "position": position, "context": torch.tensor(s["kept"], dtype=torch.int32)}
    if case["cache"] != "q4_1":
        return out | pools
    s |= {n + "_pool": x for n, x in pools.items()} | {"contexts": s["kept"]}
    return out | {n: torch.cat([_exact_cached(s, case, n + "_pool", b) for b in range(len(s["kept"]))]) for n in "kv"}
