"""The cache, attention and sampling steps between the projections of a decode
step, as measurable cases: their plain forms in elementary torch operations,
the library's calls for the same work, and their definitions in 64 bits.

A case's "op" is one of
  append  new tokens' keys and values (head RMSNorm and rotary positions on the
          way, q rotated too) into a paged cache: qk_kv_append
  attend  attention of the new tokens over that cache: qk_paged_attention
  sample  next tokens by temperature, top-k, top-p and min-p from given
          uniforms: qk_sample
Sizes are those of the Qwen3-4B layers (32 query heads, 8 key/value heads of
128, vocabulary 151936, rotary base 1e6) and generic smaller ones. The lengths
of a ragged batch follow from its case alone.
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
VOCABULARY = 151936
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}


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


def _append(name, sequences, new, context, **more):
    return {"name": name, "op": "append", "sequences": sequences, "new": new, "context": context, "mix": 1,
            "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "cache": "f16", "q": "f32", "rotary": 128,
            "interleaved": False, "norm": True, "base": 1e6, "head_major": False} | more


def _attend(name, sequences, new, context, **more):
    return {"name": name, "op": "attend", "sequences": sequences, "new": new, "context": context, "mix": 1,
            "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "cache": "f16", "q": "f32", "window": 0,
            "lse": False, "head_major": False} | more


def _sample(name, rows, vocabulary, **more):
    return {"name": name, "op": "sample", "rows": rows, "vocabulary": vocabulary, "k": 0, "p": 1.0, "min_p": 0.0,
            "temperature": 0.8, "mixed": False} | more


def listed():
    return [
        # one token of a chat session: the smallest call, one for each layer of every token
        _append("append-1", 1, 1, 1000),
        # a decode step of sixty-four sequences, 16-bit queries, pages of 64 with the heads outside
        _append("append-64", 64, 1, 4000, cache="bf16", q="same", page=64, head_major=True),
        # prompts of five requests prefilled together, ragged; a small model with
        # neighbouring pairs, half of the head rotated and no head norm
        _append("append-ragged", 5, 900, 1500, q_heads=14, kv_heads=2, dim=64, rotary=32, interleaved=True,
                norm=False, base=1e4, page=24),
        # a long prompt in one chunk, behind a long context
        _append("append-4096", 1, 4096, 100000, page=64),
        # one token of a chat session over what was said before
        _attend("attend-1", 1, 1, 1000),
        # a decode step of sixty-four sequences of very different lengths
        _attend("attend-64", 64, 1, 8192),
        # a few sequences of very long contexts, 16-bit queries
        _attend("attend-long", 3, 1, 131072, cache="bf16", q="same", page=64, head_major=True),
        # a chunk of a prompt behind a context, with the log-sums that a caller merges parts by
        _attend("attend-chunk", 1, 512, 4096, lse=True),
        # short prompts, decode rows and drafted tokens in one ragged call, sliding window
        _attend("attend-mixed", 12, 300, 3000, q_heads=28, kv_heads=4, window=1000, page=24, q="same"),
        # the largest: a long prompt, odd in its length, behind as long a context
        _attend("attend-4095", 1, 4095, 8190, cache="bf16", q="same", page=64),
        # the next token of one chat session with the filters that chat models recommend
        _sample("sample-1", 1, VOCABULARY, k=20, p=0.95, temperature=0.6),
        # a large batch whose requests have filters of their own
        _sample("sample-200", 200, VOCABULARY, mixed=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "sample", "sample"])
    most = [work(c) for c in listed() if c["op"] == op]
    most = {m: max(w[m] for w in most) for m in ("bytes", "flops")}
    while True:
        case = _drawn(rng, op)
        if all(work(case)[m] <= most[m] for m in most):
            case.pop("name")
            return case


def _drawn(rng, op):
    if op == "sample":
        rows = _log(rng, 1, 200)
        return _sample("", rows, _log(rng, 1000, VOCABULARY), k=rng.choice([0, 1, 7, 40, _log(rng, 2, 1000)]),
                       p=rng.choice([1.0, 0.9, rng.uniform(0.1, 0.999)]), min_p=rng.choice([0.0, 0.0, rng.uniform(0.001, 0.3)]),
                       temperature=round(rng.uniform(0.2, 1.5), 3), mixed=rng.random() < 0.4)
    q_heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (28, 4), (14, 2), (8, 8), (9, 3)])
    more = {"q_heads": q_heads, "kv_heads": kv_heads, "dim": rng.choice([64, 128, 128]), "mix": rng.randrange(1000),
            "page": rng.choice([8, 16, 24, 64, 256]), "cache": rng.choice(["f16", "f16", "bf16"]),
            "q": rng.choice(["f32", "f32", "same"]), "head_major": rng.random() < 0.3}
    if op == "append":
        new = rng.choice([1, _log(rng, 2, 4096)])
        sequences = _log(rng, 1, 64 if new == 1 else 8)
        return _append("", sequences, new, new + _log(rng, 1, 100000 // sequences),
                       **more | {"rotary": rng.choice([more["dim"], more["dim"], more["dim"] // 2]), "norm": rng.random() < 0.6,
                                 "interleaved": rng.random() < 0.3, "base": rng.choice([1e4, 5e5, 1e6])})
    more |= {"lse": rng.random() < 0.3, "window": rng.choice([0, 0, 0, _log(rng, 10, 4000)])}
    kind = rng.choice(["decode", "decode", "chunk", "chunk", "long"])
    if kind == "decode":
        sequences = _log(rng, 1, 128)
        return _attend("", sequences, 1, _log(rng, 1, min(32768, (1 << 19) // sequences)), **more)
    if kind == "long":
        return _attend("", rng.randint(1, 3), 1, _log(rng, 20000, 131072), **more)
    sequences = _log(rng, 1, 8)
    new = _log(rng, 2, 4095 // sequences)
    return _attend("", sequences, new, new + _log(rng, 1, 8192 // sequences), **more)


def _lengths(case):
    """New tokens and context (these included) of each sequence; the first has the most."""
    rng, B = random.Random(case["mix"]), case["sequences"]
    new = [case["new"]] + [_log(rng, 1, case["new"]) for _ in range(B - 1)]
    before = [case["context"] - case["new"]] + [rng.randint(0, case["context"] - case["new"]) for _ in range(B - 1)]
    return new, [n + b for n, b in zip(new, before)]


def _seen(case):
    """(keys that any new token of a sequence sees, pairs of new token and key) summed over the sequences."""
    keys = pairs = 0
    for n, c in zip(*_lengths(case)):
        w = case["window"] or c
        keys += min(c, w + n - 1)
        full = max(0, min(n, w - (c - n)))  # tokens whose window reaches the first key
        pairs += full * (c - n) + full * (full + 1) // 2 + (n - full) * w
    return keys, pairs


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocabulary"]
        # each logit once; the subtraction, the exponential and the running sum
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 3 * n}
    D, Hq, Hkv = case["dim"], case["q_heads"], case["kv_heads"]
    tokens = sum(_lengths(case)[0])
    q_size = 4 if case["q"] == "f32" else 2
    if case["op"] == "append":
        # fp32 q, k, v in; q and the cache's rows out
        return {"bytes": tokens * D * (4 * (Hq + 2 * Hkv) + q_size * Hq + 2 * 2 * Hkv),
                "flops": tokens * D * (Hq + Hkv) * (7 if case["norm"] else 3)}
    keys, pairs = _seen(case)
    return {"bytes": keys * Hkv * D * 2 * 2 + tokens * Hq * D * 2 * q_size + (4 * tokens * Hq if case["lse"] else 0),
            "flops": 4 * pairs * Hq * D}


def _randn(rng, *shape):
    return torch.randn(*shape, device=DEVICE, generator=rng)


def _pool(case, pages, rng):
    """One of the cache's two arrays: what is seen as [page, slot, head, dim]."""
    H, P, D, t = case["kv_heads"], case["page"], case["dim"], DTYPES[case["cache"]]
    if case["head_major"]:
        return _randn(rng, pages, H, P, D).to(t).permute(0, 2, 1, 3)
    return _randn(rng, pages, P, H, D).to(t)


def prepare(case, seed):
    rng = torch.Generator(device=DEVICE)
    rng.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "sample":
        R, V = case["rows"], case["vocabulary"]
        s["logits"] = _randn(rng, R, V) * 2.5  # a body of unlikely tokens and a few likely ones
        likely = torch.randint(0, V, (R, 12), device=DEVICE, generator=rng)
        s["logits"].scatter_(1, likely, 8 + 6 * torch.rand(R, 12, device=DEVICE, generator=rng))
        pick = lambda of, t: torch.tensor(of, dtype=t, device=DEVICE)[  # noqa: E731
            torch.randint(0, len(of), (R,), device=DEVICE, generator=rng)]
        mixed = case["mixed"]
        s["temperature"] = pick([0.0, 0.3, 0.7, 1.0, 1.3] if mixed else [case["temperature"]], torch.float32)
        s["top_k"] = pick([0, 1, 20, 50, 300] if mixed else [case["k"]], torch.int32)
        s["top_p"] = pick([0.5, 0.9, 0.95, 1.0] if mixed else [case["p"]], torch.float32)
        s["min_p"] = pick([0.0, 0.0, 0.05] if mixed else [case["min_p"]], torch.float32)
        s["uniform"] = torch.rand(R, device=DEVICE, generator=rng)
        s["token"] = torch.empty(R, dtype=torch.int32, device=DEVICE)
        s["probability"] = torch.empty(R, dtype=torch.float32, device=DEVICE)
        return s
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
    s |= {"table": table, "new": new, "contexts": context,
          "start": torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=DEVICE),
          "context": torch.tensor(context, dtype=torch.int32, device=DEVICE),
          "k_pool": _pool(case, pages, rng), "v_pool": _pool(case, pages, rng),
          "fault": torch.zeros(1, dtype=torch.int32, device=DEVICE)}
    q_type = DTYPES[case["cache" if case["q"] == "same" else "q"]]
    s["out"] = torch.empty(T, Hq, D, dtype=q_type, device=DEVICE)
    if case["op"] == "append":
        s |= {"q": _randn(rng, T, Hq, D) * 2, "k": _randn(rng, T, Hkv, D) * 2, "v": _randn(rng, T, Hkv, D)}
        for name in ("q_norm", "k_norm"):
            s[name] = 1 + 0.2 * _randn(rng, D) if case["norm"] else None
    else:
        s["q"] = (_randn(rng, T, Hq, D) * 1.5).to(q_type)
        s["lse"] = torch.empty(T, Hq, dtype=torch.float32, device=DEVICE) if case["lse"] else None
    return s


# ------------------------------------------------------------- plain forms --

def _places(s, T):
    """Sequence and position of every new token."""
    t = torch.arange(T, device=DEVICE)
    seq = torch.searchsorted(s["start"], t.to(torch.int32), right=True) - 1
    return seq, t - s["start"][seq + 1] + s["context"][seq]


def _plain_append(s):
    case = s["case"]
    D, r, P = case["dim"], case["rotary"], case["page"]
    seq, pos = _places(s, s["k"].shape[0])
    turn = pos.double()[:, None] * case["base"] ** (-torch.arange(0, r, 2, device=DEVICE, dtype=torch.float64) / r)
    cos, sin = turn.cos().float()[:, None], turn.sin().float()[:, None]

    def rotated(x, weight):
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        a, b = a * cos - b * sin, b * cos + a * sin
        out = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([out, x[..., r:]], -1)

    page, slot = s["table"][seq, pos // P].long(), pos % P
    s["k_pool"][page, slot] = rotated(s["k"], s["k_norm"]).to(s["k_pool"].dtype)
    s["v_pool"][page, slot] = s["v"].to(s["v_pool"].dtype)
    return {"q": rotated(s["q"], s["q_norm"]).to(s["out"].dtype), "k": s["k_pool"], "v": s["v_pool"]}


def _plain_attend(s):
    case = s["case"]
    D, Hq, Hkv, P = case["dim"], case["q_heads"], case["kv_heads"], case["page"]
    B, N, C, T, G = len(s["new"]), max(s["new"]), max(s["contexts"]), s["q"].shape[0], Hq // Hkv
    j = torch.arange(C, device=DEVICE)
    page, slot = s["table"][:, j // P].long(), (j % P).expand(B, C)
    keys = s["k_pool"][page, slot].permute(0, 2, 3, 1).float()    # [B, Hkv, D, C]
    values = s["v_pool"][page, slot].permute(0, 2, 1, 3).float()  # [B, Hkv, C, D]
    seq, pos = _places(s, T)
    i = torch.arange(T, device=DEVICE) - s["start"][seq]
    q = torch.zeros(B, N, Hq, D, device=DEVICE)
    q[seq, i] = s["q"].float()
    at = torch.full((B, N), -1, dtype=torch.long, device=DEVICE)
    at[seq, i] = pos
    hidden = j > at[:, :, None]
    if case["window"]:
        hidden |= j <= at[:, :, None] - case["window"]
    q = q.view(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, D)
    score = (q @ keys.contiguous()).view(B, Hkv, G, N, C)
    score *= D ** -0.5
    score.masked_fill_(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, Hkv, G * N, C) @ values.contiguous()).view(B, Hkv, G, N, D) / torch.where(total == 0, 1, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)[seq, i].to(s["out"].dtype)
    if not case["lse"]:
        return {"out": out}
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(B, N, Hq)[seq, i]
    return {"out": out, "lse": lse}


def _plain_sample(s):
    logits, V = s["logits"], s["logits"].shape[1]
    heat = s["temperature"].double()[:, None]
    z = torch.where(logits.isnan(), -math.inf, logits).double()
    ordered, index = z.sort(dim=-1, descending=True, stable=True)  # 64 bits: the draw's borders
    w = ((ordered - ordered[:, :1]) / torch.where(heat == 0, 1, heat)).exp()
    rank = torch.arange(V, device=DEVICE)
    k = torch.where(s["top_k"] <= 0, V, s["top_k"])[:, None]
    w = torch.where(rank < torch.where(heat == 0, 1, k), w, 0)
    running = w.cumsum(-1)
    p = s["top_p"].double()[:, None]
    w = torch.where((running - w < p * running[:, -1:]) | (p >= 1) | (rank == 0), w, 0)
    w = torch.where((w >= s["min_p"].double()[:, None]) | (rank == 0), w, 0)
    w = torch.zeros_like(w).scatter_(1, index, w)  # in the order of the vocabulary
    running = w.cumsum(-1)
    total = running[:, -1:]
    beyond = running > s["uniform"].double()[:, None] * total
    token = torch.where(beyond & (w > 0), rank, V).amin(-1)
    last = torch.where(w > 0, rank, -1).amax(-1)
    token = torch.where(token == V, last, token)
    share = w.gather(1, token[:, None]) / total
    return {"token": token.to(torch.int32), "probability": share[:, 0].float()}


# ------------------------------------------------------ the library's calls --

def _handles(s):
    """What a program makes once and keeps: the descriptions of its cache and batch, and the workspace."""
    if "handles" in s:
        return s["handles"]
    qk, case = _package(), s["case"]
    if case["op"] == "sample":
        n = qk.sample_workspace_size(case["rows"], case["vocabulary"])
        s["handles"] = (qk, torch.zeros(max(n, 256), dtype=torch.uint8, device=DEVICE))
        return s["handles"]
    pool = s["k_pool"]
    cache = qk.KVCache(k=pool.data_ptr(), v=s["v_pool"].data_ptr(), type=TYPE_IDS[case["cache"]], pages=pool.shape[0],
                       page_size=case["page"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                       page_stride=pool.stride(0), token_stride=pool.stride(1), head_stride=pool.stride(2),
                       fault=s["fault"].data_ptr())
    batch = qk.KVBatch(sequences=case["sequences"], tokens=sum(s["new"]), token_start=s["start"].data_ptr(),
                       context=s["context"].data_ptr(), page_table=s["table"].data_ptr(), table_stride=s["table"].stride(0))
    q_type = TYPE_IDS[case["cache" if case["q"] == "same" else "q"]]
    if case["op"] == "append":
        rope = qk.Rope(q_norm=s["q_norm"].data_ptr() if case["norm"] else None,
                       k_norm=s["k_norm"].data_ptr() if case["norm"] else None, eps=EPS, base=case["base"],
                       dims=case["rotary"], interleaved=case["interleaved"])
        s["handles"] = (qk, cache, batch, rope, q_type)
        return s["handles"]
    n = qk.paged_attention_workspace_size(cache, batch, q_type, case["q_heads"], case["window"], case["context"])
    s["handles"] = (qk, cache, batch, torch.zeros(max(n, 256), dtype=torch.uint8, device=DEVICE), q_type)
    return s["handles"]


def _run_own(s):
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    D, Hq, Hkv = case.get("dim"), case.get("q_heads"), case.get("kv_heads")
    if case["op"] == "append":
        qk, cache, batch, rope, q_type = _handles(s)
        qk.kv_append(cache, batch, s["q"].data_ptr(), Hq * D, s["k"].data_ptr(), Hkv * D, s["v"].data_ptr(), Hkv * D, Hq,
                     rope, s["out"].data_ptr(), q_type, stream)
        return {"q": s["out"], "k": s["k_pool"], "v": s["v_pool"]}
    if case["op"] == "attend":
        qk, cache, batch, workspace, q_type = _handles(s)
        qk.paged_attention(cache, batch, s["q"].data_ptr(), q_type, Hq * D, Hq, D ** -0.5, case["window"],
                           case["context"], s["out"].data_ptr(), s["lse"].data_ptr() if case["lse"] else None,
                           workspace.data_ptr(), workspace.numel(), stream)
        return {"out": s["out"], "lse": s["lse"]} if case["lse"] else {"out": s["out"]}
    qk, workspace = _handles(s)
    qk.sample(s["logits"].data_ptr(), case["rows"], case["vocabulary"], case["vocabulary"], s["temperature"].data_ptr(),
              s["top_k"].data_ptr(), s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["uniform"].data_ptr(),
              s["token"].data_ptr(), s["probability"].data_ptr(), workspace.data_ptr(), workspace.numel(), stream)
    return {"token": s["token"], "probability": s["probability"]}


def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["case"]["op"]](s)


# ---------------------------------------------- the definitions in 64 bits --

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s, case)


def _exact_append(s, case):
    D, r, P = case["dim"], case["rotary"], case["page"]
    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    q_out, at = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE), 0
    speed = torch.exp(torch.arange(r // 2, device=DEVICE, dtype=torch.float64) * (-2 * math.log(case["base"]) / r))
    for b, (n, c) in enumerate(zip(s["new"], s["contexts"])):
        pos = torch.arange(c - n, c, device=DEVICE)
        spin = torch.polar(torch.ones(n, r // 2, dtype=torch.float64, device=DEVICE), pos[:, None] * speed)[:, None]

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

        pages = s["table"][b].long()[pos // P]
        q_out[at:at + n] = turned(s["q"][at:at + n], s["q_norm"])
        k_pool[pages, pos % P] = turned(s["k"][at:at + n], s["k_norm"])
        v_pool[pages, pos % P] = s["v"][at:at + n].double()
        at += n
    return {"q": q_out, "k": k_pool, "v": v_pool}


def _exact_attend(s, case):
    D, P, G = case["dim"], case["page"], case["q_heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    lse, at = torch.empty(out.shape[:2], dtype=torch.float64, device=DEVICE), 0
    for b, (n, c) in enumerate(zip(s["new"], s["contexts"])):
        pages = s["table"][b, :-(-c // P)].long()
        K = s["k_pool"][pages].reshape(-1, case["kv_heads"], D)[:c].double()
        V = s["v_pool"][pages].reshape(-1, case["kv_heads"], D)[:c].double()
        pos = torch.arange(c - n, c, device=DEVICE)[:, None]
        key = torch.arange(c, device=DEVICE)
        seen = (key <= pos) & ((key > pos - case["window"]) if case["window"] else (key >= 0))
        for h in range(case["q_heads"]):
            x = s["q"][at:at + n, h].double() @ K[:, h // G].T.contiguous() / math.sqrt(D)
            x = torch.where(seen, x, -math.inf)
            lse[at:at + n, h] = torch.logsumexp(x, -1)
            out[at:at + n, h] = torch.exp(x - lse[at:at + n, h, None]) @ V[:, h // G].contiguous()
        at += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_sample(s, case):
    """Row by row on the host: the kept set as a list, then the walk along the vocabulary."""
    tokens, shares = [], []
    rows = zip(s["logits"].cpu().double().unbind(), *(s[n].tolist() for n in ("temperature", "top_k", "top_p", "min_p", "uniform")))
    for z, heat, k, p, min_p, u in rows:
        z = z.masked_fill(z.isnan(), -math.inf)
        if heat == 0:
            tokens.append(int(z.argmax()))
            shares.append(1.0)
            continue
        order = torch.argsort(z, descending=True, stable=True)[:k if k > 0 else None]
        w = torch.exp((z[order] - z[order[0]]) / heat)
        if p < 1:
            before = torch.cumsum(w, 0) - w
            count = max(1, int((before < p * w.sum()).sum()))
            order, w = order[:count], w[:count]
        stay = w >= min_p
        stay[0] = True
        order, w = order[stay], w[stay]
        order, back = order.sort()
        w = w[back]
        total = w.sum()
        at = min(int(torch.searchsorted(torch.cumsum(w, 0), u * total, right=True)), len(w) - 1)
        tokens.append(int(order[at]))
        shares.append(float(w[at] / total))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "probability": torch.tensor(shares, dtype=torch.float64)}
