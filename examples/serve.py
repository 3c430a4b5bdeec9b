"""Several chat sessions served together: prompts prefilled in one ragged batch,
then one token a session and step, on synthetic weights of the Qwen3-4B layer
shapes. Shows the cache append, the paged attention and the sampler between the
library's projections, and the decode step as one captured graph that serves
every length. With --cache q4_1 the cache takes a third of the memory; with --keep
sessions that grow past so many tokens are cut to those that gathered the most
attention weight and the latest --recent ones, after every step.

    python examples/serve.py --layers 4 --prompts 300 17 1 64 --tokens 32
    python examples/serve.py --layers 4 --prompts 2000 300 --tokens 32 --cache q4_1 --keep 512 --recent 64
"""
from __future__ import annotations

import argparse
import importlib.util
import pathlib
import sys
import time

import numpy as np

ROOT = pathlib.Path(__file__).resolve().parents[1]
HIDDEN, FFN, Q_HEADS, KV_HEADS, HEAD = 2560, 9728, 32, 8, 128
EPS, ROPE_BASE, PAGE = 1e-6, 1e6, 64


def package():
    """The package, whose folder's name is not a Python identifier."""
    if "qk_amd" not in sys.modules:
        path = ROOT / "qwen3-4b-q4_k_m-inference-engine_amd" / "__init__.py"
        spec = importlib.util.spec_from_file_location("qk_amd", path)
        sys.modules["qk_amd"] = module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    sys.modules["qk_amd"].load()
    return sys.modules["qk_amd"]


class Server:
    def __init__(self, qk, layers: int, prompts: list[int], tokens: int, vocabulary: int = 151936, seed: int = 1,
                 cache: str = "f16", keep: int = 0, recent: int = 64):
        self.qk, self.vocabulary, self.sessions, self.keep_tokens = qk, vocabulary, len(prompts), keep
        self.rng = np.random.default_rng(seed)
        q4, q6 = qk.TYPE_Q4_K, qk.TYPE_Q6_K
        shapes = {"q": (q4, HIDDEN, Q_HEADS * HEAD), "k": (q4, HIDDEN, KV_HEADS * HEAD), "v": (q6, HIDDEN, KV_HEADS * HEAD),
                  "o": (q4, Q_HEADS * HEAD, HIDDEN), "gate": (q4, HIDDEN, FFN), "up": (q4, HIDDEN, FFN),
                  "down": (q6, FFN, HIDDEN)}

        def weight(qtype, K, N, at):
            w = qk.DeviceBuffer(N * qk.row_bytes(qtype, K))
            qk.synth_superblocks(w, qtype, N, K, seed * 1000 + at, 2e-4 if qtype == q4 else 1e-4, 2e-3)
            return w, qtype, K, N

        floats = lambda n: qk.DeviceBuffer(4 * n)  # noqa: E731
        ones = lambda n: qk.DeviceBuffer.from_array(np.ones(n, np.float32))  # noqa: E731
        # the cache: pages enough for every session's last token, one table for all layers
        self.held = [-(-(p + tokens) // PAGE) for p in prompts]
        pages = sum(self.held)
        order = self.rng.permutation(pages).astype(np.int32)
        table = np.zeros((self.sessions, max(self.held)), np.int32)
        for s, n in enumerate(self.held):
            table[s, :n] = order[sum(self.held[:s]):][:n]
        self.table = qk.DeviceBuffer.from_array(table)
        self.context = qk.DeviceBuffer(4 * self.sessions)
        self.fault = qk.DeviceBuffer.from_array(np.zeros(1, np.uint32))
        self.layers, self.keep = [], []
        kind = {"f16": qk.TYPE_F16, "bf16": qk.TYPE_BF16, "q4_1": qk.TYPE_Q4_1}[cache]
        values = pages * PAGE * KV_HEADS * HEAD
        pool_bytes = values // qk.Q4_1_VALUES * qk.Q4_1_BYTES if cache == "q4_1" else 2 * values
        for i in range(layers):
            pools = [qk.DeviceBuffer(pool_bytes) for _ in range(2)]
            cache = qk.KVCache(k=pools[0].ptr, v=pools[1].ptr, type=kind, pages=pages, page_size=PAGE,
                               kv_heads=KV_HEADS, head_dim=HEAD, page_stride=PAGE * KV_HEADS * HEAD, token_stride=HEAD,
                               head_stride=PAGE * HEAD, fault=self.fault.ptr)
            norms = {n: ones(d) for n, d in (("attn", HIDDEN), ("ffn", HIDDEN), ("q", HEAD), ("k", HEAD))}
            rope = qk.Rope(q_norm=norms["q"].ptr, k_norm=norms["k"].ptr, eps=EPS, base=ROPE_BASE, dims=HEAD)
            weights = {n: weight(*s, 100 * i + j) for j, (n, s) in enumerate(shapes.items())}
            # what an eviction goes by, of every slot and head (a token's begins when it is met)
            slots = pages * PAGE * KV_HEADS
            gathered = [qk.DeviceBuffer(4 * slots) for _ in range(2)] if keep else None
            evict = qk.KVWeights(weight=gathered[0].ptr, position=gathered[1].ptr) if keep else None
            self.layers.append((weights, norms, rope, cache, evict))
            self.keep += [pools, gathered]
        self.final_norm, self.lm_head = ones(HIDDEN), weight(q6, HIDDEN, vocabulary, 99999)
        # activations of the most rows that a call has
        T = max(sum(prompts), self.sessions)
        self.x, self.n, self.q, self.k, self.v, self.a, self.y, self.h = (
            floats(T * d) for d in (HIDDEN, HIDDEN, Q_HEADS * HEAD, KV_HEADS * HEAD, KV_HEADS * HEAD, Q_HEADS * HEAD,
                                    HIDDEN, FFN))
        self.last = floats(self.sessions * HIDDEN)
        self.lse = floats(T * Q_HEADS)
        self.logits = floats(self.sessions * vocabulary)
        self.ffn_ws = qk.DeviceBuffer.from_array(np.zeros(qk.ffn_workspace_size(), np.uint8))
        self.longest = max(p + tokens for p in prompts)
        self.prefill = self.batch(prompts)
        self.decode = self.batch([1] * self.sessions)
        cache = self.layers[0][3]
        batches = (self.prefill, self.decode)
        need = max(qk.paged_attention_workspace_size(cache, b, qk.TYPE_F32, Q_HEADS, 0, self.longest) for b in batches)
        if keep:
            self.budget, self.latest = (qk.DeviceBuffer.from_array(np.full(self.sessions, n, np.int32)) for n in (keep, recent))
            self.cut = qk.DeviceBuffer(4 * self.sessions)
            self.weigh_ws = qk.DeviceBuffer(max(256, *(qk.kv_weigh_workspace_size(cache, b, qk.TYPE_F32, Q_HEADS, self.longest)
                                                       for b in batches)))
            self.evict_ws = qk.DeviceBuffer(qk.kv_evict_workspace_size(cache, self.decode, self.longest))
        self.attn_ws = qk.DeviceBuffer.from_array(np.zeros(max(need, 256), np.uint8))
        self.sample_ws = qk.DeviceBuffer.from_array(np.zeros(qk.sample_workspace_size(self.sessions, vocabulary), np.uint8))
        # every session samples its own way
        cycle = lambda of, t: qk.DeviceBuffer.from_array(np.resize(np.asarray(of, t), self.sessions))  # noqa: E731
        self.filters = (cycle([0.6, 0.0, 1.0, 0.8], np.float32), cycle([20, 0, 0, 50], np.int32),
                        cycle([0.95, 1.0, 0.9, 1.0], np.float32), cycle([0.0, 0.0, 0.0, 0.05], np.float32))
        self.uniform, self.token = qk.DeviceBuffer(4 * self.sessions), qk.DeviceBuffer(4 * self.sessions)
        # tokens in the cache, and tokens that there have been
        self.lengths, self.counts, self.seen = np.array(prompts, np.int32), np.array(prompts, np.int32), qk.DeviceBuffer(4 * self.sessions)

    def batch(self, new):
        start = self.qk.DeviceBuffer.from_array(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        self.keep.append(start)
        return self.qk.KVBatch(sequences=self.sessions, tokens=sum(new), token_start=start.ptr, context=self.context.ptr,
                               page_table=self.table.ptr, table_stride=max(self.held))

    def embed(self, tokens):
        """Synthetic embeddings of host token ids, uploaded to x."""
        rows = [np.random.default_rng(int(t)).standard_normal(HIDDEN, np.float32) for t in tokens]
        self.x.upload(np.stack(rows))

    def forward(self, batch, stream=None):
        """All layers over the rows in x; nothing is allocated for up to 8 rows."""
        qk, T = self.qk, batch.tokens
        matmul = lambda x, w, y: qk.matmul(x, w[0], w[1], w[2], w[3], y, T, stream)  # noqa: E731
        for w, norms, rope, cache, evict in self.layers:
            qk.rms_norm(self.x, norms["attn"], self.n, T, HIDDEN, EPS, stream)
            if T <= 8:
                qk.matmul_segments(self.n, T, HIDDEN, [(w[n][0], w[n][1], w[n][3], y) for n, y in
                                                       (("q", self.q), ("k", self.k), ("v", self.v))], stream)
            else:
                for n, y in (("q", self.q), ("k", self.k), ("v", self.v)):
                    matmul(self.n, w[n], y)
            width = KV_HEADS * HEAD
            qk.kv_append_at(cache, batch, self.seen, self.q, Q_HEADS * HEAD, self.k, width, self.v, width, Q_HEADS, rope,
                            self.q, qk.TYPE_F32, stream)
            qk.paged_attention(cache, batch, self.q, qk.TYPE_F32, Q_HEADS * HEAD, Q_HEADS, HEAD ** -0.5, 0, self.longest,
                               self.a, self.lse, self.attn_ws, self.attn_ws.nbytes, stream)
            if evict:
                qk.kv_weigh(cache, batch, self.seen, self.q, qk.TYPE_F32, Q_HEADS * HEAD, Q_HEADS, HEAD ** -0.5, self.lse,
                            self.longest, evict, self.weigh_ws, self.weigh_ws.nbytes, stream)
                qk.kv_evict(cache, batch, self.seen, evict, self.budget, self.latest, self.longest, self.cut, self.evict_ws,
                            self.evict_ws.nbytes, stream)
            matmul(self.a, w["o"], self.y)
            qk.residual_add(self.x, self.y, T * HIDDEN, stream)
            qk.rms_norm(self.x, norms["ffn"], self.n, T, HIDDEN, EPS, stream)
            qk.ffn(self.n, None, 0.0, w["gate"][0], w["up"][0], w["gate"][1], w["down"][0], w["down"][1], HIDDEN, FFN,
                   self.h, self.y, T, self.ffn_ws, self.ffn_ws.nbytes, stream)
            qk.residual_add(self.x, self.y, T * HIDDEN, stream)

    def choose(self, rows, stream=None):
        """Logits of `rows` [sessions x HIDDEN] and each session's next token."""
        qk, (w, qtype, K, N) = self.qk, self.lm_head
        qk.rms_norm(rows, self.final_norm, self.last, self.sessions, HIDDEN, EPS, stream)
        qk.matmul(self.last, w, qtype, K, N, self.logits, self.sessions, stream)
        temperature, top_k, top_p, min_p = self.filters
        qk.sample(self.logits, self.sessions, N, N, temperature, top_k, top_p, min_p, self.uniform, self.token, None,
                  self.sample_ws, self.sample_ws.nbytes, stream)

    def next_inputs(self):
        self.uniform.upload(self.rng.random(self.sessions, np.float32))
        self.context.upload(self.lengths)
        self.seen.upload(self.counts)

    def prompt(self, ids):
        """Prompts of all sessions in one ragged batch; the first tokens."""
        self.embed(np.concatenate(ids))
        self.next_inputs()
        self.forward(self.prefill)
        x = self.x.download(np.float32).reshape(-1, HIDDEN)
        ends = np.cumsum([len(i) for i in ids]) - 1
        self.y.upload(x[ends])
        self.choose(self.y)
        self.qk.synchronize()
        return self.token.download(np.uint32)

    def step(self, tokens, graph=None, stream=None):
        """One token a session; `graph` if the step was captured."""
        if self.keep_tokens:  # the step before cut its layers to this
            self.lengths = np.minimum(self.lengths, self.keep_tokens).astype(np.int32)
        self.lengths += 1
        self.counts += 1
        self.embed(tokens)
        self.next_inputs()
        if graph is None:
            self.record(stream)
        else:
            graph.launch(stream)
        self.qk.synchronize(stream)
        return self.token.download(np.uint32)

    def record(self, stream=None):
        self.forward(self.decode, stream)
        self.choose(self.x, stream)


def serve(qk, layers, prompts, tokens, vocabulary=151936, seed=1, captured=True, **cache):
    """Token ids [tokens x sessions] and seconds a decode step; `cache`: its type and budget, see Server."""
    server = Server(qk, layers, prompts, tokens, vocabulary, seed, **cache)
    ids = [server.rng.integers(0, vocabulary, n) for n in prompts]
    out = [server.prompt(ids)]
    stream = graph = None
    if captured:
        if len(prompts) > 8:
            raise ValueError("the captured step serves up to 8 sessions: larger products take a workspace")
        stream = qk.Stream()
        graph = qk.Graph.capture(stream, lambda: server.record(stream))
    started = time.perf_counter()
    while len(out) < tokens:
        out.append(server.step(out[-1], graph, stream))
    seconds = (time.perf_counter() - started) / max(1, tokens - 1)
    qk.kv_check(server.layers[0][3])
    qk.ffn_workspace_check(server.ffn_ws)
    if captured:
        graph.destroy()
        stream.destroy()
    return np.stack(out), seconds, server


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--prompts", type=int, nargs="+", default=[300, 17, 1, 64])
    parser.add_argument("--tokens", type=int, default=32)
    parser.add_argument("--seed", type=int, default=1)
    parser.add_argument("--cache", choices=["f16", "bf16", "q4_1"], default="f16", help="what keys and values are held in")
    parser.add_argument("--keep", type=int, default=0, help="tokens that a session's cache is cut to (0: all)")
    parser.add_argument("--recent", type=int, default=64, help="of these the latest ones, whatever they gathered")
    args = parser.parse_args()
    tokens, seconds, _ = serve(package(), args.layers, args.prompts, args.tokens, seed=args.seed, cache=args.cache,
                               keep=args.keep, recent=args.recent)
    for s, n in enumerate(args.prompts):
        print(f"session {s} ({n} prompt tokens): {' '.join(map(str, tokens[:, s]))}")
    print(f"{seconds * 1e3:.2f} ms a step of {len(args.prompts)} sessions and {args.layers} layers, host work included")


if __name__ == "__main__":
    main()
