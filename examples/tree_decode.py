"""A small decoder with a paged key/value cache: a prompt, then greedy decoding token by
token and, in a fork of the same sequence, by verifying trees of drafted tokens. Both
give the same tokens; the second takes fewer steps.

    python examples/tree_decode.py

Weights are random and the drafts come from a stand-in for a small model (the known
continuation, made wrong now and then, beside branches that are wrong), so only the
arithmetic and the cache's bookkeeping are real. The projections, the per-head norms with
the rotation and the cache write, the attention, the cache's moves and the argmax run on
the GPU; the norms between them, SwiGLU and the residuals run on the host."""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "jalapenos-at-home_amd"))
import mx4hip  # noqa: E402

HIDDEN, LAYERS, Q_HEADS, KV_HEADS, HEAD, FFN, VOCAB = 512, 3, 8, 2, 128, 1024, 2048
PAGE, PAGES, POSITIONS, EPS = 16, 64, 512, 1e-6


def rms_norm(x):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)


class Model:
    def __init__(self, ctx, seed=1):
        self.ctx = ctx

        def weight(i, rows, cols):
            return ctx.synth_weight(seed * 1000 + i, rows, cols, sigma=cols ** -0.5)
        width, kv_width = Q_HEADS * HEAD, KV_HEADS * HEAD
        self.embedding, self.head = weight(0, VOCAB, HIDDEN), weight(10 * LAYERS, VOCAB, HIDDEN)
        self.layers = [dict(qkv=[weight(10 * i + j, rows, HIDDEN) for j, rows in ((1, width), (2, kv_width), (3, kv_width))],
                            o=weight(10 * i + 4, HIDDEN, width), gate_up=[weight(10 * i + j, FFN, HIDDEN) for j in (5, 6)],
                            down=weight(10 * i + 7, HIDDEN, FFN)) for i in range(LAYERS)]
        ones = np.full(HEAD, 0x3f80, np.uint16)  # bf16 1.0
        self.q_norm, self.k_norm = ctx.to_device(ones), ctx.to_device(ones)
        self.rope = ctx.buffer(POSITIONS * HEAD * 4)
        ctx.rope_table(POSITIONS, HEAD, 1e6, self.rope)
        row = KV_HEADS * PAGE * HEAD
        self.k, self.v = (ctx.to_device(np.zeros(LAYERS * PAGES * row, np.uint16)) for _ in range(2))
        self.cache = mx4hip.KvCache(self.k, self.v, LAYERS, PAGES, KV_HEADS, PAGE, HEAD)
        self.pages = mx4hip.Pages(PAGES, PAGE)

    def project(self, x, weights):
        """x . W^T of several weights: device rows of f32."""
        xd = x if isinstance(x, mx4hip.DeviceBuffer) else self.ctx.to_device(np.ascontiguousarray(x, np.float32))
        xtype = mx4hip.F32 if xd is not x else mx4hip.BF16
        m = xd.nbytes // (weights[0].cols * (4 if xtype == mx4hip.F32 else 2))
        out = [self.ctx.buffer(m * w.rows * 4) for w in weights]
        if m <= 32:
            self.ctx.matmul_group(xd.ptr, xtype, m, weights, [y.ptr for y in out])
        else:
            for w, y in zip(weights, out):
                self.ctx.matmul(xd, xtype, m, w, y)
        self.ctx.synchronize()  # (the buffers live no longer than this call's caller)
        return out

    def host(self, y, m):
        return y.download(np.float32).reshape(m, -1)

    def step(self, seq, tokens, depth=None, masks=None):
        """Appends tokens to a sequence; the token that the model puts behind each. depth, masks: of a
        tree (each token's place behind the cached ones, and which of the new ones it sees)."""
        ctx, n = self.ctx, len(tokens)
        cached, _ = self.pages.table(seq)
        copies = self.pages.write(seq, cached, cached + n)
        if copies:  # the last page is another sequence's too
            ctx.cache_copy_pages(self.cache, ctx.to_device(np.array(copies, np.uint32)), len(copies))
            ctx.synchronize()
        _, table = self.pages.table(seq)
        dev = [ctx.to_device(np.array(a, np.uint32)) for a in ([0, n], [cached], table)]
        self.batch, self.batch_arrays = mx4hip.Batch(1, n, n, *dev, len(table)), dev
        positions = None if depth is None else ctx.to_device(np.array(depth, np.uint32) + np.uint32(cached))
        tree = None if masks is None else ctx.to_device(np.array(masks, np.uint64))
        words = 1 if masks is None else len(masks) // n

        rows, ids = ctx.buffer(n * HIDDEN * 2), ctx.to_device(np.array(tokens, np.uint32))
        ctx.embed(self.embedding, ids, n, rows)
        x = (rows.download(np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(n, HIDDEN)
        q, attended = ctx.buffer(n * Q_HEADS * HEAD * 2), ctx.buffer(n * Q_HEADS * HEAD * 2)
        for i, layer in enumerate(self.layers):
            qkv = self.project(rms_norm(x), layer["qkv"])
            ctx.qk_norm_rope(*qkv, mx4hip.F32, 0, Q_HEADS, self.q_norm, self.k_norm, EPS, self.rope, POSITIONS, self.batch,
                             self.cache, i, q, positions)
            ctx.attention(q, Q_HEADS, self.batch, self.cache, i, attended, tree, words)
            x = x + self.host(self.project(attended, [layer["o"]])[0], n)
            gate, up = (self.host(y, n) for y in self.project(rms_norm(x), layer["gate_up"]))
            x = x + self.host(self.project(gate / (1 + np.exp(-gate)) * up, [layer["down"]])[0], n)
        logits = self.project(rms_norm(x), [self.head])[0]
        best = ctx.buffer(n * 4)
        ctx.argmax_rows(logits, n, VOCAB, best)
        return best.download(np.uint32).tolist()

    def keep(self, seq, path):
        """Of the step's new tokens, only these (ascending) stay, behind what was cached."""
        tokens, _ = self.pages.table(seq)
        if path != list(range(len(path))):
            self.ctx.cache_keep(self.cache, self.batch, self.ctx.to_device(np.array(path, np.uint32)),
                                self.ctx.to_device(np.array([len(path)], np.uint32)), len(path))
            self.ctx.synchronize()
        self.pages.trim(seq, tokens - self.batch.tokens + len(path))


def decode(model, seq, last, count):
    """count tokens behind `last`, one a step."""
    out = []
    while len(out) < count:
        last = model.step(seq, [last])[0]
        out.append(last)
    return out


def draft(rng, last, truth, deep=4, wide=2):
    """(tokens, parents) of a tree under `last`: the continuation, with wrong branches beside it."""
    tokens, parents, trunk = [last], [-1], 0
    for true in truth[:deep]:
        branches = rng.integers(0, VOCAB, wide).tolist()
        if rng.random() < 0.75:
            branches[int(rng.integers(wide))] = true
        at = [len(tokens) + i for i in range(wide)]
        tokens += branches
        parents += [trunk] * wide
        trunk = at[branches.index(true)] if true in branches else at[0]
    return tokens, parents


def decode_trees(model, seq, last, truth, rng):
    """(tokens, steps): `truth`'s tokens again, by verifying drafted trees."""
    out, steps = [], 0
    while len(out) < len(truth):
        tokens, parents = draft(rng, last, truth[len(out):])
        depth, masks = [], []
        for i, p in enumerate(parents):  # a token sees its ancestors and itself
            depth.append(depth[p] + 1 if p >= 0 else 0)
            masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        best = model.step(seq, tokens, depth, masks)
        path, node = [0], 0
        while True:  # as far as the drafts are what the model says
            out.append(best[node])
            node = next((i for i, p in enumerate(parents) if p == node and tokens[i] == best[node]), None)
            if node is None or len(out) == len(truth):
                break
            path.append(node)
        model.keep(seq, path)
        last, steps = out[-1], steps + 1
    return out, steps


def main(count=48, prompt=45, seed=3):
    with mx4hip.Context() as ctx:
        rng = np.random.default_rng(seed)
        model = Model(ctx)
        seq = model.pages.open()
        last = model.step(seq, rng.integers(0, VOCAB, prompt).tolist())[-1]
        fork = model.pages.fork(seq)
        plain = decode(model, seq, last, count)
        trees, steps = decode_trees(model, fork, last, plain, rng)
        free = model.pages.free_count()
        for s in (seq, fork):
            model.pages.close_sequence(s)
        model.pages.close()
        return plain, trees, steps, free


if __name__ == "__main__":
    plain, trees, steps, free = main()
    print("token by token:", plain)
    print(f"in {steps} steps of drafted trees:", "the same" if trees == plain else trees)
    print("pages free at the end:", free, "of", PAGES)
    sys.exit(trees != plain)
