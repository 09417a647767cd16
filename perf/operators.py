"""The operators between the projections of a decoder step: what is measured.

Four operators over a paged key/value cache, as a serving program with
speculative decoding calls them for every layer of a step (the first two) and
once a step for all layers (the others):

* "rope": per-head norm of q and k, the rotation by position, and k and v
  written to their places in the cache;
* "attention": queries over the cache: single tokens, trees of drafted tokens,
  prompts;
* "copy": pages copied in every layer (a fork's copy on write);
* "keep": the accepted tokens of a drafted tree moved to the front.

Shapes: the heads and widths of the model family the benchmark names (head
size 128, 8 k / v heads, 16 or 32 q heads, 28 or 36 layers) and generic ones.
Lengths of sequences in a batch are spread over a range, as a server sees them.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
THETA = 1e6


def listed():
    middle = {"q_heads": 16, "kv_heads": 8, "head_dim": 128, "page": 16}
    large = {"q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16}
    return [
        # one decoded token of one user: the smallest call of a step, all latency
        {"name": "rope_step", "kind": "rope", **middle, "x": "f32", "seqs": 1, "new": "1-1", "cached": "777-777", "tree": False},
        # a long prompt's projections, as the f32 products come
        {"name": "rope_prompt", "kind": "rope", **large, "x": "f32", "seqs": 1, "new": "4093-4093", "cached": "0-0", "tree": False},
        # one user decoding after a document of some pages
        {"name": "attention_decode", "kind": "attention", **middle, "seqs": 1, "new": "1-1", "cached": "4111-4111", "tree": False},
        # a server's batch of decoding users, short and long
        {"name": "attention_decode_batch", "kind": "attention", **large, "seqs": 32, "new": "1-1", "cached": "100-8000", "tree": False},
        # a drafted tree verified near the end of a long context
        {"name": "attention_tree_long", "kind": "attention", **large, "seqs": 1, "new": "25-25", "cached": "39000-39000", "tree": True},
        # a batch of users whose drafts are verified together, larger pages
        {"name": "attention_tree_batch", "kind": "attention", **large, "page": 64, "seqs": 12, "new": "9-32", "cached": "300-6000", "tree": True},
        # chunks of prompts beside users that decode
        {"name": "attention_chunks", "kind": "attention", **large, "seqs": 6, "new": "1-900", "cached": "0-3500", "tree": False},
        # a whole long prompt: the largest case
        {"name": "attention_prompt", "kind": "attention", **large, "seqs": 1, "new": "8001-8001", "cached": "0-0", "tree": False},
        # one user's last page copied before a fork writes to it
        {"name": "copy_one", "kind": "copy", **middle, "layers": 28, "pages": 64, "count": 1},
        # a batch forked into several samples
        {"name": "copy_batch", "kind": "copy", **large, "layers": 36, "pages": 192, "count": 45},
        # one user's verify step accepted some of a tree
        {"name": "keep_one", "kind": "keep", **middle, "layers": 28, "seqs": 1, "new": "9-9", "cached": "777-777"},
        # a batch's verify steps
        {"name": "keep_batch", "kind": "keep", **large, "layers": 36, "seqs": 24, "new": "16-32", "cached": "40-200"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _span(rng, lo, hi):
    """A range of lengths inside lo..hi: one length, or a spread."""
    a, b = sorted((_log_int(rng, lo, hi), _log_int(rng, lo, hi)))
    return "%d-%d" % (b if rng.random() < 0.3 else a, b)


def _ends(span):
    lo, hi = span.split("-")
    return int(lo), int(hi)


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8])
    return {"q_heads": kv * rng.choice([1, 2, 4, 4, 5, 7, 8]), "kv_heads": kv, "head_dim": rng.choice([64, 128, 128, 256]),
            "page": rng.choice([16, 32, 64, 256])}


def draw(rng):
    kind = rng.choice(["rope", "decode", "tree", "prompt", "attention", "copy", "keep"])
    case = {"kind": kind, **_heads(rng)}
    if kind == "rope":
        tokens = _log_int(rng, 1, 4000 * 32 * 128 // (case["q_heads"] + 16) // case["head_dim"])
        seqs = _log_int(rng, 1, max(1, min(64, tokens)))
        case.update(x=rng.choice(["f32", "bf16"]), seqs=seqs, new=_span(rng, 1, max(1, tokens // seqs)),
                    cached=_span(rng, 1, 4000), tree=tokens // seqs <= 64 and rng.random() < 0.5)
    elif kind == "copy":
        layers = rng.randint(8, 36)
        page_bytes = layers * case["kv_heads"] * case["head_dim"] * case["page"] * 4
        pages = max(8, min(512, (400 << 20) // page_bytes))
        case.update(layers=layers, pages=pages, count=_log_int(rng, 1, min(45, pages // 3)))
    elif kind == "keep":
        # more than one page holds a sequence, but the pools stay of moderate size
        seqs = _log_int(rng, 1, 24)
        case.update(layers=rng.randint(8, 36), seqs=seqs, new=_span(rng, 2, 64), cached=_span(rng, 1, 200), page=rng.choice([16, 32]))
    else:
        heads = case["q_heads"] * max(128, case["head_dim"])
        pairs = 8000 * 8000 * 32 * 128  # rows by keys by head size of a pass, at most
        case["kind"] = "attention"
        if kind == "decode":
            new, cached, seqs = "1-1", _span(rng, 1, 30000), _log_int(rng, 1, 64)
        elif kind == "tree":
            new, cached, seqs = _span(rng, 2, 64), _span(rng, 1, 30000), _log_int(rng, 1, 24)
        elif kind == "prompt":
            n = _log_int(rng, 65, math.isqrt(pairs // heads))
            new, cached, seqs = "%d-%d" % (n, n), "0-0", _log_int(rng, 1, 4)
        else:  # prompts' chunks and decoding users in one batch
            new, cached, seqs = "1-%d" % _log_int(rng, 65, 1500), "0-%d" % _log_int(rng, 2, 6000), _log_int(rng, 2, 8)
        rows, behind = _ends(new)[1], _ends(cached)[1]
        cost = seqs * heads * rows * (behind + rows)
        keys = seqs * (behind + rows) * case["kv_heads"] * case["head_dim"]
        seqs = max(1, min(seqs, int(seqs * pairs / cost), int(seqs * (100 << 20) / keys)))
        case.update(seqs=seqs, new=new, cached=cached, tree=kind == "tree")
    return case


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """New and cached tokens of every sequence, from the case alone (work() has to know them)."""
    rng = random.Random(repr(sorted((key, x) for key, x in case.items() if key != "name")))

    def pick(span):
        lo, hi = _ends(span)
        if lo == 0:
            return rng.choice([0, _log_int(rng, 1, hi)]) if hi else 0
        return _log_int(rng, lo, hi)

    new = [pick(case["new"]) for _ in range(case["seqs"])]
    cached = [pick(case["cached"]) for _ in range(case["seqs"])]
    new[0] = _ends(case["new"])[1]  # the longest is there
    return new, cached


def _trees(new, rng):
    """A random tree for every sequence: each token's mask of the tokens on its path (itself too) and its depth.
    Trees come padded to a fixed size now and then: padding sees nothing of the tree."""
    masks, depths, paths = [], [], []
    for n in new:
        mask, depth, parent = [], [], []
        used = n if n < 8 or rng.random() < 0.7 else n - rng.randint(1, n // 4)
        for j in range(n):
            p = -1 if j == 0 else max(0, j - 1 - int(rng.expovariate(0.5)))
            if j >= used:
                mask.append(0)
                depth.append(0)
                continue
            mask.append((mask[p] if j else 0) | 1 << j)
            depth.append(depth[p] + 1 if j else 0)
            parent.append(p)
        path, j = [], rng.randrange(used // 2, used)
        while j >= 0:
            path.append(j)
            j = parent[j]
        masks += mask
        depths += depth
        paths.append(path[::-1])
    return masks, depths, paths


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _batch(case, seed):
    """The step's tokens and where they live: pages in shuffled order, some of the pool in nobody's use."""
    new, cached = _lengths(case)
    rng = random.Random(seed)
    page = case["page"]
    need = [max(1, -(-(n + c) // page)) for n, c in zip(new, cached)]
    total = sum(need) + max(2, sum(need) // 8)
    order = list(range(total))
    rng.shuffle(order)
    width, table, at = max(need), [], 0
    for n in need:
        table.append(order[at:at + n] + [0] * (width - n))
        at += n
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    s = {"new": new, "cached_list": cached, "pages": total, "start": _ints(start), "cached": _ints(cached), "table": _ints(table),
         "tokens": start[-1], "max_new": max(new)}
    if case.get("tree") or case["kind"] == "keep":
        masks, depths, paths = _trees(new, rng)
        s["tree"] = torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64)).cuda()
        s["positions"] = _ints([cached[i] + d for i, n in enumerate(new) for d in depths[start[i]:start[i] + n]])
        s["paths"] = paths
    return s


def _noise(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, d, hk, page = case["kind"], case["head_dim"], case["kv_heads"], case["page"]
    s = {"case": case}
    if kind == "copy":
        layers, pages, count = case["layers"], case["pages"], case["count"]
        order = list(range(pages))
        random.Random(seed).shuffle(order)
        s["pairs"] = _ints([[order[i], order[count + i]] for i in range(count)])
        s["pages"], s["layers"] = pages, layers
    else:
        s.update(_batch(case, seed))
        s["layers"] = case.get("layers", 2)
    # keys look like rotated, normalised vectors; values are of unit size, channels differing
    shape = (s["layers"], s["pages"], hk, page, d)
    s["k"] = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    s["v"] = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    channel = 0.3 * _noise(g, hk, 1, d)
    for layer in range(s["layers"]):
        s["k"][layer] = 1.2 * _noise(g, *shape[1:])
        s["v"][layer] = _noise(g, *shape[1:]) + channel
    if kind == "rope":
        hq, t = case["q_heads"], s["tokens"]
        x = 0.7 * _noise(g, t, (hq + 2 * hk) * d) * (1 + _noise(g, (hq + 2 * hk) * d).abs())
        x = x.to(torch.float32 if case["x"] == "f32" else torch.bfloat16)
        # one product gives q | k | v side by side: rows of all three
        s["xq"], s["xk"], s["xv"] = x[:, :hq * d], x[:, hq * d:(hq + hk) * d], x[:, (hq + hk) * d:]
        s["q_norm"] = (1 + 0.3 * _noise(g, d)).to(torch.bfloat16)
        s["k_norm"] = (1 + 0.3 * _noise(g, d)).to(torch.bfloat16)
        most = max(n + c for n, c in zip(s["new"], s["cached_list"]))
        angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * \
            THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s["table_rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["q_out"] = torch.empty(t, hq, d, dtype=torch.bfloat16, device="cuda")
    elif kind == "attention":
        s["q"] = (1.2 * _noise(g, s["tokens"], case["q_heads"], d)).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
    elif kind == "keep":
        most = max(len(p) for p in s["paths"])
        s["kept"] = _ints([p + [0] * (most - len(p)) for p in s["paths"]])
        s["kept_count"] = _ints([len(p) for p in s["paths"]])
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ plain forms


def _owner(s):
    """Of every new token: its sequence and its place among the sequence's new ones."""
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(s["start"][1:].long(), t, right=True)
    return seq, t - s["start"].long()[seq]


def _place(s, seq, position):
    """Page and row in it of a sequence's position."""
    page = s["case"]["page"]
    return s["table"].long()[seq, position // page], position % page


def _plain_rope(s):
    case = s["case"]
    d, half = case["head_dim"], case["head_dim"] // 2
    seq, index = _owner(s)
    slot = s["cached"].long()[seq] + index
    position = s["positions"].long() if case["tree"] else slot
    cos, sin = s["table_rope"][position].unsqueeze(1).split(half, -1)

    def turned(x, w):
        x = x.float().unflatten(-1, (-1, d))
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = x.split(half, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)

    page, row = _place(s, seq, slot)
    s["k"][1][page, :, row] = turned(s["xk"], s["k_norm"])
    s["v"][1][page, :, row] = s["xv"].float().unflatten(-1, (-1, d)).to(torch.bfloat16)
    return {"q": turned(s["xq"], s["q_norm"]), "k": s["k"][1], "v": s["v"][1]}


def _plain_attention(s):
    case = s["case"]
    d, hk, group = case["head_dim"], case["kv_heads"], case["q_heads"] // case["kv_heads"]
    new, cached = s["start"].long().diff(), s["cached"].long()
    most, keys = s["max_new"], int(s["table"].shape[1]) * case["page"]
    key = torch.arange(keys, device="cuda")
    i = torch.arange(most, device="cuda")
    # every sequence padded to the longest: [seqs, kv heads, rows, keys]
    page, row = _place(s, torch.arange(case["seqs"], device="cuda")[:, None], key.expand(case["seqs"], -1))
    k = s["k"][1][page, :, row].float().permute(0, 2, 3, 1)
    v = s["v"][1][page, :, row].float().permute(0, 2, 1, 3)
    token = (s["start"].long()[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][token].float().unflatten(2, (hk, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    j = key - cached[:, None]  # [seqs, keys]: a key's place among the new tokens
    if case["tree"]:
        bit = (s["tree"][token][:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1
        sees = (j[:, None, :] < 0) | ((j[:, None, :] < new[:, None, None]) & (bit == 1))
    else:
        sees = j[:, None, :] <= i[:, None]
    sees = sees[:, None, :, None, :].expand(-1, 1, -1, group, -1).flatten(2, 3)
    score = torch.matmul(q, k) * d ** -0.5
    score = score.masked_fill_(~sees, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    out = out.unflatten(2, (most, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    return out[i < new[:, None]].to(torch.bfloat16)


def _plain_copy(s):
    src, dst = s["pairs"].long().unbind(1)
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return {"k": s["k"], "v": s["v"]}


def _plain_keep(s):
    at = torch.arange(s["kept"].shape[1], device="cuda").expand_as(s["kept"])
    live = at < s["kept_count"][:, None]
    seq, at = live.nonzero().unbind(1)
    first = s["cached"].long()[seq]
    sp, sr = _place(s, seq, first + s["kept"].long()[live])
    dp, dr = _place(s, seq, first + at)
    s["k"][:, dp, :, dr] = s["k"][:, sp, :, sr]
    s["v"][:, dp, :, dr] = s["v"][:, sp, :, sr]
    return {"k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------ the framework's operators

_context = None


def _ctx():
    """The process's context, on torch's own stream."""
    global _context
    if _context is None:
        # the package folder's name is no Python identifier; its binding is a module in it
        sys.path.insert(0, os.path.join(os.getcwd(), "jalapenos-at-home_amd"))
        import mx4hip

        _context = mx4hip.Context(0)
        _context.set_stream(torch.cuda.current_stream().cuda_stream or mx4hip.STREAM_LEGACY)
    return _context


def _handles(s):
    """The cache's and the step's descriptors, which a program keeps for all layers' calls."""
    if "handles" not in s:
        import mx4hip

        case = s["case"]
        cache = mx4hip.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), s["layers"], s["pages"], case["kv_heads"], case["page"],
                               case["head_dim"])
        batch = None
        if case["kind"] != "copy":
            batch = mx4hip.Batch(case["seqs"], s["tokens"], s["max_new"], s["start"].data_ptr(), s["cached"].data_ptr(),
                                 s["table"].data_ptr(), s["table"].shape[1])
        s["handles"] = cache, batch
    return s["handles"]


def _own(s):
    case, ctx = s["case"], _ctx()
    cache, batch = _handles(s)
    kind = case["kind"]
    if kind == "rope":
        import mx4hip

        xt = mx4hip.F32 if case["x"] == "f32" else mx4hip.BF16
        ctx.qk_norm_rope(s["xq"].data_ptr(), s["xk"].data_ptr(), s["xv"].data_ptr(), xt, s["xq"].stride(0), case["q_heads"],
                         s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), EPS, s["table_rope"].data_ptr(), s["table_rope"].shape[0],
                         batch, cache, 1, s["q_out"].data_ptr(), s["positions"].data_ptr() if case["tree"] else None)
        return {"q": s["q_out"], "k": s["k"][1], "v": s["v"][1]}
    if kind == "attention":
        ctx.attention(s["q"].data_ptr(), case["q_heads"], batch, cache, 1, s["out"].data_ptr(),
                      tree=s["tree"].data_ptr() if case["tree"] else None)
        return s["out"]
    if kind == "copy":
        ctx.cache_copy_pages(cache, s["pairs"].data_ptr(), case["count"])
    else:
        ctx.cache_keep(cache, batch, s["kept"].data_ptr(), s["kept_count"].data_ptr(), s["kept"].shape[1])
    return {"k": s["k"], "v": s["v"]}


def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "attention": _plain_attention, "copy": _plain_copy, "keep": _plain_keep}[s["case"]["kind"]](s)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    d, hk, hq, page = case["head_dim"], case["kv_heads"], case["q_heads"], case["page"]
    if case["kind"] == "copy":
        return {"bytes": case["count"] * (8 + 2 * case["layers"] * 2 * hk * page * d * 2), "flops": 0}
    new, cached = _lengths(case)
    t = sum(new)
    if case["kind"] == "rope":
        size = 4 if case["x"] == "f32" else 2
        return {"bytes": t * ((hq + 2 * hk) * d * (size + 2) + 4 * d), "flops": t * (hq + hk) * d * 7}
    if case["kind"] == "keep":
        # a path's tokens but the first, which stays in place (trees are as deep as half their logarithm or so, or more)
        moved = sum(max(1, round(math.log2(n))) for n in new)
        return {"bytes": moved * case["layers"] * 2 * hk * d * 2 * 2, "flops": 0}
    keys = sum(n + c for n, c in zip(new, cached))
    inside = t if case["tree"] else sum(n * (n + 1) // 2 for n in new)
    pairs = sum(n * c for n, c in zip(new, cached)) + inside
    return {"bytes": keys * 2 * hk * d * 2 + 2 * t * hq * d * 2, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    d, hk, page = case["head_dim"], case["kv_heads"], case["page"]
    if case["kind"] == "copy":
        k, v = s["k"].double(), s["v"].double()
        for src, dst in s["pairs"].tolist():
            k[:, dst], v[:, dst] = k[:, src].clone(), v[:, src].clone()
        return {"k": k, "v": v}
    table = s["table"].tolist()
    if case["kind"] == "keep":
        k, v = s["k"].double(), s["v"].double()
        for i, path in enumerate(s["paths"]):
            for to, j in enumerate(path):  # a path ascends, so nothing is overwritten before it has moved
                a, b = s["cached_list"][i] + j, s["cached_list"][i] + to
                for x in (k, v):
                    x[:, table[i][b // page], :, b % page] = x[:, table[i][a // page], :, a % page]
        return {"k": k, "v": v}
    if case["kind"] == "rope":
        k, v = s["k"][1].double(), s["v"][1].double()
        places = [(i, s["cached_list"][i] + j) for i, n in enumerate(s["new"]) for j in range(n)]
        position = s["positions"].tolist() if case["tree"] else [p for _, p in places]
        table_rope = s["table_rope"].double()[torch.tensor(position, device="cuda")]
        # the rotation as a product of complex numbers
        unit = torch.complex(table_rope[:, :d // 2], table_rope[:, d // 2:])[:, None]
        made = {}
        for name, weight in (("xq", "q_norm"), ("xk", "k_norm")):
            x = s[name].double().reshape(len(places), -1, d)
            x = x / ((x ** 2).sum(-1, keepdim=True) / d + EPS).sqrt() * s[weight].double()
            x = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * unit
            made[name] = torch.cat([x.real, x.imag], -1)
        at_page = torch.tensor([table[i][p // page] for i, p in places], device="cuda")
        at_row = torch.tensor([p % page for _, p in places], device="cuda")
        k[at_page, :, at_row] = made["xk"]
        v[at_page, :, at_row] = s["xv"].double().reshape(len(places), -1, d)
        return {"q": made["xq"], "k": k, "v": v}
    group = case["q_heads"] // hk
    out = torch.zeros(s["tokens"], case["q_heads"], d, dtype=torch.float64, device="cuda")
    first = 0
    for i, (n, c) in enumerate(zip(s["new"], s["cached_list"])):
        if n == 0:
            continue
        pages = torch.tensor(table[i][:-(-(n + c) // page)], device="cuda")
        sees = torch.ones(n, n + c, dtype=torch.bool, device="cuda")
        if case["tree"]:
            bits = np.array(s["tree"].tolist()[first:first + n], dtype=np.int64).view(np.uint64)
            sees[:, c:] = torch.from_numpy(((bits[:, None] >> np.arange(n, dtype=np.uint64)) & np.uint64(1)).astype(bool)).cuda()
        else:
            sees[:, c:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        some = sees.any(1)
        for h in range(case["q_heads"]):
            kd = s["k"][1][pages, h // group].reshape(-1, d)[:n + c].double()
            vd = s["v"][1][pages, h // group].reshape(-1, d)[:n + c].double()
            score = s["q"][first:first + n, h].double() @ kd.t() / math.sqrt(d)
            weight = torch.softmax(torch.where(sees, score, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))[some], -1)
            out[first:first + n, h][some] = weight @ vd
        first += n
    return out
