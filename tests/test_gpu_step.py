"""The operators over a paged cache against plain sums in 64 bits.

Tolerances, from the arithmetic: bf16 has 8 significant bits, so a result rounded
once is off by at most U = 2^-8 of itself. Attention's weights are rounded to bf16
too, in the numerator and in the sum that divides it (2 U of the weighted sum of
|v|), and carry the scores' f32 error (head_dim products of a dot, then exp).
Copies are exact."""
import numpy as np
import pytest

from test_gpu_parity import ctx, mx4  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu

NAN_BITS = 0x7fc0
U = 2.0 ** -8


def to_bits(x):
    """f32 to bf16, to nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(NAN_BITS), r)


def from_bits(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


class Step:
    """A call's tokens over a cache of shuffled pages. Every row that holds no
    token is NaN, in k and v, and so are the pages of nobody."""

    def __init__(self, mx4, ctx, rng, new, cached, kv_heads, head_dim, page, layers=1, layer=0, pad_layer=0, spare=3, at=0):
        self.mx4, self.ctx, self.new, self.cached = mx4, ctx, new, cached
        self.hk, self.d, self.page, self.layer = kv_heads, head_dim, page, layer
        need = [-(-(n + c) // page) for n, c in zip(new, cached)]
        self.pages = at + sum(need) + spare
        self.width = max(1, max(need))
        order = at + rng.permutation(sum(need) + spare)
        self.table = np.full((len(new), self.width), self.pages - 1, np.uint32)
        i = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[i:i + n]
            i += n
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.tokens = int(self.start[-1])
        self.row = kv_heads * page * head_dim
        self.stride = self.pages * self.row + pad_layer
        self.layers = layers
        if at == 0:
            size = (layers, self.stride)
            self.kv = [np.full(size, NAN_BITS, np.uint16) for _ in range(2)]
        self.dev = {n: ctx.to_device(np.asarray(a, np.uint32)) for n, a in
                    [("start", self.start), ("cached", cached), ("table", self.table)]}
        self.batch = mx4.Batch(len(new), self.tokens, max(1, max(new)), self.dev["start"], self.dev["cached"], self.dev["table"],
                               self.width)

    def at(self, s, p):
        """Elements of sequence s's position p of every head, [kv_heads, d] indexes of a layer."""
        base = int(self.table[s, p // self.page]) * self.row + (p % self.page) * self.d
        return base + np.arange(self.hk)[:, None] * self.page * self.d + np.arange(self.d)

    def fill(self, rng, past_only=False):
        for x in self.kv:
            for s, (n, c) in enumerate(zip(self.new, self.cached)):
                for p in range(c if past_only else n + c):
                    x[:, self.at(s, p)] = to_bits(rng.standard_normal((self.layers, self.hk, self.d)))
        return self.up()

    def up(self):
        self.k, self.v = (self.ctx.to_device(x) for x in self.kv)
        self.cache = self.mx4.KvCache(self.k, self.v, self.layers, self.pages, self.hk, self.page, self.d, self.stride)
        return self

    def down(self):
        return [b.download(np.uint16).reshape(self.layers, self.stride) for b in (self.k, self.v)]

    def rows(self, s, side):
        """A sequence's keys or values, [positions, kv_heads, d] in 64 bits."""
        n = self.new[s] + self.cached[s]
        out = np.empty((n, self.hk, self.d))
        for p in range(n):
            out[p] = from_bits(self.kv[side][self.layer][self.at(s, p)])
        return out


def reference(step, q, q_heads, sees, scale=None):
    """(outputs, bounds) [tokens, q_heads, d]; sees(s, i) -> which positions token i of sequence s sees."""
    d, group = step.d, q_heads // step.hk
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros((step.tokens, q_heads, d))
    tol = np.zeros_like(out)
    for s in range(len(step.new)):
        k, v = step.rows(s, 0), step.rows(s, 1)
        for i in range(step.new[s]):
            t = step.start[s] + i
            on = sees(s, i)
            if not on.any():
                continue
            for h in range(q_heads):
                kk, vv = k[on, h // group], v[on, h // group]
                x = kk @ q[t, h] * scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[t, h] = w @ vv
                slip = 2 * (d + 4) * 2.0 ** -24 * (np.abs(kk) @ np.abs(q[t, h]) * scale).max() + 2.0 ** -18
                tol[t, h] = U * np.abs(out[t, h]) + (2 * U + 2 * slip) * 1.01 * (w @ np.abs(vv)) + 1e-30
    return out, tol


def chain(step):
    def sees(s, i):
        on = np.zeros(step.new[s] + step.cached[s], bool)
        on[:step.cached[s] + i + 1] = True
        return on
    return sees


def from_masks(step, masks, words):
    def sees(s, i):
        m = masks[(step.start[s] + i) * words:(step.start[s] + i + 1) * words]
        bits = [int(m[j // 64]) >> (j % 64) & 1 for j in range(step.new[s])]
        return np.concatenate([np.ones(step.cached[s], bool), np.array(bits, bool)])
    return sees


def random_tree(rng, step, words, empty=0.1):
    masks = np.zeros((step.tokens, words), np.uint64)
    for s, n in enumerate(step.new):
        for j in range(n):
            if rng.random() < empty:
                continue  # padding: sees nothing of the tree
            parent = int(rng.integers(max(0, j - 4), j)) if j else -1
            row = masks[step.start[s] + j]
            if parent >= 0:
                row |= masks[step.start[s] + parent]
            row[j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return masks


def attend(step, rng, q_heads, masks=None, words=1, scale=0.0, pad=0, amplify=1.0):
    """The operator's outputs as f32 and the queries; rows of q and out `pad` elements apart."""
    ctx = step.ctx
    width = q_heads * step.d
    q = to_bits(amplify * rng.standard_normal((step.tokens, width + pad)))
    if pad:
        q[:, width:] = NAN_BITS
    out = ctx.to_device(np.full((step.tokens, width + pad), 0x1234, np.uint16))
    tree = None if masks is None else ctx.to_device(masks)
    qd = ctx.to_device(q)
    stride = width + pad if pad else 0
    ctx.attention(qd, q_heads, step.batch, step.cache, step.layer, out, tree, words, scale, stride, stride)
    got = out.download(np.uint16).reshape(step.tokens, width + pad)
    assert np.all(got[:, width:] == 0x1234)
    return from_bits(got[:, :width]).reshape(step.tokens, q_heads, step.d), from_bits(q[:, :width]).reshape(
        step.tokens, q_heads, step.d).astype(np.float64)


def near(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:5].tolist(), got[bad][:5], want[bad][:5], tol[bad][:5])


SHAPES = [
    # new tokens, cached tokens, q heads, kv heads, head size, page
    ([1], [0], 1, 1, 64, 16), ([1], [1], 2, 1, 128, 16), ([1], [15], 4, 1, 256, 16), ([1], [16], 8, 8, 64, 32),
    ([1], [31], 5, 1, 128, 16), ([1], [32], 12, 4, 128, 64), ([1], [33], 16, 2, 64, 16), ([1], [4500], 8, 2, 128, 16),
    ([1, 1, 1, 1, 1], [700, 3, 0, 64, 129], 16, 8, 128, 16), ([0, 1, 0, 3, 0], [5, 6, 0, 7, 90], 4, 2, 64, 16),
    ([2], [0], 4, 1, 128, 16), ([5, 9], [100, 0], 20, 4, 128, 16), ([17], [3000], 4, 1, 128, 64), ([16], [50], 8, 2, 256, 128),
    ([33, 1, 40], [3, 2100, 31], 14, 2, 64, 32), ([65], [0], 4, 4, 128, 16), ([130, 3], [77, 400], 8, 2, 128, 16),
    ([300], [0], 3, 1, 128, 256), ([257, 70, 1], [130, 0, 1000], 6, 2, 64, 16), ([90], [5], 16, 2, 256, 16),
    ([3] * 70, list(range(70)), 2, 1, 64, 16),
]


@pytest.mark.parametrize("new,cached,hq,hk,d,page", SHAPES)
def test_attention_chain(mx4, ctx, new, cached, hq, hk, d, page):
    rng = np.random.default_rng(hq * 1000 + d + sum(new) + sum(cached))
    step = Step(mx4, ctx, rng, new, cached, hk, d, page).fill(rng)
    got, q = attend(step, rng, hq)
    near(got, *reference(step, q, hq, chain(step)))


TREES = [([1], [0], 4, 2, 64, 16, 1), ([9], [0], 8, 2, 128, 16, 1), ([9, 1, 5], [40, 0, 18], 8, 8, 64, 16, 1),
         ([32, 17], [900, 31], 8, 2, 128, 32, 1), ([64], [5], 5, 1, 128, 16, 1), ([63, 2, 0, 33], [1, 0, 9, 70], 4, 1, 256, 16, 2),
         ([100], [33], 8, 2, 128, 64, 2), ([7], [5000], 32, 8, 128, 16, 1), ([150, 20], [10, 300], 4, 4, 64, 16, 3)]


@pytest.mark.parametrize("new,cached,hq,hk,d,page,words", TREES)
def test_attention_tree(mx4, ctx, new, cached, hq, hk, d, page, words):
    rng = np.random.default_rng(hq * 77 + d + sum(new) + sum(cached))
    step = Step(mx4, ctx, rng, new, cached, hk, d, page).fill(rng)
    masks = random_tree(rng, step, words)
    got, q = attend(step, rng, hq, masks, words)
    near(got, *reference(step, q, hq, from_masks(step, masks.reshape(-1), words)))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [6, 90])
def test_attention_rows_without_keys_are_zero(mx4, ctx, d, new):
    rng = np.random.default_rng(d + new)
    step = Step(mx4, ctx, rng, [new, 2], [0, 3], 2, d, 16).fill(rng)
    masks = random_tree(rng, step, 2, empty=0.0)
    masks[1] = 0
    masks[new - 1] = 0
    got, q = attend(step, rng, 8, masks, 2)
    assert np.all(got[1] == 0) and np.all(got[new - 1] == 0)
    near(got, *reference(step, q, 8, from_masks(step, masks.reshape(-1), 2)))


@pytest.mark.parametrize("new,cached", [([12], [20]), ([80], [3]), ([12, 100], [0, 64])])
@pytest.mark.parametrize("bad", ["nan_v", "inf_v", "nan_k", "inf_k"])
def test_attention_masked_places_have_no_part(mx4, ctx, new, cached, bad):
    """One new token's key or value is NaN or infinite: whoever does not see it
    is right, whoever does gets what the formula gives."""
    rng = np.random.default_rng(len(bad) + sum(new))
    hq, words = 8, 2
    step = Step(mx4, ctx, rng, new, cached, 2, 128, 16).fill(rng)
    masks = random_tree(rng, step, words, empty=0.0)
    planted = 5
    side = 1 if bad.endswith("v") else 0
    where = step.at(0, cached[0] + planted)[0, 40:43]
    step.kv[side][0][where] = NAN_BITS if bad.startswith("nan") else 0x7f80
    step.up()
    got, q = attend(step, rng, hq, masks, words)
    clean = Step.__new__(Step)
    clean.__dict__.update(step.__dict__)
    clean.kv = [x.copy() for x in step.kv]
    clean.kv[side][0][where] = 0
    want, tol = reference(clean, q, hq, from_masks(step, masks.reshape(-1), words))
    sees = masks[:, 0] >> np.uint64(planted) & np.uint64(1) == 1
    sees[new[0]:] = False
    assert sees.any() and not sees.all()
    hit = np.zeros(got.shape, bool)
    if bad.endswith("v"):
        hit[np.ix_(sees, range(4), range(40, 43))] = True
    else:
        hit[np.ix_(sees, range(4))] = True
    near(got[~hit], want[~hit], tol[~hit])
    if bad == "inf_v":
        assert np.all(got[hit] == np.inf)
    elif bad != "inf_k":  # (an infinite score of either sign: its rows are left to the formula)
        assert np.all(np.isnan(got[hit]))


@pytest.mark.parametrize("new,cached,hq,hk,d,page", [
    # steps whose short and long sequences take different kernels
    ([1, 40, 2, 90, 1, 0, 1, 33] + [1] * 13, [900, 3, 70, 0, 5, 8, 2000, 31] + list(range(13)), 8, 2, 128, 16),
    ([30] + [1] * 20, [500] + [130] * 20, 12, 4, 64, 32), ([1] * 19 + [9, 70], [40] * 20 + [600], 8, 2, 256, 16),
    # more than a wave's lanes: sequences that are cut, and a row's chunks
    ([1, 2] * 40, [300, 0, 10, 1500] * 20, 4, 2, 64, 16), ([40, 30] * 36, [20, 200, 3] * 24, 2, 1, 64, 16),
    ([1], [20000], 8, 1, 128, 16), ([40], [9000], 4, 1, 64, 16),
    # one sequence of more row blocks than the device takes at a time, and beside a longer one
    ([600], [0], 128, 128, 64, 16), ([600, 1], [0, 3000], 64, 64, 64, 16),
    # chunks that have to grow to fit, of more than a wave's lanes; more row blocks than fit, and a long way
    ([40] * 100, [560] * 100, 4, 1, 64, 16), ([600, 1, 500], [0, 3000, 20], 64, 64, 64, 16),
])
def test_attention_batches(mx4, ctx, new, cached, hq, hk, d, page):
    rng = np.random.default_rng(hq * 1000 + d + sum(new) + sum(cached))
    step = Step(mx4, ctx, rng, new, cached, hk, d, page).fill(rng)
    got, q = attend(step, rng, hq)
    near(got, *reference(step, q, hq, chain(step)))


@pytest.mark.parametrize("new,cached,hq,hk,d,page", [(1, 70000, 64, 64, 64, 16), (2, 140003, 64, 32, 128, 16),
                                                   (40, 9001, 64, 64, 64, 16), (70, 20000, 32, 32, 128, 64), (33, 40000, 16, 16, 256, 16)])
def test_attention_long_way_of_one_workgroup(mx4, ctx, new, cached, hq, hk, d, page):
    """Many heads and keys, so that a workgroup walks through many entries of the page table --
    of few pages, each of which many entries name: a key's weight counts as often as it stands there."""
    rng = np.random.default_rng(new + cached)
    pages, entries, group = 37, -(-(new + cached) // page), hq // hk
    kv = [to_bits(rng.standard_normal((pages, hk, page, d))) for _ in range(2)]
    table = rng.integers(0, pages, entries).astype(np.uint32)
    k, v = (ctx.to_device(x) for x in kv)
    dev = [ctx.to_device(np.asarray(x, np.uint32)) for x in ([0, new], [cached], table)]
    q = to_bits(rng.standard_normal((new, hq, d)))
    out = ctx.buffer(q.nbytes)
    ctx.attention(ctx.to_device(q), hq, mx4.Batch(1, new, new, *dev, entries), mx4.KvCache(k, v, 1, pages, hk, page, d), 0, out)
    got = from_bits(out.download(np.uint16)).reshape(q.shape)
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    kf, vf = (from_bits(x).astype(np.float64).transpose(1, 0, 2, 3).reshape(hk, pages * page, d) for x in kv)
    qf = from_bits(q).astype(np.float64)
    for i in range(new):
        at = np.arange(cached + i + 1)
        times = np.bincount(table[at // page].astype(np.int64) * page + at % page, minlength=pages * page)
        for h in range(hq):
            x = kf[h // group] @ qf[i, h] * d ** -0.5
            w = times * np.exp(x - x[times > 0].max())
            w /= w.sum()
            want[i, h] = w @ vf[h // group]
            slip = 2 * (d + 4) * 2.0 ** -24 * (np.abs(kf[h // group]) @ np.abs(qf[i, h]) * d ** -0.5).max() + 2.0 ** -18
            tol[i, h] = U * np.abs(want[i, h]) + (2 * U + 2 * slip) * 1.01 * (w @ np.abs(vf[h // group])) + 1e-30
    near(got, want, tol)


@pytest.mark.parametrize("new,cached", [([12], [20]), ([80], [3]), ([2], [40]), ([12, 100], [131, 94]), ([300], [1000])])
@pytest.mark.parametrize("back", [1, 3])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_attention_cached_values_that_are_not_finite(mx4, ctx, new, cached, back, bad):
    """Every row of the sequence sees the cached keys, also those that stand in a tile with new ones."""
    rng = np.random.default_rng(sum(new) + back)
    step = Step(mx4, ctx, rng, new, cached, 2, 128, 16).fill(rng)
    where = step.at(0, cached[0] - back)[1, 60:62]
    step.kv[1][0][where] = 0
    step.up()
    masks = random_tree(rng, step, 5)
    sees = from_masks(step, masks.reshape(-1), 5)
    _, q = attend(step, np.random.default_rng(8), 4, masks, 5)
    want, tol = reference(step, q, 4, sees)
    step.kv[1][0][where] = to_bits(np.float32(bad))
    step.up()
    got, _ = attend(step, np.random.default_rng(8), 4, masks, 5)
    hit = np.zeros(got.shape, bool)
    hit[:new[0], 2:, 60:62] = True
    near(got[~hit], want[~hit], tol[~hit])
    assert np.array_equal(got[hit], np.full(hit.sum(), bad, np.float32), equal_nan=True)


@pytest.mark.parametrize("new,cached", [([1], [2000]), ([20], [333]), ([150], [0])])
def test_attention_large_scores(mx4, ctx, new, cached):
    """Scores of thousands, and a maximum that grows with every key."""
    rng = np.random.default_rng(5)
    step = Step(mx4, ctx, rng, new, cached, 2, 128, 16).fill(rng)
    got, q = attend(step, rng, 4, amplify=300.0)
    near(got, *reference(step, q, 4, chain(step)))
    for p in range(new[0] + cached[0]):
        step.kv[0][0][step.at(0, p)] = to_bits(np.full((2, 128), 0.02 * (p + 1)))
    step.up()
    q1 = np.ones((step.tokens, 4, 128), np.float32)
    out = ctx.buffer(step.tokens * 4 * 128 * 2)
    ctx.attention(ctx.to_device(to_bits(q1)), 4, step.batch, step.cache, 0, out)
    got = from_bits(out.download(np.uint16)).reshape(q1.shape)
    near(got, *reference(step, q1.astype(np.float64), 4, chain(step)))


@pytest.mark.parametrize("new,cached", [([3, 1], [30, 500]), ([80, 70], [0, 20])])
def test_attention_layers_strides_scale(mx4, ctx, new, cached):
    rng = np.random.default_rng(8)
    step = Step(mx4, ctx, rng, new, cached, 2, 64, 16, layers=3, layer=2, pad_layer=24).fill(rng)
    got, q = attend(step, rng, 6, scale=0.31, pad=16)
    near(got, *reference(step, q, 6, chain(step), 0.31))


def test_attention_same_bits_twice_and_in_a_pass(mx4, ctx):
    """A recorded step follows the lengths in device memory from replay to replay."""
    rng = np.random.default_rng(9)
    step = Step(mx4, ctx, rng, [1, 1, 1], [900, 40, 2999], 2, 128, 16).fill(rng)
    hq = 8
    q = ctx.to_device(to_bits(rng.standard_normal((3, hq * 128))))
    out = ctx.buffer(3 * hq * 128 * 2)
    run = lambda: ctx.attention(q, hq, step.batch, step.cache, 0, out)  # noqa: E731
    run()
    first = out.download(np.uint16)
    run()
    assert np.array_equal(out.download(np.uint16), first)
    recorded = ctx.record(run)
    for cached in ([900, 40, 2999], [5, 40, 0], [899, 17, 1500], [900, 40, 2999]):
        step.dev["cached"].upload(np.array(cached, np.uint32))
        out.upload(np.zeros(3 * hq * 128, np.uint16))
        recorded.launch()
        ctx.synchronize()
        replay = out.download(np.uint16)
        run()
        assert np.array_equal(replay, out.download(np.uint16))
        step.cached = cached
        qf = from_bits(q.download(np.uint16)).reshape(3, hq, 128).astype(np.float64)
        near(from_bits(replay).reshape(3, hq, 128), *reference(step, qf, hq, chain(step)))
    assert np.array_equal(replay, first)
    recorded.release()


def test_attention_on_another_stream(mx4, ctx):
    rng = np.random.default_rng(10)
    step = Step(mx4, ctx, rng, [4], [3000], 2, 128, 16).fill(rng)
    with mx4.Context(0) as other:  # (its stream, and the device's default one)
        ctx.synchronize()
        for stream in (mx4.lib().mx4_get_stream(other.handle), mx4.STREAM_LEGACY):
            ctx.set_stream(stream)
            try:
                got, q = attend(step, rng, 8)
            finally:
                ctx.synchronize()
                ctx.set_stream(None)
            near(got, *reference(step, q, 8, chain(step)))
    got, q = attend(step, rng, 8)
    near(got, *reference(step, q, 8, chain(step)))


def rotated(x, w, eps, position, theta, d):
    x = x.astype(np.float64).reshape(x.shape[0], -1, d)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    half = d // 2
    if theta is not None:
        angle = position[:, None, None] * theta ** (-2.0 * np.arange(half) / d)
        c, s = np.cos(angle), np.sin(angle)
    else:
        c, s = np.ones((1, 1, half)), np.zeros((1, 1, half))
    a, b = x[..., :half], x[..., half:]
    y = np.concatenate([a * c - b * s, b * c + a * s], -1)
    size = np.tile(np.abs(a) + np.abs(b), 2)
    # one rounding to bf16, and f32 in the norm (a sum of d squares), the table and the rotation
    return y, U * np.abs(y) * 1.001 + (d + 16) * 2.0 ** -24 * size + 1e-30


@pytest.mark.parametrize("xt", ["f32", "bf16"])
@pytest.mark.parametrize("new,cached,hq,hk,d,page", [
    ([1], [0], 1, 1, 64, 16), ([1], [777], 16, 8, 128, 16), ([0, 1, 3], [9, 15, 16], 5, 1, 256, 32), ([37], [30], 32, 8, 128, 64),
    ([2] * 100, list(range(100)), 3, 3, 64, 16), ([1100], [3], 2, 1, 128, 16)])
@pytest.mark.parametrize("form", ["plain", "fused", "tree", "bare"])
def test_norm_rotation_and_cache_write(mx4, ctx, xt, new, cached, hq, hk, d, page, form):
    rng = np.random.default_rng(sum(new) + d)
    step = Step(mx4, ctx, rng, new, cached, hk, d, page, layers=2, layer=1, pad_layer=8)
    step.fill(rng, past_only=True)
    t, eps, theta, most = step.tokens, 1e-6, 1e6, max(n + c for n, c in zip(new, cached))
    widths = [hq * d, hk * d, hk * d]
    pad = 16 if form == "fused" else 0
    x = rng.standard_normal((t, sum(widths) + pad)).astype(np.float32) * 3
    if xt == "bf16":
        x = from_bits(to_bits(x))
    enc, size = (to_bits, 2) if xt == "bf16" else (lambda a: np.ascontiguousarray(a, np.float32), 4)
    edges = np.cumsum([0] + widths)
    parts = [x[:, a:b] for a, b in zip(edges, edges[1:])]
    if form == "fused":
        whole = ctx.to_device(enc(x))
        ptrs = [whole.ptr + int(e) * size for e in edges[:3]]
        stride = x.shape[1]
    else:
        bufs = [ctx.to_device(enc(p)) for p in parts]
        ptrs, stride = [b.ptr for b in bufs], 0
    w = [to_bits(1 + 0.5 * rng.standard_normal(d)) for _ in range(2)]
    wd = [ctx.to_device(a) for a in w]
    rope = ctx.buffer(most * d * 4)
    ctx.rope_table(most, d, theta, rope)
    place = np.concatenate([np.arange(c, c + n) for n, c in zip(new, cached)])
    position = rng.integers(0, most, t) if form == "tree" else place
    pd = ctx.to_device(position.astype(np.uint32)) if form == "tree" else None
    bare = form == "bare"
    out_pad = 8 if form == "fused" else 0
    out = ctx.to_device(np.full((t, hq * d + out_pad), 0x1234, np.uint16))
    ctx.qk_norm_rope(*ptrs, mx4.BF16 if xt == "bf16" else mx4.F32, stride, hq, None if bare else wd[0], None if bare else wd[1],
                     eps, None if bare else rope, most, step.batch, step.cache, 1, out, pd, hq * d + out_pad if out_pad else 0)
    got = out.download(np.uint16).reshape(t, -1)
    assert np.all(got[:, hq * d:] == 0x1234)
    args = (eps, position, None if bare else theta, d)
    near(from_bits(got[:, :hq * d]).reshape(t, hq, d), *rotated(parts[0], None if bare else from_bits(w[0]), *args))
    k, ktol = rotated(parts[1], None if bare else from_bits(w[1]), *args)
    after = step.down()
    want_v = to_bits(parts[2].reshape(t, hk, d))
    for s in range(len(new)):
        for i in range(new[s]):
            at, token = step.at(s, cached[s] + i), step.start[s] + i
            near(from_bits(after[0][1][at]), k[token], ktol[token])
            assert np.array_equal(after[1][1][at], want_v[token])
            for side in (0, 1):
                after[side][1][at] = step.kv[side][1][at]
    # nothing else was written
    assert np.array_equal(after[0], step.kv[0]) and np.array_equal(after[1], step.kv[1])


@pytest.mark.parametrize("positions,d,theta", [(1, 64, 1e4), (300, 128, 1e6), (41000, 128, 1e6), (5, 2, 500.0)])
def test_rope_table(mx4, ctx, positions, d, theta):
    out = ctx.buffer(positions * d * 4)
    ctx.rope_table(positions, d, theta, out)
    angle = np.arange(positions)[:, None] * theta ** (-2.0 * np.arange(d // 2) / d)
    want = np.concatenate([np.cos(angle), np.sin(angle)], 1)
    # one rounding to f32; an angle of up to 2^16 in 64 bits is off by 2^-36 or so
    assert np.abs(out.download(np.float32).reshape(want.shape) - want).max() <= 2.0 ** -24 + 2.0 ** -34


@pytest.mark.parametrize("layers,hk,d,page,pages,count", [(1, 1, 64, 16, 2, 1), (3, 2, 128, 16, 9, 4), (2, 3, 256, 64, 30, 15), (40, 1, 64, 16, 5, 2)])
def test_copy_pages(mx4, ctx, layers, hk, d, page, pages, count):
    rng = np.random.default_rng(pages)
    row = hk * page * d
    stride = pages * row + 8
    kv = [rng.integers(0, 65536, (layers, stride), dtype=np.uint16) for _ in range(2)]
    dev = [ctx.to_device(x) for x in kv]
    cache = mx4.KvCache(dev[0], dev[1], layers, pages, hk, page, d, stride)
    order = rng.permutation(pages)
    pairs = [(order[i], order[count + i]) for i in range(count)]
    extra = [(pages, pairs[0][0]), (pairs[0][0], pages), (2 ** 32 - 1, 2 ** 32 - 1)]  # past the cache: left out
    ctx.cache_copy_pages(cache, ctx.to_device(np.array(pairs + extra, np.uint32)), count + len(extra))
    for x in kv:
        for a, b in pairs:
            x[:, b * row:(b + 1) * row] = x[:, a * row:(a + 1) * row]
    for x, b in zip(kv, dev):
        assert np.array_equal(b.download(np.uint16).reshape(x.shape), x)
    ctx.cache_copy_pages(cache, None, 0)


@pytest.mark.parametrize("new,cached,kept,hk,d,page", [
    ([1], [0], [[0]], 1, 64, 16), ([9], [10], [[0, 2, 3, 8]], 8, 128, 16), ([9], [14], [[1, 2, 3, 4, 5, 6, 7, 8]], 2, 64, 16),
    ([0, 5, 64, 3], [7, 16, 31, 0], [[], [0, 4], list(range(0, 64, 2)), [2]], 3, 128, 16),
    ([200], [5], [list(range(1, 200))], 2, 256, 32), ([70, 70], [0, 90], [list(range(30, 70)), [69]], 5, 128, 64),
    ([4, 3] * 50, list(range(100)), [[0, 2, 3], [1]] * 50, 5, 64, 16)])
def test_keep(mx4, ctx, new, cached, kept, hk, d, page):
    rng = np.random.default_rng(sum(new))
    step = Step(mx4, ctx, rng, new, cached, hk, d, page, layers=3, pad_layer=8).fill(rng)
    most = max(1, max(map(len, kept))) + 1
    lists = np.full((len(new), most), 7777, np.uint32)  # past a list's count, and no new token: left out
    counts = np.array([len(x) for x in kept], np.uint32)
    for s, x in enumerate(kept):
        lists[s, :len(x)] = x
        if len(x) + 1 <= new[s]:
            counts[s] += 1
    ctx.cache_keep(step.cache, step.batch, ctx.to_device(lists), ctx.to_device(counts), most)
    for x in step.kv:
        for s, path in enumerate(kept):
            rows = [x[:, step.at(s, cached[s] + j)].copy() for j in path]
            for j, r in enumerate(rows):
                x[:, step.at(s, cached[s] + j)] = r
    for side, x in zip(step.down(), step.kv):
        assert np.array_equal(side, x)


def test_a_recorded_step(mx4, ctx):
    """Norms, rotation, attention, kept tokens and a page copy in one pass: each replay gives what the
    calls give, with the lengths, lists and pairs that the device holds then."""
    rng = np.random.default_rng(21)
    hq, hk, d, page = 8, 2, 128, 16
    step = Step(mx4, ctx, rng, [9, 30], [200, 31], hk, d, page, layers=2, layer=1).fill(rng)
    rows = rng.standard_normal((step.tokens, (hq + 2 * hk) * d)).astype(np.float32)
    x, norm, rope = ctx.to_device(rows), ctx.to_device(to_bits(rng.uniform(0.5, 2, d))), ctx.buffer(300 * d * 4)
    ctx.rope_table(300, d, 1e6, rope)
    q, out = ctx.buffer(step.tokens * hq * d * 2), ctx.buffer(step.tokens * hq * d * 2)
    masks = ctx.to_device(random_tree(rng, step, 1, empty=0.0))
    kept, counts = ctx.to_device(np.zeros((2, 6), np.uint32)), ctx.to_device(np.zeros(2, np.uint32))
    pairs = ctx.to_device(np.zeros((1, 2), np.uint32))
    width = rows.shape[1]

    def run():
        ctx.qk_norm_rope(x.ptr, x.ptr + hq * d * 4, x.ptr + (hq + hk) * d * 4, mx4.F32, width, hq, norm, norm, 1e-6, rope, 300,
                         step.batch, step.cache, 1, q)
        ctx.attention(q, hq, step.batch, step.cache, 1, out, masks)
        ctx.cache_keep(step.cache, step.batch, kept, counts, 6)
        ctx.cache_copy_pages(step.cache, pairs, 1)

    def state(cached, lists, pair):
        step.dev["cached"].upload(np.array(cached, np.uint32))
        kept.upload(np.array([list(x) + [0] * (6 - len(x)) for x in lists], np.uint32))
        counts.upload(np.array([len(x) for x in lists], np.uint32))
        pairs.upload(np.array([pair], np.uint32))
        for buf, x in zip((step.k, step.v), step.kv):
            buf.upload(x)
        out.upload(np.zeros(out.nbytes, np.uint8))

    recorded = ctx.record(run)
    for cached, lists, pair in [([200, 31], [[0, 3, 8], [1, 2, 20, 29]], (2, 5)), ([3, 0], [[], [0]], (1, 0)),
                                ([150, 17], [[8], [4, 5, 6, 7, 8, 9]], (4, 4)), ([200, 31], [[0, 3, 8], [1, 2, 20, 29]], (2, 5))]:
        state(cached, lists, pair)
        recorded.launch()
        ctx.synchronize()
        replay = [out.download(np.uint16)] + step.down()
        state(cached, lists, pair)
        run()
        ctx.synchronize()
        for a, b in zip(replay, [out.download(np.uint16)] + step.down()):
            assert np.array_equal(a, b)
    recorded.release()


def test_offsets_past_32_bits(mx4, ctx):
    """Pages whose elements start past 2^32 of the cache."""
    rng = np.random.default_rng(12)
    hk, d, page, hq, at = 8, 128, 64, 16, 65536 + 5
    step = Step(mx4, ctx, rng, [40, 1], [100, 500], hk, d, page, at=at)
    assert at * step.row > 2 ** 32
    count = step.pages * step.row
    step.k, step.v = ctx.buffer(2 * count), ctx.buffer(2 * count)
    step.cache = mx4.KvCache(step.k, step.v, 1, step.pages, hk, page, d)
    low = at * step.row
    local = [np.full(count - low, NAN_BITS, np.uint16) for _ in range(2)]
    for x in local:
        for s, (n, c) in enumerate(zip(step.new, step.cached)):
            for p in range(n + c):
                x[step.at(s, p) - low] = to_bits(rng.standard_normal((hk, d)))
    step.k.upload(local[0], 2 * low)
    step.v.upload(local[1], 2 * low)
    step.rows = lambda s, side: np.stack([from_bits(local[side][step.at(s, p) - low]).astype(np.float64)
                                          for p in range(step.new[s] + step.cached[s])])
    got, q = attend(step, rng, hq)
    near(got, *reference(step, q, hq, chain(step)))
    # the cache write
    x = rng.standard_normal((step.tokens, (hq + 2 * hk) * d)).astype(np.float32)
    xd = ctx.to_device(x)
    out = ctx.buffer(step.tokens * hq * d * 2)
    ctx.qk_norm_rope(xd.ptr, xd.ptr + hq * d * 4, xd.ptr + (hq + hk) * d * 4, mx4.F32, x.shape[1], hq, None, None, 0.0, None, 0,
                     step.batch, step.cache, 0, out)
    for s in range(2):
        for i in range(step.new[s]):
            spot, token = step.at(s, step.cached[s] + i) - low, step.start[s] + i
            local[0][spot] = to_bits(x[token, hq * d:(hq + hk) * d].reshape(hk, d))
            local[1][spot] = to_bits(x[token, (hq + hk) * d:].reshape(hk, d))
    # a page copied up, tokens kept
    spare = sorted(set(range(at, step.pages)) - set(step.table[0, :3]) - set(step.table[1]))[0]
    src = int(step.table[1, 0])
    ctx.cache_copy_pages(step.cache, ctx.to_device(np.array([[src, spare]], np.uint32)), 1)
    ctx.cache_keep(step.cache, step.batch, ctx.to_device(np.array([[3, 30], [0, 0]], np.uint32)),
                   ctx.to_device(np.array([2, 1], np.uint32)), 2)
    for y in local:
        y[(spare - at) * step.row:(spare - at + 1) * step.row] = y[(src - at) * step.row:(src - at + 1) * step.row]
        moved = [y[step.at(0, 100 + j) - low].copy() for j in (3, 30)]
        for j, r in enumerate(moved):
            y[step.at(0, 100 + j) - low] = r
    for b, y in zip((step.k, step.v), local):
        assert np.array_equal(b.download(np.uint16, count - low, 2 * low), y)
    step.k.free()
    step.v.free()


def test_wrong_numbers_stay_inside_the_cache(mx4, ctx):
    """Page numbers past the cache, lengths past the table, a token count past
    its bound: no write lands anywhere, and the calls end well."""
    rng = np.random.default_rng(13)
    step = Step(mx4, ctx, rng, [4, 20], [10, 40], 2, 64, 16).fill(rng)
    step.dev["table"].upload(np.full(step.table.shape, 2 ** 32 - 1, np.uint32))
    step.dev["cached"].upload(np.array([10, 2 ** 31], np.uint32))
    x = ctx.to_device(rng.standard_normal((step.tokens, 8 * 64)).astype(np.float32))
    out = ctx.buffer(step.tokens * 4 * 64 * 2)
    ctx.qk_norm_rope(x, x, x, mx4.F32, 8 * 64, 4, None, None, 0.0, None, 0, step.batch, step.cache, 0, out)
    ctx.cache_keep(step.cache, step.batch, ctx.to_device(np.array([[1, 3], [2, 9]], np.uint32)),
                   ctx.to_device(np.array([2, 900], np.uint32)), 2)
    for side, y in zip(step.down(), step.kv):
        assert np.array_equal(side, y)
    few = mx4.Batch(2, step.tokens, 6, step.dev["start"], step.dev["cached"], step.dev["table"], step.width)
    step.dev["cached"].upload(np.array([10, 40], np.uint32))
    step.dev["table"].upload(step.table)
    mark = ctx.to_device(np.full(step.tokens * 4 * 64, 0x1234, np.uint16))
    q = to_bits(rng.standard_normal((step.tokens, 4, 64)))
    ctx.attention(ctx.to_device(q), 4, few, step.cache, 0, mark)
    got = mark.download(np.uint16).reshape(step.tokens, 4, 64)
    assert np.all(got[10:] == 0x1234)  # the second sequence's tokens past the bound
    want, tol = reference(step, from_bits(q).astype(np.float64), 4, chain(step))
    near(from_bits(got[:10]), want[:10], tol[:10])


def test_starts_that_do_not_ascend_end_well(mx4, ctx):
    """Every second sequence claims all tokens, so that their work counts to 2^32: what comes of it is
    nobody's, but nothing beside the outputs and the scratch is written, and later calls are right."""
    rng = np.random.default_rng(31)
    tokens, heads, d, page, seqs = 65536, 8, 64, 4096, 2048
    side = np.full((3, 1, page, d), 0x3f80, np.uint16)
    k, v = ctx.to_device(side), ctx.to_device(side)
    start = ctx.to_device(np.array([0, tokens] * (seqs // 2) + [0], np.uint32))
    cached, table = ctx.to_device(np.full(seqs, 65536, np.uint32)), ctx.to_device(rng.integers(0, 3, (seqs, 32)).astype(np.uint32))
    q, out = ctx.to_device(to_bits(rng.standard_normal((tokens, heads * d)))), ctx.buffer(tokens * heads * d * 2)
    after = ctx.to_device(np.full(1 << 20, 0x1234, np.uint16))
    ctx.attention(q, heads, mx4.Batch(seqs, tokens, tokens, start, cached, table, 32), mx4.KvCache(k, v, 1, 3, 1, page, d), 0, out)
    ctx.synchronize()
    assert np.array_equal(k.download(np.uint16), side.ravel()) and np.array_equal(v.download(np.uint16), side.ravel())
    assert np.all(after.download(np.uint16) == 0x1234)
    step = Step(mx4, ctx, rng, [40, 1], [900, 3000], 2, 64, 16).fill(rng)
    got, q = attend(step, rng, 8)
    near(got, *reference(step, q, 8, chain(step)))


def test_refusals(mx4, ctx):
    rng = np.random.default_rng(14)
    step = Step(mx4, ctx, rng, [2], [3], 2, 64, 16).fill(rng)
    buf = ctx.buffer(1 << 16)
    d = step.dev

    def cache(**kw):
        a = dict(k=step.k, v=step.v, layers=1, pages=step.pages, kv_heads=2, page_tokens=16, head_dim=64, layer_stride=0)
        a.update(kw)
        return mx4.KvCache(**a)

    def batch(**kw):
        a = dict(seqs=1, tokens=2, max_tokens=2, start=d["start"], cached=d["cached"], table=d["table"], table_stride=step.width)
        a.update(kw)
        return mx4.Batch(**a)

    def attention(b=None, c=None, q=buf, hq=4, layer=0, out=buf, tree=None, words=1, scale=0.0, qs=0, os=0):
        ctx.attention(q, hq, b or batch(), c or cache(), layer, out, tree, words, scale, qs, os)

    def rope(b=None, c=None, q=buf, xt=mx4.F32, stride=0, hq=4, norm=None, eps=1e-6, table=None, n=0, layer=0, out=buf, os=0):
        ctx.qk_norm_rope(q, buf, buf, xt, stride, hq, norm, norm, eps, table, n, b or batch(), c or cache(), layer, out, None, os)

    bad_caches = [dict(k=None), dict(k=step.k.ptr + 8), dict(layers=0), dict(pages=0), dict(kv_heads=0), dict(page_tokens=8),
                  dict(page_tokens=48), dict(page_tokens=8192), dict(head_dim=80), dict(layer_stride=8), dict(layers=40000),
                  dict(layer_stride=step.pages * 2048 + 4)]
    bad_batches = [dict(start=None), dict(cached=None), dict(table=None), dict(seqs=0), dict(table_stride=0), dict(max_tokens=0),
                   dict(max_tokens=3), dict(seqs=70000), dict(table=d["table"].ptr + 2)]
    calls = [lambda f=f, kw=kw: f(c=cache(**kw)) for f in (attention, rope) for kw in bad_caches]
    calls += [lambda f=f, kw=kw: f(b=batch(**kw)) for f in (attention, rope) for kw in bad_batches]
    calls += [lambda kw=kw: attention(**kw) for kw in [
        dict(q=None), dict(out=None), dict(hq=0), dict(hq=3), dict(layer=1), dict(q=buf.ptr + 2), dict(out=buf.ptr + 8),
        dict(tree=buf, words=0), dict(tree=buf.ptr + 4), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
        dict(qs=100), dict(qs=260), dict(os=1 << 33)]]
    calls += [lambda kw=kw: rope(**kw) for kw in [
        dict(q=None), dict(out=None), dict(hq=0), dict(xt=2), dict(layer=1), dict(q=buf.ptr + 4), dict(norm=buf.ptr + 2),
        dict(eps=-1.0), dict(eps=float("nan")), dict(table=buf, n=0), dict(stride=100), dict(stride=(258, 0, 0)), dict(os=4)]]
    calls += [lambda: ctx.rope_table(0, 64, 1e4, buf), lambda: ctx.rope_table(4, 63, 1e4, buf), lambda: ctx.rope_table(4, 64, 0.0, buf),
              lambda: ctx.rope_table(4, 64, float("nan"), buf), lambda: ctx.rope_table(4, 64, 1e4, None),
              lambda: ctx.cache_copy_pages(cache(), None, 1), lambda: ctx.cache_copy_pages(cache(pages=0), buf, 1),
              lambda: ctx.cache_keep(cache(), batch(), None, buf, 1), lambda: ctx.cache_keep(cache(), batch(seqs=0), buf, buf, 1)]
    for i, call in enumerate(calls):
        with pytest.raises(mx4.Mx4Error) as e:
            call()
        assert 1 <= e.value.status <= 4 or e.value.status == 9, i
    attention(b=batch(tokens=0, max_tokens=0))  # nothing to do
    rope(b=batch(tokens=0, max_tokens=0))


def test_more_rows_than_32_bits_count_are_refused(mx4, ctx):
    """Refused from the sizes alone: nothing of this size is there, and nothing is launched."""
    buf = ctx.to_device(np.zeros(1 << 18, np.uint32))
    for tokens, seqs, heads, kv_heads in [(1 << 30, 1, 2, 1), (1 << 20, 1, 2048, 8), (4, 65535, 65535, 65535)]:
        cache = mx4.KvCache(buf, buf, 1, 1, kv_heads, 16, 64)
        with pytest.raises(mx4.Mx4Error, match="2\\^31"):
            ctx.attention(buf, heads, mx4.Batch(seqs, tokens, 1, buf, buf, buf, 1), cache, 0, buf)


def test_example_decodes_the_same_tokens_by_trees(mx4):
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "tree_decode.py"
    spec = importlib.util.spec_from_file_location("tree_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    plain, trees, steps, free = example.main()
    assert trees == plain and len(set(plain)) > 8
    assert steps < len(plain)
    both = -(-(45 + len(plain)) // example.PAGE)
    assert free == example.PAGES - (2 * both - 45 // example.PAGE)
