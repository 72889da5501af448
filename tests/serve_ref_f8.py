"""Plain 64-bit forms of the operators over a paged cache in 8 bits (include/mtg_verify.h: mtg_rope_append_f8_dev,
mtg_paged_attn_f8_dev), in numpy."""
import numpy as np

import serve_ref

BLOCK = 16


def _values():
    """The value of each e4m3 code: s eeee mmm, bias 7, subnormal where e = 0, NaN where all of e and m are set."""
    v = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v[c] = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        if c & 127 == 127:
            v[c] = np.nan
        if c & 128:
            v[c] = -v[c]
    return v


VALUES = _values()


def step(x):
    """The distance of e4m3 numbers around x."""
    return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6))) - 3)


def codes(x):
    """The nearest codes, ties to even; of what is not finite 127 (NaN)."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x)
    y = np.abs(np.where(ok, x, 0.0))
    _, e = np.frexp(np.maximum(y, 2.0 ** -6))
    q = np.ldexp(np.round(np.ldexp(y, 4 - e)), e - 4)  # steps of 2^(e - 4) for y of 2^(e - 1) and more
    assert (q <= 448).all()
    bits = q.astype(np.float32).view(np.uint32)  # exact: the same mantissa with 20 more bits, bias 127 instead of 7
    c = np.where(q >= 2.0 ** -6, (bits >> 20) - (120 << 3), (q * 512).astype(np.uint32)).astype(np.uint8)
    c |= np.where(np.signbit(x) & ok, 128, 0).astype(np.uint8)
    return np.where(ok, c, 127).astype(np.uint8)


def is_nan(c):
    return c & 127 == 127


def exponent(top):
    """The least e >= -100 with top <= 448 * 2^e, of numbers or arrays: 448 is 0.875 * 2^9."""
    m, x = np.frexp(top)
    return np.where(np.asarray(top) > 0, np.maximum(x - 9 + (m > 0.875), -100), -100)


class Batch(serve_ref.Batch):
    """As serve_ref.Batch, with codes kc, vc [page][head][place][dim] and scales ks, vs [page][head][block]. What no
    sequence holds are codes NaN and scales of 255 or of any size. `k` and `v` are the values in 64 bits."""

    def __init__(self, rng, lens, kv_heads, dim, page, filled=True, spread=2.0, **kw):
        super().__init__(rng, lens, kv_heads, dim, page, kv="f32", filled=filled, **kw)
        self.kv = "f8"
        blocks = page // BLOCK
        for name in "kv":
            x = getattr(self, name).reshape(self.n_pages, kv_heads, blocks, BLOCK, dim).astype(np.float64)
            x = x * 2.0 ** (spread * rng.standard_normal((self.n_pages, kv_heads, blocks, 1, 1)))
            top = np.where(np.isnan(x), 0.0, np.abs(x)).max((3, 4))
            e = exponent(top).astype(np.int64)
            held = ~np.isnan(x).all((3, 4))
            scale = np.where(held, e + 127, rng.choice([0, 255, 127, 250], size=e.shape)).astype(np.uint8)
            c = codes(x / 2.0 ** e[..., None, None])
            setattr(self, name + "c", c.reshape(self.n_pages, kv_heads, page, dim))
            setattr(self, name + "s", scale)
        self.values()

    def values(self):
        """k and v from the codes and scales as they stand."""
        for name in "kv":
            s = np.minimum(getattr(self, name + "s"), 254).astype(np.float64) - 127
            setattr(self, name, VALUES[getattr(self, name + "c")] * 2.0 ** np.repeat(s, BLOCK, axis=2)[..., None])


def append(batch, name, new, size):
    """Rows `new` [row][head][dim] in 64 bits into the codes and scales of `name`. Returns (codes, scales low, scales
    high, value, tolerance, kind): scales may be low or high where the largest element, off by what 32 bits make of `size`
    (None: it is exact), lies on a border; kind of a place: 0 as it was, 1 earlier row of a block (codes follow the
    scale), 2 new row (value within tolerance, given the scale)."""
    c, s = getattr(batch, name + "c").copy(), getattr(batch, name + "s")
    low, high = s.copy().astype(np.int64), s.copy().astype(np.int64)
    value, slack = np.full(c.shape, np.nan), np.zeros(c.shape)
    kind = np.zeros(c.shape[:1] + c.shape[2:3], np.int64)  # [page][place]
    blocks = {}
    for t, (b, p) in batch.positions().items():
        page = batch.page_of(b, p)
        if page < 0:
            continue
        place = p % batch.page
        value[page, :, place] = new[t]
        if size is not None:
            slack[page, :, place] = size[t]
        kind[page, place] = 2
        first = int(batch.kv_len[b]) - int(batch.q_start[b + 1] - batch.q_start[b])
        blocks[page, place // BLOCK] = max(0, first - (p - p % BLOCK))
    for (page, block), before in blocks.items():
        places = np.arange(BLOCK * block, BLOCK * block + BLOCK)
        kind[page, places[:before]] = 1
        rows = places[kind[page, places] == 2]
        for h in range(c.shape[1]):
            x, w = value[page, h][rows], slack[page, h][rows]
            ok = np.isfinite(x)
            e = [int(exponent((np.abs(x[ok]) + sign * w[ok]).max(initial=0.0))) for sign in (-1, 1)]
            if before:
                e = [max(i, min(int(s[page, h, block]), 254) - 127) for i in e]
            low[page, h, block], high[page, h, block] = e[0] + 127, e[1] + 127
    return c, low, high, value, slack, kind


def check_append(batch, name, got_codes, got_scales, new, size):
    """The codes and scales that a call left, against append()."""
    c, low, high, value, slack, kind = append(batch, name, new, size)
    was = getattr(batch, name + "s").astype(np.int64)
    assert ((got_scales >= low) & (got_scales <= high)).all(), np.argwhere((got_scales < low) | (got_scales > high))[:5]
    exp = np.minimum(got_scales, 254).astype(np.int64) - 127
    exp = np.repeat(exp, BLOCK, axis=2)[..., None]
    old = np.repeat(np.minimum(was, 254) - 127, BLOCK, axis=2)[..., None]
    kind = kind[:, None, :, None]
    k0 = np.broadcast_to(kind == 0, c.shape)
    assert np.array_equal(got_codes[k0], c[k0])
    k1 = np.broadcast_to(kind == 1, c.shape)
    follow = np.where(exp == old, c, np.where(is_nan(c), c, codes(np.where(is_nan(c), 0.0, VALUES[c]) * 2.0 ** np.clip(old - exp, -400, 0).astype(float))))
    same = (got_codes == follow) | (is_nan(got_codes) & is_nan(follow))
    assert same[k1].all(), np.argwhere(k1 & ~same)[:5]
    k2 = np.broadcast_to(kind == 2, c.shape)
    finite = np.isfinite(value)
    assert is_nan(got_codes)[k2 & ~finite].all() and not is_nan(got_codes)[k2 & finite].any()
    x = np.where(k2 & finite, value, 0.0) / 2.0 ** exp
    w = np.where(k2 & finite, slack, 0.0) / 2.0 ** exp
    # within half a step of what 32 bits make of the value
    far = np.abs(np.where(k2 & finite, VALUES[got_codes], 0.0) - x)
    tol = w + step(np.abs(x) + w) / 2
    assert (far <= tol).all(), (np.argwhere(far > tol)[:5], (far / tol).max())


def attend(batch, q, scale, window=0, sink=0):
    """serve_ref.attend with the first `sink` positions beside the window. Also floor[row][head][d]: the sum of |v| over
    the weights' sum, the largest weight being 1."""
    n, heads, dim = q.shape
    group = heads // batch.kv_heads
    out, size, sharp, floor = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros((n, heads)), np.zeros(q.shape)
    cache = {}
    for t, (b, p) in batch.positions().items():
        if b not in cache:
            cache[b] = batch.keys(b, int(batch.kv_len[b]))
        pos, k, v = cache[b]
        see = pos <= p
        if window:
            see &= (pos > p - window) | (pos < sink)
        for h in range(heads):
            if not see.any():
                out[t, h] = 0.0
                continue
            kk, vv = k[see, h // group], v[see, h // group]
            z = kk @ q[t, h].astype(np.float64) * scale
            w = np.exp(z - z.max())
            floor[t, h] = np.abs(vv).sum(0) / w.sum()
            w /= w.sum()
            out[t, h] = w @ vv
            size[t, h] = w @ np.abs(vv)
            sharp[t, h] = abs(scale) * (np.abs(kk) @ np.abs(q[t, h].astype(np.float64))).max()
    return out, size, sharp, floor


def attend_tolerance(batch, q, got, scale, io, keys):
    """serve_ref.attend_tolerance, which takes the cached values as exact and a weight's error as relative to it, and what
    that leaves out where values lie far apart: a weight, 2^7 or more where it is the largest, is at last off by half a
    step of f16's smallest numbers, 2^-25, which is 2^-32 of the largest weight, times |v| of its key; and codes of small
    blocks beside large ones by 2^-25 of the largest scale of the sequence's keys, for each element of k and v."""
    want, size, sharp, floor = got
    tol = serve_ref.attend_tolerance(want, size, sharp, io, keys, batch.dim) + 2.0 ** -32 * floor
    group = q.shape[1] // batch.kv_heads
    largest = {}
    for t, (b, p) in batch.positions().items():
        if b not in largest:
            ids = sorted({(batch.page_of(b, x), x % batch.page // BLOCK) for x in range(0, max(0, int(batch.kv_len[b])), BLOCK)})
            ids = [i for i in ids if i[0] >= 0]
            largest[b] = [np.array([2.0 ** max([min(int(s[i, h, j]), 254) - 127 for i, j in ids] + [-127]) for h in range(batch.kv_heads)])
                          for s in (batch.ks, batch.vs)]
        k, v = (x[np.arange(q.shape[1]) // group] * 2.0 ** -25 for x in largest[b])
        d = abs(scale) * np.abs(q[t].astype(np.float64)).sum(-1) * k
        tol[t] += 2 * size[t] * d[:, None] + v[:, None]
    return tol


def seen_blocks(batch, b, window=0, sink=0):
    """[(page, block)] of sequence b's blocks in pages, and whether some row of it sees one of their positions."""
    last = int(batch.kv_len[b]) - 1
    first = last + 1 - int(batch.q_start[b + 1] - batch.q_start[b])
    oldest = first - window + 1 if window else 0
    out = []
    for x in range(0, last + 1, BLOCK):
        page = batch.page_of(b, x)
        if page >= 0:
            out.append(((page, x % batch.page // BLOCK), any(j <= last and (j >= oldest or j < sink) for j in range(x, x + BLOCK))))
    return out


def attend_tolerance_seen(batch, q, got, scale, io, keys, window=0, sink=0):
    """attend_tolerance with the largest scale of the blocks that rows of the sequence see."""
    want, size, sharp, floor = got
    tol = serve_ref.attend_tolerance(want, size, sharp, io, keys, batch.dim) + 2.0 ** -32 * floor
    heads = np.arange(q.shape[1]) * batch.kv_heads // q.shape[1]
    largest = {}
    for t, (b, p) in batch.positions().items():
        if b not in largest:
            ids = [i for i, seen in seen_blocks(batch, b, window, sink) if seen]
            largest[b] = [np.array([2.0 ** max([min(int(s[i, h, j]), 254) - 127 for i, j in ids] + [-127]) for h in range(batch.kv_heads)])
                          for s in (batch.ks, batch.vs)]
        k, v = (x[heads] * 2.0 ** -25 for x in largest[b])
        d = abs(scale) * np.abs(q[t].astype(np.float64)).sum(-1) * k
        tol[t] += 2 * size[t] * d[:, None] + v[:, None]
    return tol


def attend_tolerance_own(batch, q, got, scale, io, keys, window=0, sink=0):
    """How far a row may be off by the keys it sees itself: serve_ref.attend_tolerance, and a weight, 2^7 or more where it is
    the largest, by half a step of f16's smallest numbers, 2^-32 of the largest weight, times the codes of its key in the
    largest scale of V among the keys that the row sees. Codes of K and V add nothing."""
    want, size, sharp, _ = got
    tol = serve_ref.attend_tolerance(want, size, sharp, io, keys, batch.dim)
    group = q.shape[1] // batch.kv_heads
    cache = {}
    for t, (b, p) in batch.positions().items():
        if b not in cache:
            pos, k, v = batch.keys(b, int(batch.kv_len[b]))
            ids = np.array([batch.page_of(b, x) for x in pos], np.int64)
            e = np.minimum(batch.vs[ids, :, pos % batch.page // BLOCK], 254).astype(np.int64) - 127
            cache[b] = pos, k, v, 2.0 ** e
        pos, k, v, s = cache[b]
        see = pos <= p
        if window:
            see &= (pos > p - window) | (pos < sink)
        if not see.any():
            continue
        for h in range(q.shape[1]):
            z = k[see, h // group] @ q[t, h].astype(np.float64) * scale
            size_of = s[see, h // group]
            codes_of = np.abs(v[see, h // group]) / size_of[:, None]
            tol[t, h] += 2.0 ** -32 * codes_of.sum(0) * size_of.max() / np.exp(z - z.max()).sum()
    return tol
