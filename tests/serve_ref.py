"""Plain 64-bit forms of the serving operators (include/mtg_verify.h: mtg_rope_append_dev,
mtg_paged_attn_dev, mtg_logits_step_dev) and batches of sequences over a pool of pages, in numpy."""
import numpy as np

TYPES = {"f32": np.float32, "f16": np.float16}
# half a step of each type, relative to the value: what one rounding may be off
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25}  # half a step of the smallest numbers


class Batch:
    """Sequences with (new rows, cache length) in `lens`, their pages scattered over a pool. Rows before
    the first sequence (`lead`) and behind the last (`tail`) belong to none. What no sequence holds is NaN."""

    def __init__(self, rng, lens, kv_heads, dim, page, kv="f16", lead=0, tail=0, spare=2, filled=True):
        self.lens, self.kv_heads, self.dim, self.page, self.kv = lens, kv_heads, dim, page, kv
        need = [-(-max(0, length) // page) for _, length in lens]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((max(1, len(lens)), max(need + [1]) + 1), -7, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        starts = [lead]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.q_start = np.array(starts, np.int32)
        self.kv_len = np.array([length for _, length in lens], np.int32)
        self.n_tokens = starts[-1] + tail
        shape = (self.n_pages, kv_heads, page, dim)
        self.k, self.v = (np.full(shape, np.nan, TYPES[kv]) for _ in range(2))
        if filled:
            for b, (_, length) in enumerate(lens):
                for p in range(max(0, length)):
                    where = (self.table[b, p // page], slice(None), p % page)
                    self.k[where] = rng.standard_normal((kv_heads, dim))
                    self.v[where] = rng.standard_normal((kv_heads, dim))

    def positions(self):
        """{row: (sequence, position)} of the rows that belong to a sequence."""
        out = {}
        for b in range(len(self.lens)):
            s, e = int(self.q_start[b]), int(self.q_start[b + 1])
            for t in range(s, e):
                out[t] = (b, int(self.kv_len[b]) - (e - s) + t - s)
        return out

    def page_of(self, b, p):
        if p < 0 or p // self.page >= self.table.shape[1]:
            return -1
        i = int(self.table[b, p // self.page])
        return i if 0 <= i < self.n_pages else -1

    def keys(self, b, hi):
        """Keys and values of positions 0 .. hi-1 that lie in pages: (positions, k, v) in 64 bits."""
        where = [(p, self.page_of(b, p)) for p in range(max(0, hi))]
        where = [(p, i) for p, i in where if i >= 0]
        pos = np.array([p for p, _ in where], np.int64)
        ids = np.array([i for _, i in where], np.int64)
        take = lambda a: a[ids, :, pos % self.page].astype(np.float64)  # noqa: E731  [key][head][dim]
        return pos, take(self.k), take(self.v)


def attend(batch, q, scale, window=0):
    """(out, bound): rows outside every sequence are NaN. bound[row][head][d]: sum of the weights times |v|
    over the weights' sum, and sharp[row][head]: scale * max_j sum_d |q_d k_jd|, for tolerances."""
    n, heads, dim = q.shape
    group = heads // batch.kv_heads
    out = np.full(q.shape, np.nan)
    size = np.zeros(q.shape)
    sharp = np.zeros((n, heads))
    cache = {}
    for t, (b, p) in batch.positions().items():
        if b not in cache:
            cache[b] = batch.keys(b, int(batch.kv_len[b]))
        pos, k, v = cache[b]
        see = pos <= p
        if window:
            see &= pos > p - window
        for h in range(heads):
            if not see.any():
                out[t, h] = 0.0
                continue
            kk, vv = k[see, h // group], v[see, h // group]
            z = kk @ q[t, h].astype(np.float64) * scale
            w = np.exp(z - z.max())
            w /= w.sum()
            out[t, h] = w @ vv
            size[t, h] = w @ np.abs(vv)
            sharp[t, h] = abs(scale) * (np.abs(kk) @ np.abs(q[t, h].astype(np.float64))).max()
    return out, size, sharp


def attend_tolerance(out, size, sharp, io, keys, dim):
    """How far a row may be off. Scores: sums of dim products in 32 bits, each addition off by half a step of a
    partial sum of at most `sharp`, adding up as a random walk (four times its spread), f32 rows in parts of
    22 bits or more (2^-21); an error d of the scores changes the weighted mean by 2 d times `size`. Sums over the
    keys likewise in 32 bits. Weights for f16 rows are rounded to f16 once (2^-11 of each weight). At last the rounding
    of the output, and with f16 that of what it rounds."""
    step = 2.0 ** -24
    d = sharp[..., None] * (4 * np.sqrt(dim) * step + 2.0 ** -21)
    tol = size * (2 * d + 4 * np.sqrt(keys + 64) * step + 2.0 ** -21)
    if io == "f16":
        tol = tol + size * HALF["f16"]
    return tol + np.abs(out) * HALF[io] * 1.01 + TINY[io]


def freqs(rot, base=1e6):
    return base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))


def rotate(x, pos, f, rot, interleaved, mscale, gain=None, eps=1e-6):
    """One row [heads][dim] in 64 bits: (values, size) where size bounds what a value is made of."""
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    i = np.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    c, s = np.cos(pos * f) * mscale, np.sin(pos * f) * mscale
    y, size = x.copy(), np.abs(x)
    y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, a] * s + x[:, b] * c
    size[:, a] = size[:, b] = (np.abs(x[:, a]) + np.abs(x[:, b])) * abs(mscale)
    return y, size


def rotate_tolerance(y, size, to):
    """The angle is off by 2^-25 turns (2 pi 2^-25) and its cos / sin by a step; the norm's sum of 64 or 128 squares
    and its four further operations by 32 half steps at most, the rotation by 4 more: 2^-18 of the size covers their
    sum (5.0 + 2 + 36 half steps of 2^-24 make 2^-18.6); then the rounding to the output's type."""
    return size * 2.0 ** -18 + np.abs(y) * HALF[to] + TINY[to]


def logits_row(x, history, penalties, bias, allowed):
    """One row in 64 bits: (y, size), size bounding what the operations round. history: ids, bias: [(id, value)]
    in list order, allowed: bool per id or None."""
    y = x.astype(np.float64)
    size = np.abs(y)
    rep, freq, pres = (float(np.float32(p)) for p in penalties)
    ids, times = np.unique([i for i in history if 0 <= i < len(x)], return_counts=True) if len(history) else ((), ())
    for i, c in zip(ids, times):
        if rep > 1:
            y[i] = y[i] / rep if y[i] > 0 else y[i] * rep
        size[i] = max(size[i], abs(y[i])) + 3 * (abs(freq * c) + abs(pres))
        y[i] -= freq * c + pres
    for i, value in {i: v for i, v in bias if 0 <= i < len(x)}.items():
        y[i] += float(np.float32(value))
        size[i] += abs(float(np.float32(value)))
    if allowed is not None:
        y[~allowed] = -np.inf
    return y, size


def first_max(y, allowed):
    """The lowest allowed id with the largest value, no NaN; -1 if there is none."""
    ok = ~np.isnan(y) if allowed is None else allowed & ~np.isnan(y)
    if not ok.any():
        return -1
    return int(np.flatnonzero(ok & (y == y[ok].max()))[0])
