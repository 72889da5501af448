"""Plain 64-bit form of mtg_sample_dev (include/mtg_verify.h), in numpy: the answers that a row may have. More than one is
right only where a target lies within EPS of the sum at which the answer changes."""
import numpy as np

EPS = 2.0 ** -26  # a sum's two sides, each of weights off by 2^-27


def answers(x, temperature, top_p, min_p, top_k, uniform):
    """{id: probabilities} of the ids that may be chosen; {-1: [0.0]} where no id takes part."""
    x = np.asarray(x, np.float64)
    ids = np.flatnonzero(x > -np.inf)  # no NaN is
    if not len(ids):
        return {-1: [0.0]}
    ids = ids[np.argsort(-x[ids], kind="stable")]
    y, top = x[ids], x[ids[0]]
    if not temperature > 0:
        return {int(ids[0]): [1.0]}
    T = np.float64(np.float32(temperature))
    with np.errstate(invalid="ignore", over="ignore", under="ignore"):
        w = np.where(y == top, 1.0, 0.0 if np.isinf(top) else np.exp((y - top) / T))
    n = len(w)
    k = top_k if 0 < top_k < n else n
    run = np.cumsum(w)
    cuts = [k]
    if np.float32(top_p) < 1:
        target = float(np.float32(top_p)) * run[k - 1]
        first, last = (int(np.searchsorted(run[:k], target * f)) + 1 for f in (1 - EPS, 1 + EPS))
        cuts = sorted({max(1, min(c, k)) for c in range(first, last + 1)})
    if np.float32(min_p) > 0:
        m = float(np.float32(min_p))
        lo, hi = (max(1, int((w >= m * f).sum())) for f in (1 + EPS, 1 - EPS))
        cuts = sorted({min(c, d) for c in cuts for d in range(lo, hi + 1)})
    u = 0.0 if not uniform > 0 else min(float(np.float32(uniform)), 1 - 2.0 ** -24)
    out = {}
    for cut in cuts:
        kept = run[cut - 1]
        first, last = (int(np.searchsorted(run[:cut], u * kept * f, side="right")) for f in (1 - EPS, 1 + EPS))
        for i in range(first, min(last, cut - 1) + 1):
            out.setdefault(int(ids[i]), []).append(w[i] / kept)
    return out
