"""mtg_paged_attn_f8_dev on the GPU with scales far apart in one call: those of later rows of the same call, and of keys that
only some rows of a tile see, do not reach the other rows; what a row sees of sizes far apart it sees exactly."""
import numpy as np
import pytest

from serve_ref_f8 import Batch, attend, attend_tolerance_own

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import dev  # noqa: E402
from serve_dev_f8 import Attend, Cache  # noqa: E402
from test_gpu_paged_attn_f8 import IO, _rows  # noqa: E402

# heads, kv heads, sequences (new rows, length), window, first positions, the first block whose scales are raised and behind the last
ROUTES = {
    "rows16": (2, 2, [(16, 104)], 0, 0, 6, 7),
    "rows16_window": (2, 2, [(16, 106)], 40, 0, 3, 4),
    "rows16_splits": (2, 1, [(8, 2006), (1, 77)], 0, 0, 125, 126),
    "rows32": (4, 2, [(30, 400), (12, 389)], 0, 0, 24, 25),
    "rows32_window": (4, 2, [(30, 400)], 64, 3, 19, 20),
    "rows32_splits": (4, 1, [(15, 5005), (1, 77)], 0, 0, 312, 313),
    "eight": (16, 8, [(8, 708 - 13 * i) for i in range(17)], 0, 0, 44, 45),
    "chunk": (4, 2, [(180, 600), (70, 389)], 0, 0, 30, 31),
    "chunk_window": (4, 2, [(180, 600)], 50, 5, 28, 29),
    "chunk_splits": (4, 2, [(150, 4100), (60, 2000)], 0, 0, 255, 257),
    "wide": (7, 1, [(150, 1900), (147, 700)], 0, 0, 115, 116),
    "wide_splits": (16, 1, [(70, 5000), (64, 800)], 0, 0, 309, 310),
}


def _call(b, q, io, scale, window, sink, splits):
    qd = dev(q)
    out = torch.full_like(qd, 55.0)
    Attend(Cache(b), qd, out, io, scale, window, int(b.kv_len.max()) if splits else 1, sink)()
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _compare(b, q, got, io, scale, window, sink, rows):
    form = attend(b, q, scale, window, sink)
    tol = attend_tolerance_own(b, q, form, scale, io, int(b.kv_len.max()), window, sink)
    want, tol, got = form[0][rows], tol[rows], got[rows].astype(np.float64)
    if io == "f16":  # 65,520 and more round to infinity
        huge = np.isinf(got)
        assert (np.where(got > 0, want, -want) + tol >= 65520)[huge].all()
        got = np.where(huge, want, got)
    off = np.abs(got - want)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("which,up,dim,io", [("kv", 30, 128, "f32"), ("v", 45, 64, "f16"), ("k", 45, 128, "f16"), ("v", 100, 128, "f32"),
                                             ("kv", 100, 64, "f32")])
@pytest.mark.parametrize("route", ROUTES)
def test_blocks_that_other_rows_see(route, which, up, dim, io):
    """Blocks of sequence 0 with scales 2^up larger. Rows that do not see them are as the form says, with the tolerance of
    what they see; those that see them are where V alone is larger (scores beyond 2^20 and more keep no fraction)."""
    heads, kv_heads, lens, window, sink, first, behind = ROUTES[route]
    rng = np.random.default_rng(dim + up)
    b = Batch(rng, lens, kv_heads, dim, 16, spread=1.0)
    rms = float(np.sqrt((b.k[~np.isnan(b.k)] ** 2).mean()))
    scale, q = dim ** -0.5 / max(1.0, rms), _rows(rng, b, heads, io)
    for block in range(first, behind):
        page = b.page_of(0, 16 * block)
        for x in which:
            s = getattr(b, x + "s")
            s[page, :, 0] = np.minimum(s[page, :, 0].astype(int) + up, 240)
    b.values()
    got = _call(b, q, io, scale, window, sink, "splits" in route or route == "eight")
    at = b.positions()
    sees = {t for t, (s, p) in at.items() if s == 0 and p >= 16 * first and
            (not window or p - window + 1 < 16 * behind or 16 * first < sink)}
    clear = sorted(t for t in at if t not in sees)
    assert sees and any(at[t][0] == 0 for t in clear)
    _compare(b, q, got, io, scale, window, sink, clear)
    if which == "v":
        _compare(b, q, got, io, scale, window, sink, sorted(sees))


@pytest.mark.parametrize("route,io", [(r, IO[i % 2]) for i, r in enumerate(ROUTES)])
def test_rows_whose_keys_are_of_sizes_far_apart(route, io):
    """Scales of K and of V of any size in every block, zeros among them; scores of some units all the same, for q is zero but
    in the element that K has one size in."""
    heads, kv_heads, lens, window, sink, _, _ = ROUTES[route]
    dim = 64
    rng = np.random.default_rng(len(route))
    b = Batch(rng, lens, kv_heads, dim, 16, spread=0.0)
    for s in range(len(lens)):
        for x in range(0, int(b.kv_len[s]), 16):
            page = b.page_of(s, x)
            e = rng.integers(-30, 7)
            # K: element 0 of ordinary size, whatever the block's scale: code 2^-e in a scale of 2^e, as far as codes go
            k = int(np.clip(e, -7, 6))
            b.ks[page], b.vs[page] = 127 + e, rng.choice([27, 60, 100, 110, 120, 127, 130])
            b.kc[page, :, :, 0] = rng.integers(0, 8, (kv_heads, 16)) + 8 * (7 - k) + 128 * rng.integers(0, 2, (kv_heads, 16))
    b.values()
    q = np.zeros((b.n_tokens, heads, dim))
    q[:, :, 0] = rng.uniform(-1, 1, (b.n_tokens, heads))
    q = q.astype(np.float16 if io == "f16" else np.float32)
    got = _call(b, q, io, 1.0, window, sink, "splits" in route or route == "eight")
    _compare(b, q, got, io, 1.0, window, sink, sorted(b.positions()))
