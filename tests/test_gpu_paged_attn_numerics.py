"""mtg_paged_attn_dev on the GPU where its numbers are hard to get right, against the 64-bit form
(serve_ref.attend): weighted means that nearly cancel, rows without a key beside rows whose maximum moves."""
import numpy as np
import pytest

from serve_ref import HALF, TYPES, Batch, attend, attend_tolerance

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import Attend, Cache, dev  # noqa: E402


def _call(b, q, io, scale, window=0, max_kv=0):
    qd = dev(q)
    out = torch.full_like(qd, 55.0)
    Attend(Cache(b), qd, out, io, scale, window, max_kv)()
    torch.cuda.synchronize()
    return out.cpu().numpy()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads,kv_heads,max_kv", [
    ([(1, 2), (1, 8), (1, 30), (0, 4), (1, 6)], 4, 2, 0),           # 16 pairs a tile
    ([(6, 8), (5, 12), (2, 2)], 8, 2, 0),                           # 32 pairs a tile
    ([(1, 2 + i % 30) for i in range(20)], 16, 8, 600),             # eight waves
    ([(2, 700), (1, 10), (1, 516)], 2, 2, 700),                     # splits
], ids=["16", "32", "eight", "splits"])
def test_weights_of_f16_rows_keep_22_bits(dim, lens, heads, kv_heads, max_kv):
    """Scores so small that all weights are nearly one, and values that are +x and -x in turn: the weighted mean is a
    small part of what it is made of, and weights of 11 bits (2^-12 of each, rounded) would show in it. The tolerance is
    that of f32 rows (no rounding of the weights to f16), plus the rounding of the output to f16."""
    rng = np.random.default_rng(dim + heads)
    b = Batch(rng, lens, kv_heads, dim, 16, "f16")
    for s, (_, length) in enumerate(lens):
        x = rng.standard_normal((kv_heads, dim))
        for p in range(length):
            b.v[b.page_of(s, p), :, p % 16] = -x if p % 2 else x
    q = rng.standard_normal((b.n_tokens, heads, dim)).astype(np.float16)
    scale = 0.002
    got = _call(b, q, "f16", scale, max_kv=max_kv)
    want, size, sharp = attend(b, q, scale)
    tol = attend_tolerance(want, size, sharp, "f32", int(b.kv_len.max()), dim) + np.abs(want) * HALF["f16"] * 1.01 + 2.0 ** -25
    off = np.abs(got.astype(np.float64) - want)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("io,kv", [("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 20])
def test_rows_that_see_no_page_beside_rows_whose_maximum_moves(io, kv, dim, window):
    """Positions below 912 have no page, so the first rows of a chunk see nothing and give zeros. Those behind see one
    key at 928 (in the next block of 32) whose score is far above or below all others: their maximum moves there."""
    rng = np.random.default_rng(dim + window)
    b = Batch(rng, [(128, 1032), (70, 70)], 1, dim, 16, kv, lead=1)
    b.table[0, :57] = -1
    b.k[b.page_of(0, 928), :, 0] *= TYPES[kv](20.0)
    q = rng.standard_normal((b.n_tokens, 1, dim)).astype(TYPES[io])
    scale = dim ** -0.5
    got = _call(b, q, io, scale, window)
    want, size, sharp = attend(b, q, scale, window)
    inside = sorted(b.positions())
    assert (got[1:9] == 0).all() and (got[0] == 55.0).all()   # positions 904 .. 911
    off = np.abs(got.astype(np.float64) - want)[inside]
    tol = attend_tolerance(want, size, sharp, io, 1032, dim)[inside]
    assert (off <= tol).all(), float((off / tol).max())
