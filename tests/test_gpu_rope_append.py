"""mtg_rope_append_dev on the GPU against the 64-bit form (serve_ref.rotate), with serve_ref's derived
tolerances: types, head sizes, both pair layouts, parts of the head, far positions, norms, cache
layouts, rows of no sequence, bad page ids."""
import ctypes

import numpy as np
import pytest

import mtg
from serve_ref import Batch, TYPES, freqs, rotate, rotate_tolerance

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import MTG, Cache, at, check, dev, stream  # noqa: E402

TYPE_PAIRS = [("f32", "f16"), ("f16", "f16"), ("f32", "f32")]


class Call:
    """Rows of one q|k|v product through the operator, and what they should become."""

    def __init__(self, rng, batch, io, heads, rot, inter, norm=False, mscale=1.0, positions=None, layout="page", f=None):
        self.b, self.io, self.heads, self.rot, self.inter, self.mscale = batch, io, heads, rot, inter, mscale
        n, hk, d = batch.n_tokens, batch.kv_heads, batch.dim
        self.x = rng.standard_normal((n, heads + 2 * hk, d)).astype(TYPES[io])
        self.gain = [(1 + 0.2 * rng.standard_normal(d)).astype(np.float32) for _ in range(2)] if norm else [None, None]
        self.pos, self.f = positions, freqs(rot) if f is None else f
        self.cache = Cache(batch, layout)
        self.xd = dev(self.x)
        self.out = torch.full((n, heads, d), 77.0, dtype=self.xd.dtype, device="cuda")
        w, e = (heads + 2 * hk) * d, self.xd.element_size()
        keep = [dev(self.f), *(None if g is None else dev(g) for g in self.gain), None if positions is None else dev(positions)]
        self.keep = keep
        self.d = mtg.RopeAppend(kv=self.cache.desc(), q=at(self.xd), k_new=at(self.xd) + heads * d * e,
                                v_new=at(self.xd) + (heads + hk) * d * e, q_out=at(self.out), positions=at(keep[3]),
                                freqs=at(keep[0]), q_norm=at(keep[1]), k_norm=at(keep[2]), q_stride=w, k_stride=w, v_stride=w,
                                q_out_stride=heads * d, io_type=MTG[io], n_heads=heads, rot_dim=rot, interleaved=int(inter),
                                eps=1e-6, mscale=mscale)

    def run(self, s=None):
        check(mtg.lib().mtg_rope_append_dev(ctypes.byref(self.d), stream() if s is None else s))
        torch.cuda.synchronize()

    def verify(self, q_out=None, with_q=True, with_kv=True):
        b, h, hk = self.b, self.heads, self.b.kv_heads
        got_q = (self.out if q_out is None else q_out).cpu().numpy()
        got_k, got_v = self.cache.read()
        want_k, want_v = b.k.astype(np.float64), b.v.astype(np.float64)   # what no new row fills stays
        tol_k, tol_v = np.zeros(b.k.shape), np.zeros(b.v.shape)
        rows = b.positions()
        for t in range(b.n_tokens):
            if t not in rows:
                if with_q and q_out is None:
                    assert (got_q[t] == 77.0).all(), t
                continue
            s, p = rows[t]
            at_ = p if self.pos is None else int(self.pos[t])
            if with_q:
                y, size = rotate(self.x[t, :h], at_, self.f, self.rot, self.inter, self.mscale, self.gain[0])
                assert (np.abs(got_q[t] - y) <= rotate_tolerance(y, size, self.io)).all(), ("q", t, np.abs(got_q[t] - y).max())
            page = b.page_of(s, p)
            if with_kv and page >= 0:
                y, size = rotate(self.x[t, h:h + hk], at_, self.f, self.rot, self.inter, self.mscale, self.gain[1])
                want_k[page, :, p % b.page], tol_k[page, :, p % b.page] = y, rotate_tolerance(y, size, b.kv)
                v = self.x[t, h + hk:].astype(np.float64)
                want_v[page, :, p % b.page], tol_v[page, :, p % b.page] = v, rotate_tolerance(v, 0 * v, b.kv)
        for got, want, tol in ((got_k, want_k, tol_k), (got_v, want_v, tol_v)):
            assert np.array_equal(np.isnan(got), np.isnan(want))
            fine = ~np.isnan(want)
            assert (np.abs(got[fine].astype(np.float64) - want[fine]) <= tol[fine]).all()


LENS = [(1, 1), (3, 40), (0, 17), (5, 5), (2, 33), (1, 16), (1, 17)]


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (64, 20), (128, 34), (128, 2), (64, 0)])
@pytest.mark.parametrize("inter", [False, True])
def test_rotation_and_append(io, kv, dim, rot, inter):
    rng = np.random.default_rng(dim + rot + inter)
    c = Call(rng, Batch(rng, LENS, 2, dim, 16, kv, lead=1, tail=2), io, 6, rot, inter, norm=rot % 4 == 0, mscale=1.25)
    c.run()
    c.verify()


@pytest.mark.parametrize("layout", ["page", "head", "both"])
@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
def test_cache_layouts_and_many_heads(layout, io, kv):
    """40 query heads of 5 kv heads: more than a workgroup takes at a time."""
    rng = np.random.default_rng(7)
    c = Call(rng, Batch(rng, [(4, 60), (1, 3)], 5, 128, 32, kv), io, 40, 128, False, norm=True, layout=layout)
    c.run()
    c.verify()


@pytest.mark.parametrize("inter", [False, True])
def test_far_positions(inter):
    """Positions up to 2^31 - 1 and below zero, and frequencies of a stretched context: the angle has to be
    reduced in 64 bits (in 32 it would be off by whole turns)."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [(6, 100)], 2, 128, 16, "f32")
    pos = np.array([0, 1_000_003, 2 ** 31 - 1, -5, -(2 ** 31), 131_071], np.int32)
    f, m = mtg.rope_freqs(128, 1e6, mtg.ROPE_YARN, factor=16.0, orig_ctx=8192)
    c = Call(rng, b, "f32", 4, 128, inter, positions=pos, f=f, mscale=m)
    c.run()
    c.verify()


def test_in_place_and_parts_alone():
    """q turned where it lies in the q|k|v product; q alone (no cache at all); k and v alone."""
    rng = np.random.default_rng(10)
    mk = lambda: Call(rng, Batch(rng, LENS, 2, 128, 16, "f16", tail=1), "f32", 6, 128, False, norm=True)  # noqa: E731
    c = mk()
    c.d.q_out, c.d.q_out_stride = c.d.q, c.d.q_stride
    c.run()
    c.verify(q_out=c.xd[:, :6])
    assert np.array_equal(c.xd[-1].cpu().numpy(), c.x[-1])  # the row of no sequence
    c = mk()
    c.d.k_new = c.d.v_new = None
    c.d.kv.k = c.d.kv.v = c.d.kv.page_table = None
    c.run()
    c.verify(with_kv=False)
    c = mk()
    c.d.q = c.d.q_out = None
    c.run()
    c.verify(with_q=False)
    assert (c.out == 77.0).all()


def test_bad_pages_and_positions_store_nothing():
    """Ids that are no page, rows before position 0 and behind the table: q is turned, nothing is stored.
    (tests/cpp/test_paged_kv.cpp holds the same rule on the CPU.)"""
    rng = np.random.default_rng(11)
    b = Batch(rng, [(4, 40), (5, 20), (6, 4), (3, 18)], 2, 64, 16, "f16", filled=False)
    b.table[0, 2] = b.n_pages       # positions 32 .. 39 of sequence 0
    b.table[1, 1] = 2 ** 31 - 1
    b.table[3, 1] = -2 ** 31
    c = Call(rng, b, "f16", 4, 64, False)
    c.run()
    c.verify()
    b = Batch(rng, [(3, 20)], 2, 64, 16, "f16", filled=False)
    b.kv_len[0] = 16 * b.table.shape[1] + 2   # two of the rows lie behind the table
    c = Call(rng, b, "f16", 4, 64, True)
    c.run()
    c.verify()


def test_many_sequences():
    rng = np.random.default_rng(12)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 3, 4500), rng.integers(0, 4, 4500))]
    c = Call(rng, Batch(rng, lens, 1, 64, 16, "f16", lead=2, tail=3, filled=False), "f16", 2, 64, False)
    c.run()
    c.verify()


def test_non_finite_rows_stay_by_themselves():
    rng = np.random.default_rng(13)
    c = Call(rng, Batch(rng, [(6, 30)], 2, 128, 16, "f32"), "f32", 4, 128, False, norm=True)
    x = c.x.copy()
    x[2, 1] = np.nan            # one head of q
    x[3, 4, 5] = np.inf         # one element of k
    c.xd.copy_(torch.from_numpy(x))
    c.run()
    q = c.out.cpu().numpy()
    assert np.isnan(q[2, 1]).all() and np.isfinite(q[[0, 1, 3, 4, 5]]).all() and np.isfinite(q[2, [0, 2, 3]]).all()
    k, _ = c.cache.read()
    b = c.b
    for i, p in enumerate(range(24, 30)):
        row = k[b.page_of(0, p), :, p % 16]
        assert np.isfinite(row[1]).all() and np.isfinite(row[0]).all() == (i != 3)
    c.x[2, 1] = c.x[3, 4] = 0


def test_another_stream_and_a_captured_call():
    """Captured once and replayed with other rows, positions and lengths, eager work between the replays."""
    rng = np.random.default_rng(14)
    c = Call(rng, Batch(rng, [(2, 20), (1, 9)], 2, 128, 16, "f16"), "f32", 4, 128, False, norm=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c.run(s.cuda_stream)
    c.verify()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        check(mtg.lib().mtg_rope_append_dev(ctypes.byref(c.d), stream()))
    for step in range(4):
        c.x = rng.standard_normal(c.x.shape).astype(np.float32)
        c.xd.copy_(torch.from_numpy(c.x))
        c.b.kv_len = np.array([20 - step, 9 + step], np.int32)
        c.cache.kv_len.copy_(torch.from_numpy(c.b.kv_len))
        c.cache.k.fill_(float("nan"))
        c.cache.v.fill_(float("nan"))
        c.b.k[:], c.b.v[:] = np.nan, np.nan
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        c.verify()


def test_places_beyond_32_bits():
    """Pages 2^31 elements apart: the last one lies 8 GB into the pool."""
    rng = np.random.default_rng(15)
    b = Batch(rng, [(2, 18)], 2, 64, 16, "f16", spare=1)
    b.table[0, :2] = [0, 2]
    c = Call(rng, b, "f16", 4, 64, False)
    far = 1 << 31
    pools = [torch.empty(2 * far + 4096, dtype=torch.float16, device="cuda") for _ in range(2)]
    c.d.kv.k, c.d.kv.v, c.d.kv.page_stride = at(pools[0]), at(pools[1]), far
    c.run()
    b.k[:], b.v[:] = 0, 0
    for p in (0, 2):
        for got, host in ((pools[0], b.k), (pools[1], b.v)):
            host[p] = got[p * far:p * far + 2048].view(2, 16, 64).cpu().numpy()
    for i, p in enumerate((16, 17)):
        y, size = rotate(c.x[i, 4:6], p, c.f, 64, False, 1.0)
        assert (np.abs(b.k[2, :, p - 16] - y) <= rotate_tolerance(y, size, "f16")).all()
        assert np.array_equal(b.v[2, :, p - 16], c.x[i, 6:])
