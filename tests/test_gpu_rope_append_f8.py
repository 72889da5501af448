"""mtg_rope_append_f8_dev on the GPU against the 64-bit form: q, the codes, the scales, and everything that has to stay."""
import ctypes

import numpy as np
import pytest
import torch

import mtg
import serve_ref
import serve_ref_f8 as ref
from serve_dev import TORCH, check, dev, stream
from serve_dev_f8 import Cache, append

pytestmark = pytest.mark.gpu


def run(seed, lens, heads, kv_heads, dim, page, io, rot, inter=False, norm=False, positions=False, mscale=1.0, layout="page", lead=2, tail=3,
        spread=2.0, spoil=None, in_place=False, table=None):
    rng = np.random.default_rng(seed)
    b = ref.Batch(rng, lens, kv_heads, dim, page, lead=lead, tail=tail, spread=spread)
    if table:
        table(b)
    wide = heads + 2 * kv_heads
    x = (rng.standard_normal((b.n_tokens, wide, dim)) * 2.0 ** rng.integers(-6, 6, (b.n_tokens, wide, 1))).astype(serve_ref.TYPES[io])
    if spoil:
        spoil(x)
    pos = rng.integers(-5, 1 << 20, b.n_tokens).astype(np.int32) if positions else None
    f = serve_ref.freqs(rot) if rot else None
    gains = [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) if norm else None for _ in range(2)]
    qkv = dev(x)
    out = qkv[:, :heads] if in_place else torch.full((b.n_tokens, heads, dim), 7.0, dtype=TORCH[io], device="cuda")
    c = Cache(b, layout)
    append(c, qkv, heads, kv_heads, dim, out, io, freqs=None if f is None else dev(f), rot=rot, inter=inter, mscale=mscale,
           positions=None if pos is None else dev(pos), norms=[None if g is None else dev(g) for g in gains])
    torch.cuda.synchronize()
    got = out.float().cpu().numpy().astype(np.float64)
    new_k, size_k = np.full((b.n_tokens, kv_heads, dim), np.nan), np.zeros((b.n_tokens, kv_heads, dim))
    rows = b.positions()
    f64 = np.zeros(0) if f is None else f
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(b.n_tokens):
            if t not in rows:
                want = x[t, :heads] if in_place else np.full((heads, dim), 7.0)
                assert np.array_equal(got[t], want.astype(np.float64), equal_nan=True), t
                continue
            p = int(pos[t]) if positions else rows[t][1]
            y, size = serve_ref.rotate(x[t, :heads], p, f64, rot, inter, mscale, gains[0])
            tol = serve_ref.rotate_tolerance(y, size, io)
            ok = np.isfinite(y) & np.isfinite(size)
            assert (np.abs(got[t] - y)[ok] <= tol[ok]).all(), (t, np.nanmax(np.abs(got[t] - y) / tol))
            assert not np.isfinite(got[t][~ok]).all() or ok.all()
            new_k[t], s = serve_ref.rotate(x[t, heads:heads + kv_heads], p, f64, rot, inter, mscale, gains[1])
            size_k[t] = np.where(np.isfinite(s), s, 0) * 2.0 ** -18  # what 32 bits make of it, as for q
    kc, vc, ks, vs = c.read()
    ref.check_append(b, "k", kc, ks, new_k, size_k)
    ref.check_append(b, "v", vc, vs, x[:, heads + kv_heads:].astype(np.float64), None)


LENS = [(1, 17), (3, 3), (0, 5), (16, 48), (33, 40), (1, 1), (17, 33), (5, 31), (2, 300)]


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("dim,page,layout", [(128, 16, "page"), (128, 64, "head"), (64, 32, "both"), (64, 16, "page"), (128, 32, "both")])
def test_prompts(io, dim, page, layout):
    run(1, LENS, 4, 2, dim, page, io, dim, norm=True, layout=layout)


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 16, 8), (64, 3, 1), (128, 1, 1)])
def test_single_tokens(io, dim, heads, kv_heads):
    run(2, [(1, n) for n in (1, 2, 15, 16, 17, 18, 33, 100)], heads, kv_heads, dim, 16, io, dim, lead=0, tail=0)
    run(3, [(1, 77)], heads, kv_heads, dim, 32, io, dim // 2, inter=True, norm=True, lead=0, tail=0)
    run(4, [(2, 18), (0, 40), (4, 20), (1, 31)] * 20, heads, kv_heads, dim, 32, io, dim, lead=1, tail=1)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rot", [0, 2, 6, 50, 64, 112])
def test_rotated_parts(rot, inter):
    run(5, [(20, 25), (1, 9)], 2, 2, 128, 16, "f32", rot, inter=inter, positions=True, mscale=1.25)
    run(6, [(1, 25), (1, 9)], 2, 2, 128, 16, "f32", rot, inter=inter, positions=True, norm=True)


@pytest.mark.parametrize("spread", [0.0, 12.0, 30.0])
@pytest.mark.parametrize("n", [1, 3, 14])
def test_earlier_rows_of_a_block_follow_its_scale(spread, n):
    """Scales of earlier rows from far below to far above what the new ones need, subnormal codes among the followers."""
    run(7, [(n, n + k) for k in (1, 2, 7, 15, 16, 31)] * 3, 2, 2, 64, 16, "f32", 64, spread=spread)
    run(8, [(n, n + k) for k in (1, 2, 7, 15, 16, 31)] * 3, 2, 2, 128, 32, "f16", 128, spread=spread)


def test_places_that_do_not_exist():
    """Positions below 0, behind the table, pages that are no pages; the neighbours get theirs."""
    def table(b):
        b.table[1, 0] = -1
        b.table[2, 1] = b.n_pages
        b.table[3, 0] = 1 << 30
    run(9, [(9, 4), (20, 40), (40, 40), (1, 5), (3, 20), (1, -4), (40, 90)], 2, 1, 64, 16, "f32", 64, table=table)
    run(10, [(1, 0), (1, 9), (1, 20), (1, 5), (1, 20)], 2, 1, 64, 16, "f32", 64, table=table)

    def short(b):
        b.table = np.ascontiguousarray(b.table[:, :2])
    run(11, [(50, 60), (3, 34)], 2, 1, 64, 16, "f32", 64, table=short)


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("n", [1, 2, 21])
def test_what_is_not_finite_is_nan_alone(io, n):
    def spoil(x):
        x[3::4, :, 5] = np.nan
        x[4::4, :, 9] = np.inf
        x[5::4, :, 11] = -np.inf
        x[6::7] = np.nan
    run(12, [(n, n + 3), (n, n)] * 4, 2, 2, 128, 16, io, 0, spoil=spoil)


def test_large_small_and_zero_rows():
    def spoil(x):
        x[0::6] = 0.0
        x[1::6] *= 1e30
        x[2::6] *= 1e-30
        x[3::6] = 3.4e38
        x[4::6, :, :] = 1e-44
    for n in (1, 19):
        run(13, [(n, n), (n, n + 16), (n, n)] * 3, 2, 2, 64, 16, "f32", 0, spoil=spoil, lead=0, tail=0)


def test_borders_of_a_scale():
    """Largest elements at 448 * 2^e, a step above and a step below: v, which nothing turns, exactly."""
    def spoil(x):
        for i, t in enumerate(range(x.shape[0])):
            top = np.float32(448.0 * 2.0 ** (i % 9 - 4))
            x[t] = np.clip(x[t], -0.5, 0.5)
            x[t, :, i % 64] = [top, np.nextafter(top, np.float32(0)), np.nextafter(top, np.float32(1e9))][i % 3]
    run(14, [(1, 1)] * 40, 1, 1, 64, 16, "f32", 0, spoil=spoil, lead=0, tail=0)


def test_q_in_place_and_alone():
    run(15, LENS, 4, 2, 128, 16, "f32", 128, in_place=True)
    rng = np.random.default_rng(16)
    b = ref.Batch(rng, LENS, 2, 64, 16)
    x = rng.standard_normal((b.n_tokens, 8, 64)).astype(np.float32)
    f = dev(serve_ref.freqs(64))
    c, only = Cache(b), Cache(b)
    out, alone = (torch.zeros(b.n_tokens, 4, 64, device="cuda") for _ in range(2))
    append(c, dev(x), 4, 2, 64, out, "f32", freqs=f, rot=64)
    append(only, dev(x), 4, 2, 64, alone, "f32", freqs=f, rot=64, with_kv=False)
    assert torch.equal(out, alone)
    assert all(np.array_equal(p, q) for p, q in zip(only.read(), (b.kc, b.vc, b.ks, b.vs)))
    append(only, dev(x), 4, 2, 64, None, "f32", freqs=f, rot=64, with_q=False)
    assert all(np.array_equal(p, q) for p, q in zip(only.read(), c.read()))


def test_one_at_a_time_and_all_at_once():
    """The scales are the same; codes differ only where a value was rounded below 2^-6 of a scale before: by that half a step."""
    rng = np.random.default_rng(17)
    n, dim = 40, 128
    x = (rng.standard_normal((n, 3, dim)) * 2.0 ** rng.integers(-9, 3, (n, 1, 1))).astype(np.float32)
    f = dev(serve_ref.freqs(dim))
    whole = ref.Batch(rng, [(n, n)], 1, dim, 16, filled=False)
    a = Cache(whole)
    out = torch.empty(n, 1, dim, device="cuda")
    append(a, dev(x), 1, 1, dim, out, "f32", freqs=f, rot=dim)
    step = Cache(whole)
    step.q_start, step.kv_len = dev(np.array([0, 1], np.int32)), dev(np.array([0], np.int32))
    for t in range(n):
        step.kv_len += 1
        one = torch.empty(1, 1, dim, device="cuda")
        d = append(step, dev(x[t:t + 1]), 1, 1, dim, one, "f32", freqs=f, rot=dim, call=False)
        d.a.kv.n_tokens = 1
        check(mtg.lib().mtg_rope_append_f8_dev(ctypes.byref(d), stream()))
        assert torch.equal(one[0], out[t])
    for got, want, gs, ws in zip(step.read()[:2], a.read()[:2], step.read()[2:], a.read()[2:]):
        used = np.zeros(ws.shape, bool)
        used[whole.table[0, :3]] = True
        assert np.array_equal(gs, ws)
        u, v = (ref.VALUES[np.where(ref.is_nan(c), 0, c)] for c in (got, want))
        assert (np.abs(u - v) <= np.where(np.abs(v) < 2.0 ** -6, 2.0 ** -9, 0)).all()


def test_captured_and_replayed():
    rng = np.random.default_rng(18)
    b = ref.Batch(rng, [(1, 30), (1, 16), (1, 45)], 2, 64, 16, lead=0)
    x, f = dev(rng.standard_normal((3, 8, 64)).astype(np.float32)), dev(serve_ref.freqs(64))
    eager, c = Cache(b), Cache(b)
    out, want = (torch.zeros(3, 4, 64, device="cuda") for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        append(c, x, 4, 2, 64, out, "f32", freqs=f, rot=64)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        append(c, x, 4, 2, 64, out, "f32", freqs=f, rot=64)
    append(eager, x, 4, 2, 64, want, "f32", freqs=f, rot=64)
    for i in range(4):
        x.copy_(dev((2.0 ** i * rng.standard_normal((3, 8, 64))).astype(np.float32)))
        g.replay()
        append(eager, x, 4, 2, 64, want, "f32", freqs=f, rot=64)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(np.array_equal(p, q) for p, q in zip(c.read(), eager.read())), i
