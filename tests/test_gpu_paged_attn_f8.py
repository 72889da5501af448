"""mtg_paged_attn_f8_dev on the GPU against the 64-bit form (serve_ref_f8.attend) with its derived tolerance. What no row
may see are codes NaN and scales of any size: pages of no sequence, places behind a sequence's length, and in tests of
their own the later rows of the same call."""
import ctypes

import numpy as np
import pytest

import mtg
from serve_ref import TYPES
from serve_ref_f8 import Batch, attend, attend_tolerance, is_nan

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import TORCH, at, dev  # noqa: E402
from serve_dev_f8 import Attend, Cache  # noqa: E402

IO = ["f32", "f16"]


def _rows(rng, b, heads, io, sharp=1.0):
    return (sharp * rng.standard_normal((b.n_tokens, heads, b.dim))).astype(TYPES[io])


def _compare(b, q, got, io, scale, window=0, sink=0, rows=None):
    form = attend(b, q, scale, window, sink)
    tol = attend_tolerance(b, q, form, scale, io, max(1, int(b.kv_len.max(initial=1))))
    inside = sorted(b.positions()) if rows is None else rows
    want, tol, got = form[0][inside], tol[inside], got[inside].astype(np.float64)
    if io == "f16":  # 65,520 and more round to infinity
        huge = np.isinf(got)
        assert (np.abs(want) + tol >= 65520)[huge].all() and (np.sign(got) == np.sign(want))[huge].all()
        got = np.where(huge, want, got)
    assert np.isfinite(got).all()
    off = np.abs(got - want)
    assert (off <= tol).all(), float((off / tol).max())


def _run(rng, b, heads, io, window=0, max_kv=0, layout="page", scale=None, sharp=1.0, sink=0):
    if scale is None:  # scores of some units whatever the blocks' scales are
        seen = np.abs(b.k[~np.isnan(b.k)])
        scale = b.dim ** -0.5 / max(1.0, float(np.sqrt((seen ** 2).mean())) if seen.size else 1.0)
    q = _rows(rng, b, heads, io, sharp)
    qd = dev(q)
    out = torch.full_like(qd, 55.0)
    call = Attend(Cache(b, layout), qd, out, io, scale, window, max_kv, sink)
    call()
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    _compare(b, q, got, io, scale, window, sink)
    outside = [t for t in range(b.n_tokens) if t not in b.positions()]
    assert (got[outside] == 55.0).all()
    out.fill_(55.0)
    call()  # the same call, the same bits
    assert np.array_equal(out.cpu().numpy(), got)
    return call


# single tokens, drafts, chunks; lengths around blocks of 16, 32 and 64 keys, tiles of 16 to 128 rows
FEW = [(1, 1), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (1, 200), (0, 50), (1, 129)]
DRAFTS = [(5, 5), (8, 100), (3, 47), (0, 0), (2, 300), (7, 64), (1, 12)]
CHUNK = [(70, 70), (33, 190), (0, 9), (130, 161), (64, 64), (1, 96)]


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 2), (7, 1)])
@pytest.mark.parametrize("lens", [FEW, DRAFTS, CHUNK], ids=["few", "drafts", "chunk"])
def test_against_64_bits(io, dim, heads, kv_heads, lens):
    rng = np.random.default_rng(dim + heads)
    _run(rng, Batch(rng, lens, kv_heads, dim, 16, lead=1, tail=2), heads, io)


@pytest.mark.parametrize("spread", [0.0, 8.0])
@pytest.mark.parametrize("io", IO)
def test_scales_near_and_far(io, spread):
    """All blocks of one size, and sizes up to 2^20 and more apart."""
    rng = np.random.default_rng(int(spread))
    _run(rng, Batch(rng, [(1, 500), (3, 100), (1, 40)], 2, 128, 16, spread=spread), 4, io)
    _run(rng, Batch(rng, [(100, 400), (80, 80)], 2, 128, 32, spread=spread), 4, io)


@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("layout", ["page", "head", "both"])
@pytest.mark.parametrize("io", IO)
def test_pages_and_layouts(page, layout, io):
    rng = np.random.default_rng(page)
    _run(rng, Batch(rng, [(4, 530), (1, 70), (20, 90)], 2, 64, page), 4, io, layout=layout)
    _run(rng, Batch(rng, [(150, 530)], 2, 64, page), 4, io, layout=layout)


@pytest.mark.parametrize("window,sink", [(1, 0), (1, 1), (7, 4), (32, 3), (100, 33), (100, 64), (64, 500), (90, 0), (2 ** 31 - 1, 5), (50, 2 ** 30)])
@pytest.mark.parametrize("io", IO)
def test_windows_and_first_positions(window, sink, io):
    rng = np.random.default_rng(window % 1000 + sink % 1000)
    _run(rng, Batch(rng, [(1, 400), (6, 150), (1, 3), (0, 8), (1, 130)], 2, 128, 16), 4, io, window=window, sink=sink)
    _run(rng, Batch(rng, [(180, 400), (40, 40)], 2, 128, 16), 4, io, window=window, sink=sink)
    _run(rng, Batch(rng, [(20, 333), (30, 90)], 1, 64, 64), 2, io, window=window, sink=sink)


@pytest.mark.parametrize("io", IO)
def test_first_positions_without_a_window_say_nothing(io):
    rng = np.random.default_rng(1)
    for new in (2, 90):
        b = Batch(rng, [(new, 300)], 2, 64, 16)
        q = dev(_rows(rng, b, 4, io))
        outs = [torch.empty_like(q) for _ in range(2)]
        for out, sink in zip(outs, (0, 40)):
            Attend(Cache(b), q, out, io, 0.1, sink=sink)()
        assert torch.equal(*outs)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("new,length", [(1, 6000), (8, 3001), (200, 2500)])
def test_split_keys(io, new, length):
    """Long caches, whose keys several workgroups share; max_kv below and above the real length."""
    rng = np.random.default_rng(length)
    b = Batch(rng, [(new, length), (1, 37)], 1, 128, 64)
    a = _run(rng, b, 2, io, max_kv=length)
    assert a.d.a.workspace_bytes > 0
    _run(rng, b, 2, io, max_kv=700)
    _run(rng, b, 2, io, max_kv=1)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,kv_heads", [([(70, 12000), (1, 300), (2, 5000)], 1), ([(5, 20000), (0, 7), (1, 9000)], 8),
                                           ([(7, 7000)], 1), ([(2, 9000), (9, 4100)], 4)],
                         ids=["rows", "heads", "one", "two"])
def test_many_splits(io, dim, lens, kv_heads):
    """Dozens of splits, which several teams of threads join, in the same launch or in a second one."""
    rng = np.random.default_rng(dim + kv_heads)
    b = Batch(rng, lens, kv_heads, dim, 64, lead=1, tail=1)
    a = _run(rng, b, kv_heads, io, max_kv=max(n for _, n in lens))
    assert a.d.a.workspace_bytes > 0


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("rows", [1, 9])
def test_split_keys_of_many_sequences(io, rows):
    rng = np.random.default_rng(rows)
    lens = [(rows, 40 + 61 * i) for i in range(35)] + [(0, 3000), (rows, rows), (rows, 0)]
    b = Batch(rng, lens, 2, 64, 64)
    assert _run(rng, b, 4, io, max_kv=2200).d.a.workspace_bytes > 0


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("window,sink", [(900, 0), (2049, 4), (3500, 70), (3000, 1200)])
def test_windows_over_splits(io, window, sink):
    """Splits that begin at a window's edge or among the first positions; rows of one tile whose first key lies in another split."""
    rng = np.random.default_rng(window)
    for lens in ([(3, 5000), (1, 700), (0, 9)], [(150, 4100), (2, 2000)], [(20, 3333)]):
        b = Batch(rng, lens, 2, 64, 32)
        _run(rng, b, 4, io, window=window, sink=sink)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("new", [1, 6, 150])
def test_splits_without_a_page(io, new):
    rng = np.random.default_rng(new)
    b = Batch(rng, [(new, 4000), (new, 2500)], 2, 64, 16)
    b.table[0, :70], b.table[0, 130:200], b.table[0, 230:] = -1, b.n_pages, -5
    _run(rng, b, 4, io)
    b.table[0, :], b.table[1, 1:] = -1, -1
    b.table[0, 100] = b.table[1, 0]
    _run(rng, b, 4, io)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [64, 128])
def test_batches_of_short_contexts(io, dim):
    rng = np.random.default_rng(dim)
    lens = [(1, 1), (1, 257), (2, 256), (0, 40), (1, 511), (3, 513), (1, 700), (2, 90), (1, 33), (1, 255), (1, 288), (2, 31),
            (1, 600), (1, 449), (3, 2), (1, 0), (1, 420)]
    b = Batch(rng, lens, 8, dim, 16, lead=1, tail=3)
    _run(rng, b, 16, io, max_kv=700)
    _run(rng, b, 16, io, max_kv=700, window=300)
    _run(rng, b, 16, io, max_kv=700, window=100, sink=4)
    _run(rng, b, 16, io, max_kv=300)
    b.table[4, 3], b.table[4, 20], b.table[6, :30] = -1, b.n_pages, -9
    _run(rng, b, 16, io, max_kv=700)


@pytest.mark.parametrize("io", IO)
def test_one_key_over_the_rest(io):
    """Scores far apart: the running maximum moves late and far, most weights vanish."""
    rng = np.random.default_rng(3)
    b = Batch(rng, [(1, 500), (3, 260), (160, 300)], 1, 128, 32)
    for s in range(3):
        for p in (0, 40, 200, 255):
            b.ks[b.page_of(s, p), :, p % b.page // 16] += 3
    b.values()
    _run(rng, b, 4, io, sharp=3.0)
    _run(rng, b, 4, io, scale=0.0)
    _run(rng, b, 4, io, scale=-0.02)


@pytest.mark.parametrize("io", IO)
def test_rows_without_keys(io):
    rng = np.random.default_rng(4)
    for lens in ([(5, 3), (4, 0), (2, 2)], [(150, 20), (10, 0)]):
        _run(rng, Batch(rng, lens, 2, 64, 16), 4, io)
        _run(rng, Batch(rng, lens, 2, 64, 16), 4, io, window=2, sink=1)
    b = Batch(rng, [(3, 40), (70, 200)], 2, 64, 16)
    b.table[:] = -1
    _run(rng, b, 4, io)
    b.kv_len[:] = -2 ** 31
    _run(rng, b, 4, io)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("new", [2, 150])
def test_bad_pages_take_no_part(io, new):
    rng = np.random.default_rng(5)
    b = Batch(rng, [(new, 300), (new, 170)], 2, 128, 16)
    b.table[0, 3], b.table[0, 7], b.table[1, 0] = -1, b.n_pages, 2 ** 31 - 1
    b.table[1, 1:4] = -2 ** 31
    _run(rng, b, 4, io)
    _run(rng, b, 4, io, window=40, sink=60)
    b = Batch(rng, [(new, 304)], 2, 128, 16)
    b.table = np.ascontiguousarray(b.table[:, :19])
    b.kv_len[0] = 304 + new - 1   # only the first row's position is in the table; the others see all it holds
    _run(rng, b, 4, io)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,at_", [(9, 3), (9, 0), (150, 40), (150, 149), (150, 0)])
def test_later_rows_do_not_reach_earlier_ones(io, dim, new, at_):
    """K and V of one new row are NaN: the rows before it are as if it were not there, the rows from it on
    are not finite where V is not. A window hides it again from rows further on, the first positions do not."""
    rng = np.random.default_rng(6)
    b = Batch(rng, [(new, new + 45)], 2, dim, 16)
    q = _rows(rng, b, 4, io)
    p = 45 + at_
    place = (b.page_of(0, p), slice(None), p % 16)
    good = [b.kc[place].copy(), b.vc[place].copy()]
    for hurt_k in (False, True):
        for window, sink in ((0, 0), (20, 0), (20, p), (20, p + 1)):
            b.kc[place], b.vc[place] = good
            b.vc[place][:, 5], b.vc[place][:, dim - 9] = 127, 255
            if hurt_k:
                b.kc[place] = 255
            qd = dev(q)
            out = torch.empty_like(qd)
            Attend(Cache(b), qd, out, io, 0.01, window, sink=sink)()
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            b.kc[place], b.vc[place] = good
            seen = [t for t in range(new) if t >= at_ and (not window or t < at_ + window or p < sink)]
            _compare(b, q, got, io, 0.01, window, sink, rows=[t for t in range(new) if t not in seen])
            assert not np.isfinite(got[seen][:, :, [5, dim - 9]]).any()
            if not hurt_k:
                assert np.isfinite(np.delete(got[seen], [5, dim - 9], axis=2)).all()


def test_scales_that_no_row_sees():
    """A sequence's later blocks, beyond every row's position, hold scales of 255 and codes NaN."""
    rng = np.random.default_rng(7)
    for new in (1, 5, 100):
        b = Batch(rng, [(new, 333)], 2, 64, 32, filled=True)
        b.kv_len[0] = 301
        for x in range(304, 333):
            b.kc[b.page_of(0, x), :, x % 32] = 127
            b.vc[b.page_of(0, x), :, x % 32] = 255
            b.ks[b.page_of(0, x), :, x % 32 // 16] = 255
            b.vs[b.page_of(0, x), :, x % 32 // 16] = 255
        _run(rng, b, 4, "f32")


def test_non_finite_queries_stay_by_themselves():
    rng = np.random.default_rng(7)
    for new in (4, 140):
        for io in IO:
            b = Batch(rng, [(new, 200)], 2, 64, 16)
            q = _rows(rng, b, 4, io)
            clean = q.copy()
            q[1, 2] = np.nan
            q[3, 0, 7] = np.inf
            qd = dev(q)
            out = torch.empty_like(qd)
            Attend(Cache(b), qd, out, io, 0.02)()
            got = out.cpu().numpy()
            assert not np.isfinite(got[1, 2]).any() and not np.isfinite(got[3, 0]).any()
            form = attend(b, clean, 0.02)
            tol = attend_tolerance(b, clean, form, 0.02, io, 200)
            got[1, 2], got[3, 0], form[0][1, 2], form[0][3, 0] = 0, 0, 0, 0
            assert (np.abs(got - form[0]) <= tol).all()


@pytest.mark.parametrize("scale", [-60, -90, 20, 60])
def test_caches_of_any_size(scale):
    """All scales 2^-60 to 2^60 away from one: K against the rows' scale, V in the result."""
    rng = np.random.default_rng(8)
    for new in (2, 140):
        b = Batch(rng, [(new, 260)], 1, 128, 16)
        rms = float(np.sqrt(np.nanmean(b.k ** 2)))
        b.ks[:], b.vs[:] = np.clip(b.ks.astype(int) + scale, 0, 254), np.clip(b.vs.astype(int) + scale, 0, 254)
        b.values()
        _run(rng, b, 2, "f32", scale=0.09 / rms * 2.0 ** -scale)


def test_strided_rows_and_in_place():
    rng = np.random.default_rng(9)
    for new in (3, 150):
        for io in IO:
            b = Batch(rng, [(new, 100), (1, 60)], 2, 64, 16, tail=1)
            wide = dev(rng.standard_normal((b.n_tokens, 10, 64)).astype(TYPES[io]))
            host = wide.cpu().numpy()
            Attend(Cache(b), wide[:, :4], wide[:, :4], io, 0.02)()
            torch.cuda.synchronize()
            got = wide.cpu().numpy()
            assert np.array_equal(got[:, 4:], host[:, 4:]) and np.array_equal(got[-1], host[-1])
            _compare(b, host[:, :4], got[:, :4], io, 0.02)
            out = torch.zeros(b.n_tokens, 6, 64, dtype=TORCH[io], device="cuda")
            Attend(Cache(b), dev(host)[:, 2:6], out[:, 1:5], io, 0.02)()
            got = out.cpu().numpy()
            assert (got[:, [0, 5]] == 0).all()
            _compare(b, host[:, 2:6], got[:, 1:5], io, 0.02)


def test_many_sequences_and_starts_that_make_no_sense():
    rng = np.random.default_rng(10)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 3, 4400), rng.integers(0, 20, 4400))]
    b = Batch(rng, lens, 1, 64, 16, lead=1, tail=2)
    _run(rng, b, 2, "f16")
    b = Batch(rng, [(3, 40), (2, 30), (4, 50)], 1, 64, 16)
    b.q_start[:] = [5, 2, 2 ** 31 - 1, -7]
    q = dev(_rows(rng, b, 2, "f16"))
    guard = torch.full((b.n_tokens + 8, 2, 64), 3.0, dtype=torch.float16, device="cuda")
    Attend(Cache(b), q, guard[4:-4], "f16", 0.02)()
    torch.cuda.synchronize()
    assert (guard[:4] == 3.0).all() and (guard[-4:] == 3.0).all()


def test_streams_graphs_and_workspaces():
    """Two captured calls with a workspace each, replayed on two streams at once and with new lengths, queries and
    eager calls between; each replay against the eager result and the 64-bit form."""
    rng = np.random.default_rng(11)
    b = Batch(rng, [(1, 3000), (2, 1500)], 1, 128, 16)
    cache = Cache(b)
    sides = []
    for i in range(2):
        q = dev(_rows(rng, b, 2, "f32"))
        out = torch.empty_like(q)
        call = Attend(cache, q, out, "f32", 0.02, max_kv=3000)
        assert call.d.a.workspace_bytes
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        call(s.cuda_stream)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(s.cuda_stream)
        sides.append((q, out, call, s, g))
    eager_out = torch.empty_like(sides[0][1])
    for step in range(4):
        b.kv_len = np.array([3000 - 700 * step, 3 + 499 * step], np.int32)
        cache.kv_len.copy_(torch.from_numpy(b.kv_len))
        hosts = []
        for q, *_ in sides:
            hosts.append(_rows(rng, b, 2, "f32"))
            q.copy_(torch.from_numpy(hosts[-1]))
        torch.cuda.synchronize()
        for _, _, _, s, g in sides:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (q, out, *_), host in zip(sides, hosts):
            Attend(cache, q, eager_out, "f32", 0.02, max_kv=3000)()
            torch.cuda.synchronize()
            assert torch.equal(eager_out, out)
            _compare(b, host, out.cpu().numpy(), "f32", 0.02)


def test_places_beyond_32_bits():
    """Pages 2^32 bytes apart, and their scales."""
    rng = np.random.default_rng(12)
    far = 1 << 32
    pools = [torch.empty(2 * far + 4096, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for new in (1, 30):
        b = Batch(rng, [(new, 40)], 2, 64, 16, spare=0)
        b.table[0, :3] = [1, 0, 2]
        b.n_pages = 3
        for codes, scales in ((b.kc, b.ks), (b.vc, b.vs)):  # every place holds a number, for the pages are exchanged
            codes[:] = rng.integers(0, 127, codes.shape) + 128 * rng.integers(0, 2, codes.shape)
            scales[:] = rng.integers(120, 124, scales.shape)
        b.values()
        for pool, host in zip(pools, (b.kc, b.vc)):
            for p in range(3):
                pool[p * far:p * far + 2048] = dev(host[p]).view(-1)
        scales = [torch.full((2 * far + 16,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
        for pool, host in zip(scales, (b.ks, b.vs)):
            for p in range(3):
                pool[p * far:p * far + 2] = dev(host[p]).view(-1)
        q = _rows(rng, b, 4, "f16")
        qd = dev(q)
        out = torch.empty_like(qd)
        call = Attend(Cache(b), qd, out, "f16", 0.02)
        call.d.a.kv.k, call.d.a.kv.v, call.d.a.kv.page_stride = at(pools[0]), at(pools[1]), far
        call.d.scales = mtg.F8Scales(k=at(scales[0]), v=at(scales[1]), page_stride=far, head_stride=1)
        call()
        torch.cuda.synchronize()
        _compare(b, q, out.cpu().numpy(), "f16", 0.02)
        assert not is_nan(b.kc[b.table[0, 0], :, 0]).any()
        del scales
