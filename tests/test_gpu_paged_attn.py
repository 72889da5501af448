"""mtg_paged_attn_dev on the GPU against the 64-bit form (serve_ref.attend), with serve_ref's derived
tolerance. Everything that no row may see is NaN: pages of no sequence, places behind a sequence's
length, and in tests of their own the later rows of the same call."""
import ctypes

import numpy as np
import pytest

import mtg
from serve_ref import Batch, TYPES, attend, attend_tolerance

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import TORCH, Attend, Cache, at, dev  # noqa: E402

TYPE_PAIRS = [("f32", "f16"), ("f16", "f16"), ("f32", "f32")]


def _rows(rng, b, heads, io, sharp=1.0):
    return (sharp * rng.standard_normal((b.n_tokens, heads, b.dim))).astype(TYPES[io])


def _compare(b, q, got, io, scale, window=0, rows=None):
    want, size, sharp = attend(b, q, scale, window)
    tol = attend_tolerance(want, size, sharp, io, max(1, int(b.kv_len.max(initial=1))), b.dim)
    inside = sorted(b.positions()) if rows is None else rows
    assert np.isfinite(got[inside]).all()
    off = np.abs(got[inside].astype(np.float64) - want[inside])
    assert (off <= tol[inside]).all(), float((off / tol[inside]).max())


def _run(rng, b, heads, io, window=0, max_kv=0, layout="page", scale=None, sharp=1.0):
    scale = b.dim ** -0.5 if scale is None else scale
    q = _rows(rng, b, heads, io, sharp)
    qd = dev(q)
    out = torch.full_like(qd, 55.0)
    call = Attend(Cache(b, layout), qd, out, io, scale, window, max_kv)
    call()
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    _compare(b, q, got, io, scale, window)
    outside = [t for t in range(b.n_tokens) if t not in b.positions()]
    assert (got[outside] == 55.0).all()
    out.fill_(55.0)
    call()  # the same call, the same bits
    assert np.array_equal(out.cpu().numpy(), got)
    return call


# single tokens, drafts, chunks; lengths around pages, blocks of 32 and 64 keys, tiles of 16 to 128 rows
FEW = [(1, 1), (1, 16), (1, 17), (1, 31), (1, 32), (1, 33), (1, 200), (0, 50), (1, 129)]
DRAFTS = [(5, 5), (8, 100), (3, 47), (0, 0), (2, 300), (7, 64), (1, 12)]
CHUNK = [(70, 70), (33, 190), (0, 9), (130, 161), (64, 64), (1, 96)]


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 2), (7, 1)])
@pytest.mark.parametrize("lens", [FEW, DRAFTS, CHUNK], ids=["few", "drafts", "chunk"])
def test_against_64_bits(io, kv, dim, heads, kv_heads, lens):
    rng = np.random.default_rng(dim + heads)
    _run(rng, Batch(rng, lens, kv_heads, dim, 16, kv, lead=1, tail=2), heads, io)


@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("layout", ["page", "head", "both"])
@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
def test_pages_and_layouts(page, layout, io, kv):
    rng = np.random.default_rng(page)
    _run(rng, Batch(rng, [(4, 530), (1, 70), (20, 90)], 2, 64, page, kv), 4, io, layout=layout)
    _run(rng, Batch(rng, [(150, 530)], 2, 64, page, kv), 4, io, layout=layout)


@pytest.mark.parametrize("window", [1, 7, 32, 100, 2 ** 31 - 1])
@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
def test_windows(window, io, kv):
    rng = np.random.default_rng(window % 1000)
    _run(rng, Batch(rng, [(1, 400), (6, 150), (1, 3), (0, 8)], 2, 128, 16, kv), 4, io, window=window)
    _run(rng, Batch(rng, [(180, 400), (40, 40)], 2, 128, 16, kv), 4, io, window=window)


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("new,length", [(1, 6000), (8, 3001), (200, 2500)])
def test_split_keys(io, kv, new, length):
    """Long caches, whose keys several workgroups share; max_kv below and above the real length."""
    rng = np.random.default_rng(length)
    b = Batch(rng, [(new, length), (1, 37)], 1, 128, 64, kv)
    a = _run(rng, b, 2, io, max_kv=length)
    assert a.d.workspace_bytes > 0
    _run(rng, b, 2, io, max_kv=700)
    _run(rng, b, 2, io, max_kv=1)


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,kv_heads", [([(70, 12000), (1, 300), (2, 5000)], 1), ([(5, 20000), (0, 7), (1, 9000)], 8),
                                           ([(7, 7000)], 1), ([(2, 9000), (9, 4100)], 4)],
                         ids=["rows", "heads", "one", "two"])
def test_many_splits(io, kv, dim, lens, kv_heads):
    """Dozens of splits, which several teams of threads join, in the same launch or in a second one."""
    rng = np.random.default_rng(dim + kv_heads)
    b = Batch(rng, lens, kv_heads, dim, 64, kv, lead=1, tail=1)
    a = _run(rng, b, kv_heads, io, max_kv=max(n for _, n in lens))
    assert a.d.workspace_bytes > 0


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("rows", [1, 9])
def test_split_keys_of_many_sequences(io, kv, rows):
    """More workgroups than the chip takes at once: the splits are joined by a second launch; sequences of one
    split, of several and of none among them. Then the same in one launch (a small max_kv), over the same workspace."""
    rng = np.random.default_rng(rows)
    lens = [(rows, 40 + 61 * i) for i in range(35)] + [(0, 3000), (rows, rows), (rows, 0)]
    b = Batch(rng, lens, 2, 64, 64, kv)
    a = _run(rng, b, 4, io, max_kv=2200)
    assert a.d.workspace_bytes > 0
    a.d.max_kv = 1100
    assert mtg.lib().mtg_paged_attn_workspace(ctypes.byref(a.d)) <= a.d.workspace_bytes
    cache, q, out = a.keep
    want = out.cpu().numpy()
    for _ in range(2):
        out.zero_()
        a()
        off = np.abs(out.cpu().numpy().astype(np.float64) - want)
        assert off.max() <= 4e-3 * np.abs(want).max() if io == "f16" else off.max() <= 1e-5 * np.abs(want).max()


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("window", [900, 2049, 3500])
def test_windows_over_splits(io, kv, window):
    """Splits that begin at a window's edge; rows of one tile whose first key lies in another split."""
    rng = np.random.default_rng(window)
    for lens in ([(3, 5000), (1, 700), (0, 9)], [(150, 4100), (2, 2000)], [(20, 3333)]):
        b = Batch(rng, lens, 2, 64, 32, kv)
        _run(rng, b, 4, io, window=window)


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("new", [1, 6, 150])
def test_splits_without_a_page(io, kv, new):
    """Whole splits none of whose keys lies in a page, the first and the last among them; then one page of all."""
    rng = np.random.default_rng(new)
    b = Batch(rng, [(new, 4000), (new, 2500)], 2, 64, 16, kv)
    b.table[0, :70], b.table[0, 130:200], b.table[0, 230:] = -1, b.n_pages, -5
    _run(rng, b, 4, io)
    b.table[0, :], b.table[1, 1:] = -1, -1
    b.table[0, 100] = b.table[1, 0]
    _run(rng, b, 4, io)


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
def test_batches_of_short_contexts(io, kv, dim):
    """As many workgroups as half the chip takes: lengths around blocks and around what one round of the waves takes,
    single rows and drafts, empty ones, missing pages, windows, lengths beyond max_kv; later rows that are not finite."""
    rng = np.random.default_rng(dim)
    lens = [(1, 1), (1, 257), (2, 256), (0, 40), (1, 511), (3, 513), (1, 700), (2, 90), (1, 33), (1, 255), (1, 288), (2, 31),
            (1, 600), (1, 449), (3, 2), (1, 0), (1, 420)]
    b = Batch(rng, lens, 8, dim, 16, kv, lead=1, tail=3)
    assert _run(rng, b, 16, io, max_kv=700).d.workspace_bytes == 0
    _run(rng, b, 16, io, max_kv=700, window=300)
    _run(rng, b, 16, io, max_kv=300)
    b.table[4, 3], b.table[4, 20], b.table[6, :30] = -1, b.n_pages, -9
    _run(rng, b, 16, io, max_kv=700)
    for s in (5, 2, 14):   # of their new rows only the last one sees this key
        p = int(b.kv_len[s]) - 1
        b.v[(b.page_of(s, p), slice(None), p % 16)] = np.inf
    q = _rows(rng, b, 16, io)
    qd = dev(q)
    out = torch.empty_like(qd)
    Attend(Cache(b), qd, out, io, 0.1, max_kv=700)()
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    last = [int(b.q_start[s + 1]) - 1 for s in (5, 2, 14)]
    assert np.isinf(got[last]).all()
    _compare(b, q, got, io, 0.1, rows=[t for t in sorted(b.positions()) if t not in last])


def test_calls_side_by_side_with_a_workspace_each():
    """Two streams at once, joins in the same launch and in a second one; each call as alone."""
    rng = np.random.default_rng(12)
    calls, want = [], []
    for lens, kv_heads in (([(1, 3000), (2, 1700)], 2), ([(5, 9000), (3, 8000)], 8), ([(90, 2600)], 2)):
        b = Batch(rng, lens, kv_heads, 64, 64, "f16")
        q = dev(_rows(rng, b, 2 * kv_heads, "f16"))
        for _ in range(2):
            calls.append(Attend(Cache(b), q, torch.empty_like(q), "f16", 0.125))
            calls[-1]()
            torch.cuda.synchronize()
            want.append(calls[-1].keep[2].cpu().numpy())
            calls[-1].keep[2].zero_()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, call in enumerate(calls):
            with torch.cuda.stream(streams[i % 2]):
                call()
    torch.cuda.synchronize()
    for call, w in zip(calls, want):
        assert np.array_equal(call.keep[2].cpu().numpy(), w)


def test_a_workspace_of_any_content():
    """What lies in a fresh workspace, zeros, ones or another call's leavings, does not matter."""
    rng = np.random.default_rng(2)
    b = Batch(rng, [(1, 900), (2, 700)], 2, 128, 32, "f16")
    q = _rows(rng, b, 4, "f16")
    qd = dev(q)
    out = torch.empty_like(qd)
    call = Attend(Cache(b), qd, out, "f16", 0.1)
    other = Attend(Cache(b), qd, torch.empty_like(qd), "f16", 0.2, max_kv=800)
    assert call.d.workspace_bytes >= other.d.workspace_bytes > 0
    other.d.workspace, other.d.workspace_bytes = call.d.workspace, call.d.workspace_bytes
    for fill in (0, 1, 127, 255):
        call.work.fill_(fill)
        out.zero_()
        call()
        torch.cuda.synchronize()
        _compare(b, q, out.cpu().numpy(), "f16", 0.1)
    for _ in range(3):
        other()
        out.zero_()
        call()
        torch.cuda.synchronize()
        _compare(b, q, out.cpu().numpy(), "f16", 0.1)


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
def test_one_key_over_the_rest(io, kv):
    """Scores far apart: the running maximum moves late and far, most weights vanish."""
    rng = np.random.default_rng(3)
    b = Batch(rng, [(1, 500), (3, 260), (160, 300)], 1, 128, 32, kv)
    for s in range(3):
        for p in (0, 40, 200, 255):
            page = b.page_of(s, p)
            b.k[page, :, p % b.page] *= TYPES[kv](6.0)
    _run(rng, b, 4, io, sharp=3.0)
    _run(rng, b, 4, io, scale=0.0)
    _run(rng, b, 4, io, scale=-0.2)


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
def test_rows_without_keys(io, kv):
    """More new rows than positions: the rows before position 0 see nothing and give zeros; no pages at all."""
    rng = np.random.default_rng(4)
    for lens in ([(5, 3), (4, 0), (2, 2)], [(150, 20), (10, 0)]):
        b = Batch(rng, lens, 2, 64, 16, kv)
        _run(rng, b, 4, io)
    b = Batch(rng, [(3, 40), (70, 200)], 2, 64, 16, kv)
    b.table[:] = -1
    _run(rng, b, 4, io)
    b.kv_len[:] = -2 ** 31
    _run(rng, b, 4, io)


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("new", [2, 150])
def test_bad_pages_take_no_part(io, kv, new):
    """(tests/cpp/test_paged_kv.cpp holds the rule on the CPU.) Ids outside the pool, and lengths behind the table."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [(new, 300), (new, 170)], 2, 128, 16, kv)
    b.table[0, 3], b.table[0, 7], b.table[1, 0] = -1, b.n_pages, 2 ** 31 - 1
    b.table[1, 1:4] = -2 ** 31
    _run(rng, b, 4, io)
    b = Batch(rng, [(new, 304)], 2, 128, 16, kv)
    b.table = np.ascontiguousarray(b.table[:, :19])
    b.kv_len[0] = 304 + new - 1   # only the first row's position is in the table; the others see all it holds
    _run(rng, b, 4, io)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("new,at_", [(9, 3), (150, 40), (150, 149), (150, 0)])
def test_later_rows_do_not_reach_earlier_ones(bad, io, kv, new, at_):
    """K and V of one new row are not finite: the rows before it are as if it were not there, the rows from it on
    are not finite where V is not. A window hides it again from rows further on."""
    rng = np.random.default_rng(6)
    b = Batch(rng, [(new, new + 45)], 2, 128, 16, kv)
    q = _rows(rng, b, 4, io)
    p = 45 + at_
    place = (b.page_of(0, p), slice(None), p % 16)
    good = [b.k[place].copy(), b.v[place].copy()]
    for hurt_k in (False, True):
        for window in (0, 20):
            b.k[place], b.v[place] = good
            b.v[place][:, 5] = bad
            if hurt_k:
                b.k[place] = bad
            qd = dev(q)
            out = torch.empty_like(qd)
            Attend(Cache(b), qd, out, io, 0.1, window)()
            torch.cuda.synchronize()
            got = out.cpu().numpy()
            b.k[place], b.v[place] = good
            seen = [t for t in range(new) if t >= at_ and (not window or t < at_ + window)]
            _compare(b, q, got, io, 0.1, window, rows=[t for t in range(new) if t not in seen])
            assert not np.isfinite(got[seen][:, :, 5]).any()


def test_non_finite_queries_stay_by_themselves():
    rng = np.random.default_rng(7)
    for new in (4, 140):
        for io, kv in TYPE_PAIRS:
            b = Batch(rng, [(new, 200)], 2, 64, 16, kv)
            q = _rows(rng, b, 4, io)
            clean = q.copy()
            q[1, 2] = np.nan
            q[3, 0, 7] = np.inf
            qd = dev(q)
            out = torch.empty_like(qd)
            Attend(Cache(b), qd, out, io, 0.125)()
            got = out.cpu().numpy()
            assert not np.isfinite(got[1, 2]).any() and not np.isfinite(got[3, 0]).any()
            got[1, 2], got[3, 0] = 0, 0
            want, size, sharp = attend(b, clean, 0.125)
            tol = attend_tolerance(want, size, sharp, io, 200, 64)
            want[1, 2], want[3, 0] = 0, 0
            assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("scale", [1e-6, 1.0, 3e4])
def test_rows_of_any_size(scale):
    """f32 rows and caches keep their precision where f16 would not hold them: values of 1e-6 and of 3e4."""
    rng = np.random.default_rng(8)
    for kv in ("f32", "f16"):
        for new in (2, 140):
            b = Batch(rng, [(new, 260)], 1, 128, 16, kv)
            if kv == "f32":
                b.v *= np.float32(scale)
                b.k *= np.float32(scale)
                _run(rng, b, 2, "f32", scale=0.09 / scale)
            else:
                q = np.float32(scale)
                _run(rng, b, 2, "f32", scale=0.09 / scale, sharp=q)


def test_strided_rows_and_in_place():
    """q as a slice of a wider product with its result in place, and an out with rows of its own stride."""
    rng = np.random.default_rng(9)
    for new in (3, 150):
        for io, kv in TYPE_PAIRS:
            b = Batch(rng, [(new, 100), (1, 60)], 2, 64, 16, kv, tail=1)
            wide = dev(rng.standard_normal((b.n_tokens, 10, 64)).astype(TYPES[io]))
            host = wide.cpu().numpy()
            Attend(Cache(b), wide[:, :4], wide[:, :4], io, 0.125)()
            torch.cuda.synchronize()
            got = wide.cpu().numpy()
            assert np.array_equal(got[:, 4:], host[:, 4:]) and np.array_equal(got[-1], host[-1])
            _compare(b, host[:, :4], got[:, :4], io, 0.125)
            out = torch.zeros(b.n_tokens, 6, 64, dtype=TORCH[io], device="cuda")
            Attend(Cache(b), dev(host)[:, 2:6], out[:, 1:5], io, 0.125)()
            got = out.cpu().numpy()
            assert (got[:, [0, 5]] == 0).all()
            _compare(b, host[:, 2:6], got[:, 1:5], io, 0.125)


def test_many_sequences_and_starts_that_make_no_sense():
    rng = np.random.default_rng(10)
    lens = [(int(n), int(n + k)) for n, k in zip(rng.integers(0, 3, 4400), rng.integers(0, 20, 4400))]
    b = Batch(rng, lens, 1, 64, 16, "f16", lead=1, tail=2)
    _run(rng, b, 2, "f16")
    # descending and outside starts: nothing outside the buffers is touched, the call returns
    b = Batch(rng, [(3, 40), (2, 30), (4, 50)], 1, 64, 16, "f16")
    b.q_start[:] = [5, 2, 2 ** 31 - 1, -7]
    q = dev(_rows(rng, b, 2, "f16"))
    guard = torch.full((b.n_tokens + 8, 2, 64), 3.0, dtype=torch.float16, device="cuda")
    Attend(Cache(b), q, guard[4:-4], "f16", 0.125)()
    torch.cuda.synchronize()
    assert (guard[:4] == 3.0).all() and (guard[-4:] == 3.0).all()


def test_streams_graphs_and_workspaces():
    """Two captured calls with a workspace each, replayed on two streams at once and with new lengths, queries and
    eager calls between; each replay against the eager result and the 64-bit form."""
    rng = np.random.default_rng(11)
    b = Batch(rng, [(1, 3000), (2, 1500)], 1, 128, 16, "f16")
    cache = Cache(b)
    sides = []
    for i in range(2):
        q = dev(_rows(rng, b, 2, "f32"))
        out = torch.empty_like(q)
        call = Attend(cache, q, out, "f32", 0.1, max_kv=3000)
        assert call.d.workspace_bytes
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
            eager = Attend(cache, q, eager_out, "f32", 0.1, max_kv=3000)
            eager()
            torch.cuda.synchronize()
            assert torch.equal(eager_out, out)
            _compare(b, host, out.cpu().numpy(), "f32", 0.1)


def test_places_beyond_32_bits():
    """Pages 2^31 elements apart: the last one lies 8 GB into the pool."""
    rng = np.random.default_rng(12)
    far = 1 << 31
    pools = [torch.empty(2 * far + 4096, dtype=torch.float16, device="cuda") for _ in range(2)]
    for new in (1, 30):
        b = Batch(rng, [(new, 40)], 2, 64, 16, "f16", spare=0)
        b.table[0, :3] = [1, 0, 2]
        b.n_pages = 3
        for x in (b.k, b.v):
            x[:] = rng.standard_normal(x.shape)
        for pool, host in zip(pools, (b.k, b.v)):
            for p in range(3):
                pool[p * far:p * far + 2048] = dev(host[p]).view(-1)
        q = _rows(rng, b, 4, "f16")
        out = torch.empty_like(dev(q))
        qd = dev(q)
        call = Attend(Cache(b), qd, out, "f16", 0.125)
        call.d.kv.k, call.d.kv.v, call.d.kv.page_stride = at(pools[0]), at(pools[1]), far
        call()
        torch.cuda.synchronize()
        _compare(b, q, out.cpu().numpy(), "f16", 0.125)
