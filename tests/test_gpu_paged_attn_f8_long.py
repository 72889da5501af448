"""mtg_paged_attn_f8_dev with 1,024 pairs of rows and heads or more to a sequence, which a kernel of its own takes 256 at a
time, against the 64-bit form with its derived tolerance."""
import numpy as np
import pytest

from serve_ref_f8 import Batch, attend, attend_tolerance
from test_gpu_paged_attn_f8 import IO, _compare, _rows, _run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import dev  # noqa: E402
from serve_dev_f8 import Attend, Cache  # noqa: E402

# (rows, keys) of each sequence, heads, heads of k and v: on average 1,024 pairs and more, ends on and beside tiles
SHAPES = [([(147, 147)], 7, 1), ([(300, 1100), (0, 9), (160, 161)], 7, 1), ([(512, 512)], 2, 1), ([(513, 640), (511, 530)], 2, 1),
          ([(70, 900), (60, 64), (65, 65)], 32, 2), ([(1024, 1030)], 2, 2), ([(64, 300), (1, 40), (150, 150)], 16, 1)]


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads,kv_heads", SHAPES)
def test_against_64_bits(io, dim, lens, heads, kv_heads):
    rng = np.random.default_rng(dim + heads)
    b = Batch(rng, lens, kv_heads, dim, 16, lead=1, tail=2)
    _run(rng, b, heads, io)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("layout,page", [("page", 64), ("head", 16), ("both", 512)])
def test_layouts_and_scales_far_apart(io, layout, page):
    rng = np.random.default_rng(page)
    b = Batch(rng, [(150, 777), (150, 152)], 1, 128, page, spread=6.0)
    _run(rng, b, 7, io, layout=layout)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sink", [(1, 0), (1, 1), (33, 4), (100, 70), (200, 1000), (600, 300), (900, 0)])
def test_windows_and_first_positions(io, dim, window, sink):
    rng = np.random.default_rng(window + sink)
    b = Batch(rng, [(150, 1500), (147, 147)], 1, dim, 32)
    _run(rng, b, 7, io, window=window, sink=sink)


@pytest.mark.parametrize("io", IO)
def test_split_and_whole(io):
    """One tile's sequences over many keys (split), and so many sequences that none is split."""
    rng = np.random.default_rng(2)
    _run(rng, Batch(rng, [(64, 6000)], 1, 64, 16), 16, io)
    lens = [(64 + i % 3, 300 + 41 * i) for i in range(12)]
    _run(rng, Batch(rng, lens, 2, 64, 64), 32, io, max_kv=800)


@pytest.mark.parametrize("io", IO)
def test_bad_pages_and_rows_without_keys(io):
    rng = np.random.default_rng(5)
    b = Batch(rng, [(150, 900), (150, 170)], 1, 128, 16)
    b.table[0, 3], b.table[0, 20:40], b.table[1, 0] = -1, b.n_pages, 2 ** 31 - 1
    b.table[1, 1:4] = -2 ** 31
    _run(rng, b, 7, io)
    _run(rng, b, 7, io, window=40, sink=60)
    _run(rng, Batch(rng, [(150, 20), (160, 0)], 1, 64, 16), 7, io)  # most rows lie before the first position
    b.table[:] = -1
    _run(rng, b, 7, io)
    b.kv_len[:] = -2 ** 31
    _run(rng, b, 7, io)


@pytest.mark.parametrize("io", IO)
def test_one_key_over_the_rest(io):
    rng = np.random.default_rng(3)
    b = Batch(rng, [(160, 1300)], 1, 128, 32)
    for p in (0, 40, 700, 1255):
        b.ks[b.page_of(0, p), :, p % b.page // 16] += 3
    b.values()
    _run(rng, b, 7, io, sharp=3.0)
    _run(rng, b, 7, io, scale=0.0)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("at_", [0, 36, 37, 149])
def test_later_rows_do_not_reach_earlier_ones(io, at_):
    """K and V of one new row are NaN: the rows before it, and those whose window it has left, do not see it."""
    new, dim = 150, 64
    rng = np.random.default_rng(6)
    b = Batch(rng, [(new, new + 45)], 1, dim, 16)
    q = _rows(rng, b, 7, io)
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


@pytest.mark.parametrize("io", IO)
def test_non_finite_queries_stay_by_themselves(io):
    rng = np.random.default_rng(7)
    b = Batch(rng, [(147, 200)], 1, 128, 16)
    q = _rows(rng, b, 7, io)
    clean = q.copy()
    q[1, 2], q[40, 0, 7] = np.nan, np.inf
    qd = dev(q)
    out = torch.empty_like(qd)
    Attend(Cache(b), qd, out, io, 0.02)()
    got = out.cpu().numpy()
    assert not np.isfinite(got[1, 2]).any() and not np.isfinite(got[40, 0]).any()
    form = attend(b, clean, 0.02)
    tol = attend_tolerance(b, clean, form, 0.02, io, 200)
    got[1, 2], got[40, 0], form[0][1, 2], form[0][40, 0] = 0, 0, 0, 0
    assert (np.abs(got - form[0]) <= tol).all()


def test_captured_and_replayed():
    rng = np.random.default_rng(8)
    b = Batch(rng, [(150, 1200)], 1, 128, 64)
    q = [dev(_rows(rng, b, 7, "f16")) for _ in range(3)]
    qd, out = q[0].clone(), torch.empty_like(q[0])
    call = Attend(Cache(b), qd, out, "f16", 0.05)
    want = []
    for x in q:
        qd.copy_(x)
        call()
        want.append(out.clone())
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        call(torch.cuda.current_stream().cuda_stream)
    for x, y in list(zip(q, want)) * 2:
        qd.copy_(x)
        out.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, y)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("new,length,heads", [(3, 6000, 4), (12, 4000, 2), (60, 3000, 4), (150, 3000, 7)])
def test_non_finite_queries_over_splits(new, length, heads, io):
    """Rows of NaN and infinities stay by themselves where their parts are joined."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [(new, length)], 1, 64, 16)
    q = _rows(rng, b, heads, io)
    clean = q.copy()
    q[1, 1], q[2, 0, 7] = np.nan, np.inf
    qd = dev(q)
    out = torch.empty_like(qd)
    call = Attend(Cache(b), qd, out, io, 0.02)
    assert call.d.a.workspace_bytes > 0
    call()
    got = out.cpu().numpy().astype(np.float64)
    assert not np.isfinite(got[1, 1]).any() and not np.isfinite(got[2, 0]).any()
    form = attend(b, clean, 0.02)
    tol = attend_tolerance(b, clean, form, 0.02, io, length)
    got[1, 1], got[2, 0], form[0][1, 1], form[0][2, 0] = 0, 0, 0, 0
    assert (np.abs(got - form[0]) <= tol).all()


@pytest.mark.parametrize("io", IO)
def test_many_heads_to_one(io):
    """64 heads over one kv head: single tokens, drafts and a short prompt are one to some tiles each."""
    rng = np.random.default_rng(10)
    for lens in ([(1, 900), (0, 5), (1, 33)], [(3, 700), (5, 40)], [(20, 300), (17, 17)]):
        _run(rng, Batch(rng, lens, 1, 128, 16), 64, io)
        _run(rng, Batch(rng, lens, 1, 64, 32), 64, io, window=50, sink=3)


@pytest.mark.parametrize("io", IO)
@pytest.mark.parametrize("window,sink", [(0, 0), (200, 0), (200, 4)])
@pytest.mark.parametrize("new,heads", [(3, 4), (12, 2), (60, 4), (150, 7)])
def test_scores_far_below_zero(new, heads, window, sink, io):
    """Each score is some hundreds below 0: what a split without a key says of its maximum must not count."""
    rng = np.random.default_rng(11)
    b = Batch(rng, [(new, 3000)], 1, 64, 16, spread=0.0)
    b.kc |= 128
    b.values()
    q = np.abs(_rows(rng, b, heads, io))
    qd = dev(q)
    out = torch.empty_like(qd)
    Attend(Cache(b), qd, out, io, 10.0, window, sink=sink)()
    _compare(b, q, out.cpu().numpy(), io, 10.0, window, sink)
