"""mtg_paged_attn_f8_dev on the GPU where blocks that no row sees hold scales of 255 and codes NaN: those between the first
positions and the window, up to its edges, as pages that left a window do. Against the 64-bit form, whose tolerance takes
the blocks that rows see alone, and against the same call without these blocks' pages."""
import numpy as np
import pytest

from serve_ref_f8 import Batch, attend, attend_tolerance_seen, seen_blocks

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import dev  # noqa: E402
from serve_dev_f8 import Attend, Cache  # noqa: E402
from test_gpu_paged_attn_f8 import _rows  # noqa: E402

# heads, kv heads, sequences (new rows, length), window
ROUTES = {
    "rows16": (4, 2, [(1, 400), (1, 389), (1, 371), (1, 130), (1, 64)], 100),
    "rows16_edges": (4, 2, [(2, 300 + i) for i in range(0, 36, 3)], 80),
    "rows16_splits": (4, 2, [(1, 5000), (1, 4011), (1, 700)], 2010),
    "rows32": (4, 2, [(10, 400), (12, 389), (11, 420)], 100),
    "rows32_splits": (4, 2, [(10, 5000), (12, 2500)], 1700),
    "eight": (16, 8, [(1, 700 - 13 * i) for i in range(17)], 300),
    "chunk": (4, 2, [(180, 600), (70, 389)], 100),
    "chunk_splits": (4, 2, [(150, 4100), (60, 2000)], 2049),
    "wide": (7, 1, [(150, 1900), (147, 700)], 300),
    "wide_splits": (16, 1, [(70, 5000), (64, 800)], 2500),
}


def _spoil(b, window, sink):
    """Scales of 255 and codes NaN where no row sees them. Returns the pages (of one block each) that hold nothing else."""
    n = 0
    pages = np.zeros(b.n_pages, bool)
    for s in range(len(b.lens)):
        for (page, block), seen in seen_blocks(b, s, window, sink):
            if seen:
                continue
            b.ks[page, :, block] = b.vs[page, :, block] = 255
            where = slice(16 * block, 16 * block + 16)
            b.kc[page, :, where], b.vc[page, :, where] = 127, 255
            pages[page] = b.page == 16
            n += 1
    assert n > 0
    b.values()
    return pages


def _call(b, q, io, scale, window, sink, splits):
    qd = dev(q)
    out = torch.full_like(qd, 55.0)
    Attend(Cache(b), qd, out, io, scale, window, int(b.kv_len.max()) if splits else 1, sink)()
    torch.cuda.synchronize()
    return out.cpu().numpy()


@pytest.mark.parametrize("dim,page,io", [(64, 16, "f32"), (128, 16, "f16"), (128, 64, "f32")])
@pytest.mark.parametrize("sink", [0, 20])
@pytest.mark.parametrize("route", ROUTES)
def test_blocks_that_no_row_sees(route, sink, dim, page, io):
    heads, kv_heads, lens, window = ROUTES[route]
    rng = np.random.default_rng(dim + sink)
    b = Batch(rng, lens, kv_heads, dim, page)
    rms = float(np.sqrt((b.k[~np.isnan(b.k)] ** 2).mean()))
    scale, q = dim ** -0.5 / max(1.0, rms), _rows(rng, b, heads, io)
    pages, splits = _spoil(b, window, sink), "splits" in route or route == "eight"
    got = _call(b, q, io, scale, window, sink, splits)
    form = attend(b, q, scale, window, sink)
    tol = attend_tolerance_seen(b, q, form, scale, io, int(b.kv_len.max()), window, sink)
    off = np.abs(got.astype(np.float64) - form[0])
    assert (off <= tol).all(), float((off / tol).max())
    if page == 16:
        b.table[np.isin(b.table, np.flatnonzero(pages))] = -1
        assert np.array_equal(_call(b, q, io, scale, window, sink, splits), got)
