"""mtg_paged_attn_f8_dev on the GPU by each kernel with each way to join its splits (paged_f8_routes.py), against the 64-bit
form with test_gpu_paged_attn_f8.py's comparison."""
import numpy as np
import pytest

import paged_f8_routes
import paged_routes
from serve_ref_f8 import Batch

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")

from test_gpu_paged_attn_f8 import IO, _run  # noqa: E402


# each case with both types and both sizes of heads, in two of their four pairs
PAIRS = [(c, *p) for i, c in enumerate(paged_f8_routes.CASES) for p in ((64, IO[i % 2]), (128, IO[1 - i % 2]))]


@pytest.mark.parametrize("case,dim,io", PAIRS, ids=lambda c: c[0].replace(" ", "_") if isinstance(c, tuple) else None)
def test_routes(case, dim, io):
    _, heads, kv_heads, lens, window, sink, max_kv, route = case
    rng = np.random.default_rng(dim + heads)
    b = Batch(rng, lens, kv_heads, dim, paged_f8_routes.PAGE)
    assert b.table.shape[1] == paged_routes.table_stride(lens)
    a = _run(rng, b, heads, io, window=window, max_kv=max_kv or max(n for _, n in lens), sink=sink)
    assert (a.d.a.workspace_bytes > 0) == ("alone" not in route)
