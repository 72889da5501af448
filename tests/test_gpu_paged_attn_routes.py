"""mtg_paged_attn_dev on the GPU by each kernel with each way to join its splits (paged_routes.py), against the 64-bit
form with test_gpu_paged_attn.py's comparison; then captured and replayed with other lengths over the same workspace."""
import numpy as np
import pytest

import paged_routes
from serve_ref import Batch

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import Attend, Cache, dev  # noqa: E402
from test_gpu_paged_attn import TYPE_PAIRS, _compare, _rows, _run  # noqa: E402


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", paged_routes.CASES, ids=lambda c: c[0].replace(" ", "_"))
def test_routes(case, dim, io, kv):
    _, heads, kv_heads, lens, window, max_kv, _ = case
    rng = np.random.default_rng(dim + heads)
    b = Batch(rng, lens, kv_heads, dim, paged_routes.PAGE, kv)
    assert b.table.shape[1] == paged_routes.table_stride(lens)
    a = _run(rng, b, heads, io, window=window, max_kv=max_kv or max(n for _, n in lens))
    assert (a.d.workspace_bytes > 0) == ("alone" not in paged_routes.route(case, kv))


@pytest.mark.parametrize("name", ["long contexts", "drafts, a dozen splits", "a chunk, long context", "several tokens, a dozen splits"])
def test_second_launches_replayed(name):
    """A captured call whose join is a launch of its own: shorter lengths, a sequence that runs empty, other rows."""
    case = next(c for c in paged_routes.CASES if c[0] == name)
    _, heads, kv_heads, lens, window, _, _ = case
    rng = np.random.default_rng(7)
    b = Batch(rng, lens, kv_heads, 64, paged_routes.PAGE, "f16")
    cache = Cache(b)
    q = dev(_rows(rng, b, heads, "f16"))
    out, eager_out = torch.empty_like(q), torch.empty_like(q)
    most = max(n for _, n in lens)
    call = Attend(cache, q, out, "f16", 0.125, window, most)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call(side.cuda_stream)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(side.cuda_stream)
    for step in range(4):
        b.kv_len = np.array([max(n, length // (step + 1)) for n, length in lens], np.int32)
        if step == 3:
            b.kv_len[0] = 0
        cache.kv_len.copy_(torch.from_numpy(b.kv_len))
        host = _rows(rng, b, heads, "f16")
        q.copy_(torch.from_numpy(host))
        out.fill_(55.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager = Attend(cache, q, eager_out, "f16", 0.125, window, most)
        eager()
        torch.cuda.synchronize()
        assert torch.equal(eager_out, out)
        _compare(b, host, out.cpu().numpy(), "f16", 0.125, window)
