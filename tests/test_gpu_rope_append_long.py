"""mtg_rope_append_dev for the rows of long prompts (1,024 rows or more: a thread then takes two heads, where a row has
more heads than one pass of the workgroup holds), with the 64-bit form and tolerances of test_gpu_rope_append.py."""
import ctypes

import numpy as np
import pytest

import mtg
from serve_ref import Batch

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import check  # noqa: E402
from test_gpu_rope_append import TYPE_PAIRS, Call  # noqa: E402

LONG = [(700, 800), (0, 5), (300, 310), (31, 31)]
# heads, kv heads, head_dim: 256 threads hold 16 heads of 128 or 32 of 64 at a time
HEADS = [(16, 8, 128),   # two passes, both full
         (17, 3, 128),   # two, the second one partly empty
         (24, 8, 128),   # three: the last pair of passes has one
         (40, 5, 128),   # four, two workgroups a row
         (36, 6, 64), (79, 4, 64)]


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("rot,inter", [(0, False), (0, True), (34, False), (34, True), (48, False)])
def test_long_prompts(io, kv, heads, kv_heads, dim, rot, inter):
    """rot 0 here: the whole head. Rows before the first sequence and behind the last stay as they were."""
    rng = np.random.default_rng(heads + rot)
    b = Batch(rng, LONG, kv_heads, dim, 64, kv, lead=2, tail=3, filled=False)
    c = Call(rng, b, io, heads, rot or dim, inter, norm=rot != 34, mscale=1.25 if rot == 48 else 1.0)
    c.run()
    c.verify()


@pytest.mark.parametrize("io,kv", TYPE_PAIRS)
def test_long_prompts_in_place_and_parts_alone(io, kv):
    rng = np.random.default_rng(3)
    make = lambda: Call(rng, Batch(rng, LONG, 5, 128, 64, kv, tail=1, filled=False), io, 40, 128, False, norm=True)  # noqa: E731
    c = make()
    c.d.q_out, c.d.q_out_stride = c.d.q, c.d.q_stride
    c.run()
    c.verify(q_out=c.xd[:, :40])
    assert np.array_equal(c.xd[:, 40:].cpu().numpy(), c.x[:, 40:]) and np.array_equal(c.xd[-1].cpu().numpy(), c.x[-1])
    c = make()
    c.d.k_new = c.d.v_new = None
    c.run()
    c.verify(with_kv=False)
    c = make()
    c.d.q = c.d.q_out = None
    c.run()
    c.verify(with_q=False)
    assert (c.out == 77.0).all()


def test_a_long_prompt_captured_and_replayed():
    rng = np.random.default_rng(4)
    c = Call(rng, Batch(rng, [(1200, 1300)], 8, 128, 64, "f16", filled=False), "f16", 16, 128, False, norm=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c.run(side.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        check(mtg.lib().mtg_rope_append_dev(ctypes.byref(c.d), side.cuda_stream))
    for step in range(3):
        c.x = rng.standard_normal(c.x.shape).astype(np.float16)
        c.xd.copy_(torch.from_numpy(c.x))
        c.b.kv_len = np.array([1300 - 40 * step], np.int32)
        c.cache.kv_len.copy_(torch.from_numpy(c.b.kv_len))
        for t in (c.cache.k, c.cache.v):
            t.fill_(float("nan"))
        c.b.k[:], c.b.v[:] = np.nan, np.nan
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        c.verify()
