"""mtg_rope_append_f8_dev with so many rows that a workgroup takes several heads one after the other, two to eight, the last one fewer,
queries, keys and values among them; against the 64-bit form."""
import pytest

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")

from test_gpu_rope_append_f8 import run  # noqa: E402

# sequences (rows, length), heads, kv heads: blocks x heads of 2,048 and more
SHAPES = [([(1100, 1109), (0, 3), (37, 300)], 23, 4), ([(1500, 1500)], 16, 8), ([(700, 1001), (16, 16), (801, 805)], 25, 6)]
LARGE = [([(4200, 4207)], 16, 8), ([(2100, 2105), (1, 17), (2111, 2111)], 25, 3)]


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads,kv_heads", SHAPES)
def test_several_heads_a_workgroup(lens, heads, kv_heads, dim, io):
    run(heads + dim, lens, heads, kv_heads, dim, 64, io, dim, norm=True)
    run(heads + dim, lens, heads, kv_heads, dim, 16, io, dim // 2 + 2, inter=True, positions=True, mscale=1.3, layout="both")


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads,kv_heads", LARGE)
def test_eight_heads_a_workgroup(lens, heads, kv_heads, dim, io):
    run(heads + dim, lens, heads, kv_heads, dim, 64, io, dim, norm=True, spread=6.0)
    run(heads + dim, lens, heads, kv_heads, dim, 32, io, 40, layout="head")


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_prompt_among_many_single_tokens(dim, io):
    """Few rows a sequence on average, for which a wave takes whole blocks, and one with many."""
    lens = [(1, 1 + 7 * i) for i in range(60)] + [(237, 300)] + [(1, 16), (0, 4), (2, 33)] * 14
    run(dim, lens, 6, 2, dim, 16, io, dim, norm=True)
