"""mtg_sample_dev at temperatures that are small against the distance of neighbouring logits: steps of a flat row's histogram
in which no number of the logits' type lies, with a border or the choice in or beside them; against the 64-bit form."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")

from test_gpu_sample import run  # noqa: E402

NP = {"f32": np.float32, "f16": np.float16}
# temperature at which the numbers below 32 are 12.2 steps of T / 32 apart
APART = {"f32": 1e-5, "f16": 2.0 ** -6 * 32 / 12.2}


def _row(io, top, counts):
    """counts[i] ids at the i-th number from `top` down, scattered."""
    x = []
    at = NP[io](top)
    for n in counts:
        x += [at] * n
        at = np.nextafter(at, NP[io](-np.inf))
    x = np.array(x, np.float64)
    return x[np.random.default_rng(len(x)).permutation(len(x))]


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("counts", [(10, 8000, 8000, 8000, 8000), (3, 1, 5000, 20000), (2000, 2000, 2000, 30000), (1, 40000)], ids=str)
def test_steps_without_a_logit(counts, io):
    x = _row(io, 32.0, counts)
    cases = [(f * APART[io], p, m, k, u) for f in (1.0, 0.31, 2.7) for p, m, k in
             [(1.0, 0.5, 0), (1.0, 0.3, 0), (0.9, 0.5, 0), (0.3, 0.0, 0), (1.0, 0.97, 12000), (0.99, 0.01, 7000), (1.0, 0.0, 5000), (1.0, 1e-4, 0)]
             for u in (1e-4, 0.4, 0.999)]
    run(np.repeat(x[None], len(cases), 0), [c[:3] for c in cases], [c[3] for c in cases], [c[4] for c in cases], io)


@pytest.mark.parametrize("top", [1.0, 32.0, -7.25, 1e4])
def test_any_logits_at_small_temperatures(top):
    """Random counts at up to 60 neighbouring numbers, temperatures from a step far below their distance to one far above."""
    rng = np.random.default_rng(int(abs(top)))
    rows = 40
    gap = float(np.float32(top) - np.nextafter(np.float32(top), np.float32(-np.inf)))
    x = top - gap * np.minimum(rng.integers(0, 60, (rows, 20000)), rng.integers(0, 60, (rows, 1)))
    settings = [(gap * 32 * 2.0 ** rng.uniform(-5, 4), rng.choice([1.0, 0.9, 0.4]), rng.choice([0.0, 0.5, 0.1, 1e-3]), ) for _ in range(rows)]
    run(x, settings, rng.choice([0, 0, 3000, 9000], rows), rng.random(rows).astype(np.float32))
