"""mtg_sample_dev on rows with few different logits, where a border or the choice lies among thousands of equal ones and
their ids decide, and at logits and settings that leave little to work with; against the 64-bit form."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
pytest.importorskip("torch")

from test_gpu_sample import FILTERS, run  # noqa: E402

MORE = FILTERS + [(float("inf"), 1.0, 0.0, 0), (float("inf"), 0.5, 0.5, 9000), (1e-30, 1.0, 0.0, 0), (1.0, 0.5, 0.01, 5000),
                  (0.5, 0.999999, 0.0, 0), (1.0, 1.0, 0.0, 4097)]


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("levels", [1, 2, 7, 100])
@pytest.mark.parametrize("vocab", [1000, 5000, 40001, 300000])
def test_few_different_logits(vocab, levels, io):
    rng = np.random.default_rng(vocab + levels)
    rows = 2 * len(MORE)
    x = np.linspace(-3, 4, levels)[rng.integers(0, levels, (rows, vocab))]
    f = MORE * 2
    run(x, [c[:3] for c in f], [c[3] for c in f], rng.random(rows).astype(np.float32), io)


@pytest.mark.parametrize("share", [0.5, 0.001, 0.0])
def test_large_finite_and_infinite_logits(share):
    """Logits at both ends of their type, with infinities among them or without."""
    rng = np.random.default_rng(3)
    f = MORE
    for io, most in (("f32", 3.4e38), ("f16", 65504.0)):
        for vocab in (900, 20000):
            x = rng.choice([most, -most, 0.5 * most, 0.0, -1e-7, 1e-7, 1.0], (len(f), vocab))
            x[rng.random(x.shape) < share] = np.inf
            x[rng.random(x.shape) < 0.1] = -np.inf
            x[rng.random(x.shape) < 0.1] = np.nan
            run(x, [c[:3] for c in f], [c[3] for c in f], rng.random(len(f)).astype(np.float32), io)


def test_ends_of_the_random_number_among_equal_logits():
    rng = np.random.default_rng(4)
    u = [0.0, 1e-38, 1e-7, 0.5, 1 - 2.0 ** -24, 1.0, 2.0, float("nan")]
    for vocab in (1024, 1025, 4096, 4097, 100000):
        x = np.zeros((len(u), vocab))
        run(x, [(1.0, 1.0, 0.0)] * len(u), None, u)
        run(x, [(1.0, 1.0, 0.0)] * len(u), [4099] * len(u), u)
        x[:, rng.integers(0, vocab, vocab // 2)] = -1.0
        run(x, [(1.0, 1.0, 0.0)] * len(u), None, u)
        run(x, [(1.0, 0.25, 0.0)] * len(u), None, u)
