"""mtg_sample_dev on the GPU against the 64-bit form (sample_ref): each way to an answer, every filter at its ends."""
import ctypes

import numpy as np
import pytest
import torch

import mtg
from sample_ref import answers
from serve_dev import MTG, TORCH, at, check, dev, stream

pytestmark = pytest.mark.gpu
NP = {"f32": np.float32, "f16": np.float16}


class Call:
    def __init__(self, x, settings, top_k, uniform, io, stride=None, prob=True):
        rows, self.vocab = x.shape
        stride = stride or self.vocab
        self.x = torch.full((rows * stride + 8,), float("nan"), dtype=TORCH[io], device="cuda")
        self.at = 1  # an odd start
        self.view = self.x[1:1 + rows * stride].view(rows, stride)[:, :self.vocab]
        self.view.copy_(dev(x.astype(NP[io])))
        self.settings, self.uniform = dev(np.asarray(settings, np.float32)), dev(np.asarray(uniform, np.float32))
        self.top_k = None if top_k is None else dev(np.asarray(top_k, np.int32))
        self.choice = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
        self.prob = torch.full((rows,), -7.0, device="cuda") if prob else None
        self.d = mtg.Sample(logits=at(self.view), stride=stride, settings=at(self.settings), top_k=at(self.top_k), uniform=at(self.uniform),
                            choice=at(self.choice), prob=at(self.prob), io_type=MTG[io], rows=rows, vocab=self.vocab)
        size = mtg.lib().mtg_sample_workspace(ctypes.byref(self.d))
        self.work = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        self.d.workspace, self.d.workspace_bytes = at(self.work), size

    def __call__(self, s=None):
        check(mtg.lib().mtg_sample_dev(ctypes.byref(self.d), stream() if s is None else s))


def compare(x, settings, top_k, uniform, io, choice, prob):
    x = x.astype(NP[io])
    for r in range(len(x)):
        want = answers(x[r], *settings[r], 0 if top_k is None else int(top_k[r]), uniform[r])
        got = int(choice[r])
        assert got in want, (r, got, sorted(want.items())[:4], settings[r], None if top_k is None else top_k[r], uniform[r])
        if prob is not None:  # weights to 2^-27, their sum likewise, and the rounding of the result
            assert any(abs(prob[r] - w) <= w * 2.0 ** -23 for w in want[got]), (r, prob[r], want[got])


def run(x, settings, top_k, uniform, io="f32", **kw):
    settings = [tuple(np.float32(v) for v in s) for s in settings]
    call = Call(x, settings, top_k, uniform, io, **kw)
    call()
    torch.cuda.synchronize()
    choice, prob = call.choice.cpu().numpy(), None if call.prob is None else call.prob.cpu().numpy().astype(np.float64)
    compare(x, settings, top_k, uniform, io, choice, prob)
    call()
    torch.cuda.synchronize()
    assert np.array_equal(call.choice.cpu().numpy(), choice)  # the same call, the same bits
    if prob is not None:
        assert np.array_equal(call.prob.cpu().numpy(), prob.astype(np.float32))
    return call


def logits(rng, rows, vocab, spread=2.0, peaks=20):
    x = spread * rng.standard_normal((rows, vocab))
    for r in range(rows):
        x[r, rng.integers(0, vocab, peaks)] += 12 * rng.random(peaks)
    return x


FILTERS = [  # temperature, top_p, min_p, top_k
    (1.0, 1.0, 0.0, 0), (0.7, 1.0, 0.0, 40), (1.0, 0.9, 0.0, 0), (1.0, 1.0, 0.05, 0), (0.8, 0.95, 0.01, 100), (1.3, 0.6, 0.0, 7),
    (2.5, 0.99, 0.0, 0), (2.0, 1.0, 1e-6, 0), (5.0, 0.7, 0.001, 0), (1.0, 0.999, 0.0, 3000), (0.05, 0.9, 0.1, 50), (1.0, 0.5, 0.5, 2)]


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 64, 255, 256, 257, 1000, 4096, 4097, 9001, 50257, 151936])
def test_filters(vocab, io):
    rng = np.random.default_rng(vocab)
    rows = 4 * len(FILTERS)
    x = logits(rng, rows, vocab)
    f = [FILTERS[r % len(FILTERS)] for r in range(rows)]
    run(x, [c[:3] for c in f], [c[3] for c in f], rng.random(rows).astype(np.float32), io)


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.1, 0.6, 8.0])
def test_flat_and_steep_rows(spread, io):
    """From all logits equal, where no part of the row decides by itself, to rows of a few likely ids."""
    rng = np.random.default_rng(int(spread * 1000))
    for vocab in (700, 6000, 70000):
        rows = len(FILTERS)
        run(logits(rng, rows, vocab, spread, peaks=3 if spread else 0), [c[:3] for c in FILTERS], [c[3] for c in FILTERS],
            rng.random(rows).astype(np.float32), io)


def test_ends_of_the_random_number():
    rng = np.random.default_rng(1)
    u = np.array([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, np.nan, 1e-30, 0.5, np.inf, -np.inf], np.float32)
    for vocab in (10, 5000, 60000):
        for f in FILTERS[:6]:
            run(logits(rng, len(u), vocab, 1.0), [f[:3]] * len(u), [f[3]] * len(u), u)


def test_ends_of_the_settings():
    """Filters that keep one id, all ids, or say nothing; temperatures that are none."""
    rng = np.random.default_rng(2)
    nan, inf = float("nan"), float("inf")
    cases = [(t, p, m, k) for t in (0.0, -1.0, nan, 1.0, 1e-30, 1e-42, 1e30, inf) for p, m, k in
             [(1.0, 0.0, 0), (0.0, 0.0, 0), (-1.0, 0.0, 0), (nan, nan, -3), (2.0, -1.0, 2 ** 31 - 1), (1.0, 1.0, 0), (1.0, 1.5, 0), (0.5, 0.3, 9),
              (1e-20, 0.0, 0), (1.0 - 2.0 ** -24, 0.0, 0), (1.0, 1e-40, 0), (1.0, 0.0, 1), (0.9, 0.0, 1)]]
    for vocab in (40, 30000):
        x = logits(rng, len(cases), vocab)
        x[::3, 5] = x[::3, 17] = 40.0  # two largest ones
        run(x, [c[:3] for c in cases], [c[3] for c in cases], rng.random(len(cases)).astype(np.float32))


@pytest.mark.parametrize("io", ["f32", "f16"])
def test_ids_that_take_no_part(io):
    """Masked rows: few ids left, one, none; NaN among them; infinities."""
    rng = np.random.default_rng(3)
    for vocab in (300, 5000, 151643):
        x = logits(rng, 24, vocab)
        x[0:12] = -np.inf
        x[1, vocab // 2] = -3.0
        x[2, [1, vocab - 1]] = [1.0, 1.5]
        x[3, ::97] = rng.standard_normal(len(x[3, ::97]))
        x[4] = np.nan
        x[5, 3::5] = np.nan
        x[5, 1::5] = 0.5
        x[6, [7, 9, 200]] = np.inf
        x[6, ::11] = 2.0
        x[7, 100] = np.inf
        x[8, :50] = -60000.0
        x[12, ::2] = np.nan
        x[13, 1::3] = -np.inf
        x[14, [3, 250]] = np.inf
        x[15, 8] = np.inf
        for f in FILTERS:
            run(x, [f[:3]] * 24, [f[3]] * 24, rng.random(24).astype(np.float32), io)


@pytest.mark.parametrize("k", [1, 2, 255, 256, 257, 1023, 1024, 1025, 4000, 4096, 4097, 20000, 49999, 50000, 50001])
def test_top_k_alone(k):
    rng = np.random.default_rng(k)
    for io in ("f32", "f16"):
        for spread in (2.0, 0.01):
            x = logits(rng, 6, 50000, spread)
            run(x, [(1.0, 1.0, 0.0)] * 6, [k] * 6, [0.0, 0.3, 0.9, 0.999, 0.9999999, 0.5], io)


def test_large_vocabularies_and_many_rows():
    rng = np.random.default_rng(4)
    for vocab in (262144, 262145, 400001, 1 << 20):
        x = logits(rng, len(FILTERS), vocab).astype(np.float32)
        run(x, [c[:3] for c in FILTERS], [c[3] for c in FILTERS], rng.random(len(FILTERS)).astype(np.float32))
    f = [FILTERS[r % len(FILTERS)] for r in range(600)]
    run(logits(rng, 600, 9000), [c[:3] for c in f], [c[3] for c in f], rng.random(600).astype(np.float32), "f16")


def test_the_largest_vocabulary():
    rng = np.random.default_rng(5)
    x = (2 * rng.standard_normal((2, 1 << 24))).astype(np.float32)
    run(x, [(1.0, 0.9, 0.0), (0.2, 1.0, 0.01)], [0, 100], [0.7, 0.3])


def test_strides_and_what_is_left_out():
    rng = np.random.default_rng(6)
    x = logits(rng, 5, 4999)
    s, u = [(0.9, 0.9, 0.01)] * 5, rng.random(5).astype(np.float32)
    for io in ("f32", "f16"):
        call = run(x, s, [30] * 5, u, io, stride=5011)
        other = run(x, s, [30] * 5, u, io, prob=False)
        assert torch.equal(call.choice, other.choice)
        run(x, s, None, u, io)


def test_how_often_each_id_comes():
    """Random numbers on a grid: each id's share of them is its probability, to the grid's step."""
    rng = np.random.default_rng(7)
    n = 512
    row = logits(rng, 1, 5000, 1.0)
    u = (np.arange(n) + 0.5) / n
    call = run(np.repeat(row, n, 0), [(1.0, 0.8, 0.0)] * n, [25] * n, u.astype(np.float32))
    ids, counts = np.unique(call.choice.cpu().numpy(), return_counts=True)
    prob = {int(i): float(p) for i, p in zip(call.choice.cpu(), call.prob.cpu())}
    for i, c in zip(ids, counts):
        assert abs(c / n - prob[int(i)]) <= 1.0 / n + 1e-6


def test_workspaces_of_any_content_streams_and_graphs():
    """Two captured calls on two streams, replayed with new logits and eager calls between them."""
    rng = np.random.default_rng(8)
    rows, vocab = 5, 60000
    sides = []
    for i in range(2):
        f = [FILTERS[(3 * i + r) % len(FILTERS)] for r in range(rows)]
        call = Call(logits(rng, rows, vocab), [c[:3] for c in f], [c[3] for c in f], rng.random(rows), "f32")
        for fill in (0, 1, 255):
            call.work.fill_(fill)
            call()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        call(s.cuda_stream)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(s.cuda_stream)
        sides.append((call, f, s, g))
    for step in range(4):
        hosts = []
        for call, *_ in sides:
            hosts.append(logits(rng, rows, vocab, [2.0, 0.1, 1.0, 4.0][step]).astype(np.float32))
            call.view.copy_(dev(hosts[-1]))
            call.choice.fill_(-9)
            call.uniform.copy_(torch.rand(rows))
        torch.cuda.synchronize()
        for _, _, s, g in sides:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (call, f, _, _), host in zip(sides, hosts):
            got, prob = call.choice.cpu().numpy(), call.prob.cpu().numpy()
            compare(host, [tuple(np.float32(v) for v in c[:3]) for c in f], [c[3] for c in f], call.uniform.cpu().numpy(), "f32", got, prob.astype(np.float64))
            call.choice.fill_(-9)
            call()
            torch.cuda.synchronize()
            assert np.array_equal(call.choice.cpu().numpy(), got) and np.array_equal(call.prob.cpu().numpy(), prob)
