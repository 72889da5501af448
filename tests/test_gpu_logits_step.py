"""mtg_logits_step_dev on the GPU against the 64-bit form (serve_ref.logits_row): penalties, biases, masks,
choices with ties, NaN and nothing allowed, odd vocabularies and strides, both types."""
import ctypes

import numpy as np
import pytest

import mtg
from serve_ref import HALF, TINY, TYPES, first_max, logits_row

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import MTG, at, check, dev, stream  # noqa: E402


class Step:
    """A call over host arrays: x [rows][vocab], hist / bias lists per row, mask [rows][vocab] bool or None."""

    def __init__(self, x, io, hist=None, penalties=None, bias=None, mask=None, pad=0, out_pad=0, in_place=False, want_out=True,
                 want_choice=True):
        rows, vocab = x.shape
        self.x, self.io, self.hist, self.pen, self.bias, self.mask = x.astype(TYPES[io]), io, hist, penalties, bias, mask
        wide = np.full((rows, vocab + pad), 9.0, TYPES[io])
        wide[:, :vocab] = self.x
        self.xd = dev(wide)
        self.out = self.xd if in_place else torch.full((rows, vocab + out_pad), 9.0, dtype=self.xd.dtype, device="cuda")
        self.choice = torch.full((rows,), -77, dtype=torch.int32, device="cuda")
        d = mtg.LogitsStep(logits=at(self.xd), out=at(self.out) if want_out else None, stride=vocab + pad,
                           out_stride=self.out.stride(0), choice=at(self.choice) if want_choice else None, io_type=MTG[io],
                           rows=rows, vocab=vocab)
        self.keep = []
        if hist is not None:
            d.history, d.hist_range, d.n_history = self._lists(hist)
            self.keep.append(dev(np.array(penalties, np.float32)))
            d.penalties = at(self.keep[-1])
        if bias is not None:
            d.bias_ids, d.bias_range, d.n_bias = self._lists([[i for i, _ in b] for b in bias])
            self.keep.append(dev(np.array([v for b in bias for _, v in b] + [0.0], np.float32)))
            d.bias = at(self.keep[-1])
        if mask is not None:
            words = np.packbits(mask, axis=1, bitorder="little")
            words = np.pad(words, ((0, 0), (0, -words.shape[1] % 4))).view(np.uint32)
            self.keep.append(dev(words.view(np.int32)))
            d.mask, d.mask_stride = at(self.keep[-1]), 0 if len(words) == 1 and rows > 1 else words.shape[1]
        size = mtg.lib().mtg_logits_step_workspace(ctypes.byref(d))
        if size:
            self.work = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
            d.workspace, d.workspace_bytes = at(self.work), size
        self.d = d

    def _lists(self, lists):
        flat = np.array([i for one in lists for i in one] + [0], np.int32)
        ends = np.cumsum([0] + [len(one) for one in lists])
        self.keep += [dev(flat), dev(np.stack([ends[:-1], ends[1:]], 1).astype(np.int32))]
        return at(self.keep[-2]), at(self.keep[-1]), len(flat) - 1

    def run(self, s=None):
        check(mtg.lib().mtg_logits_step_dev(ctypes.byref(self.d), stream() if s is None else s))
        torch.cuda.synchronize()
        return self

    def verify(self):
        rows, vocab = self.x.shape
        whole = self.out.cpu().numpy()
        got, choice = whole[:, :vocab], self.choice.cpu().numpy()
        assert (whole[:, vocab:] == 9.0).all()
        for r in range(rows):
            allowed = None if self.mask is None else self.mask[r if len(self.mask) > 1 else 0]
            y, size = logits_row(self.x[r], self.hist[r] if self.hist is not None else (),
                                 self.pen[r] if self.hist is not None else (1, 0, 0), self.bias[r] if self.bias is not None else (), allowed)
            if self.d.out:
                # five operations of 32 bits at most, each off by half a step of at most `size`, then the output's rounding
                fine = np.isfinite(y)
                assert np.array_equal(np.isnan(got[r]), np.isnan(y))
                odd = ~fine & ~np.isnan(y)
                assert np.array_equal(got[r][odd], y[odd].astype(TYPES[self.io]))
                with np.errstate(over="ignore"):
                    near = y[fine].astype(TYPES[self.io]).astype(np.float64)
                over = np.isinf(near)  # beyond the type's range
                off = np.abs(got[r][fine].astype(np.float64) - y[fine])
                tol = 5 * size[fine] * 2.0 ** -24 + np.abs(y[fine]) * HALF[self.io] * 1.01 + TINY[self.io]
                assert (off[~over] <= tol[~over]).all(), (r, (off / tol)[~over].max())
                assert np.isinf(got[r][fine][over]).all()
                if self.d.choice:
                    assert choice[r] == first_max(got[r], allowed), r
            elif self.d.choice:
                i, best = int(choice[r]), first_max(y, allowed)
                tol = 5 * size[best] * 2.0 ** -24 + np.abs(y[best]) * HALF[self.io] * 1.01
                assert abs(y[i] - y[best]) <= 2 * tol, (r, i, best)


def _lists(rng, rows, vocab, most):
    return [list(rng.integers(-3, vocab + 3, rng.integers(0, most + 1))) + [5, 5, 5] for _ in range(rows)]


def _biases(rng, rows, vocab, most):
    return [[(int(i), float(rng.normal() * 4)) for i in rng.integers(-2, vocab + 2, rng.integers(0, most + 1))] for _ in range(rows)]


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 4095, 4096, 4097, 20011, 151936])
def test_against_64_bits(io, vocab):
    rng = np.random.default_rng(vocab)
    rows = 5 if vocab > 5000 else 9
    x = 4 * rng.standard_normal((rows, vocab))
    pen = np.stack([rng.choice([1.0, 1.3, 0.5, 2.0], rows), rng.choice([0.0, 0.3, -0.2], rows), rng.choice([0.0, 0.5], rows)], 1)
    mask = rng.random((rows, vocab)) < 0.4
    mask[0] = False
    Step(x, io, _lists(rng, rows, vocab, 400), pen, _biases(rng, rows, vocab, 60), mask).run().verify()
    Step(x, io, _lists(rng, rows, vocab, 30), pen).run().verify()
    Step(x, io, bias=_biases(rng, rows, vocab, 10)).run().verify()
    Step(x, io, mask=mask[1:2]).run().verify()      # one row of words for all
    Step(x, io).run().verify()
    Step(x, io, _lists(rng, rows, vocab, 400), pen, want_out=False).run().verify()
    s = Step(x, io, _lists(rng, rows, vocab, 40), pen, want_choice=False).run()
    s.verify()
    assert (s.choice == -77).all()


@pytest.mark.parametrize("io", ["f32", "f16"])
def test_strides_alignment_and_in_place(io):
    """Rows that begin at any element: odd vocabularies and strides, out with another stride, out over logits."""
    rng = np.random.default_rng(2)
    for vocab, pad, out_pad in ((4999, 0, 0), (4999, 3, 0), (4099, 1, 6), (130, 5, 1)):
        x = 3 * rng.standard_normal((6, vocab))
        a = (x, io, _lists(rng, 6, vocab, 50), [(1.2, 0.1, 0.1)] * 6, _biases(rng, 6, vocab, 9), rng.random((6, vocab)) < 0.5)
        Step(*a, pad=pad, out_pad=out_pad).run().verify()
        Step(*a, pad=pad, in_place=True).run().verify()


@pytest.mark.parametrize("io", ["f32", "f16"])
def test_choices(io):
    """Ties go to the lowest id, across workgroups too; zeros of both signs tie; NaN is never chosen; nothing allowed
    gives -1; allowed minus infinity counts; what is equal after rounding ties."""
    vocab = 9000
    x = np.full((9, vocab), -5.0)
    x[0, [4500, 8999, 70]] = 2.0
    x[1, :] = 1.0
    x[2, [30]], x[2, [8000]] = -0.0, 0.0
    x[3, :] = np.nan
    x[3, 6000] = -np.inf
    x[4, :] = np.nan
    x[5, :] = -np.inf
    x[6, [4096, 100]] = np.inf
    x[7, [10, 8191]] = [1.0, 1.0 + 2.0 ** -12]   # f16: equal
    x[8, 3] = np.nan
    s = Step(x, io).run()
    s.verify()
    assert s.choice.tolist() == [70, 0, 30, 6000, -1, 0, 100, 10 if io == "f16" else 8191, 0]
    mask = np.ones((9, vocab), bool)
    mask[0, 70] = mask[1, :8998] = mask[3, 6000] = mask[6, 100] = False
    mask[2], mask[5, :17] = False, False
    s = Step(x, io, mask=mask).run()
    s.verify()
    assert s.choice.tolist() == [4500, 8998, -1, -1, -1, 17, 4096, 10 if io == "f16" else 8191, 0]
    assert (s.out[2] == -np.inf).all()


def test_non_finite_logits_and_lowest_values():
    rng = np.random.default_rng(4)
    for io in ("f32", "f16"):
        low = float(np.finfo(TYPES[io]).min)
        x = rng.standard_normal((4, 5000))
        x[0, ::3], x[1, ::5], x[2, ::2], x[3] = np.nan, np.inf, -np.inf, low
        hist = [list(range(0, 5000, 7))] * 4
        mask = rng.random((4, 5000)) < 0.5
        with np.errstate(over="ignore", invalid="ignore"):
            Step(x, io, hist, [(1.5, 0.25, 0.5)] * 4, [[(3, 1.0), (5, -2.0)]] * 4, mask).run().verify()


def test_repetition_alone_is_the_greedy_choice():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((12, 30011)).astype(np.float32)
    hist = [list(rng.integers(0, 30011, 100)) + list(np.argsort(-x[r])[:3]) for r in range(12)]
    hist = [h[-100:] for h in hist]
    s = Step(x, "f32", hist, [(1.1, 0, 0)] * 12, want_out=False).run()
    assert s.choice.tolist() == [mtg.greedy_choice(x[r], hist[r], 1.1) for r in range(12)]


def test_shared_and_cut_ranges():
    """Rows over one history that grows by one (verify rows); ranges outside the list are cut to it."""
    rng = np.random.default_rng(6)
    vocab, rows = 6000, 8
    x = rng.standard_normal((rows, vocab))
    ids = [int(i) for i in rng.integers(0, vocab, 40)]
    s = Step(x, "f32", [ids[:32 + r] for r in range(rows)], [(1.4, 0.2, 0.1)] * rows)
    flat = dev(np.array(ids, np.int32))
    ranges = dev(np.array([[0, 32 + r] for r in range(rows)], np.int32))
    s.d.history, s.d.hist_range, s.d.n_history = at(flat), at(ranges), 40
    s.run().verify()
    s.hist = [ids, ids[10:], [], [], ids[:5], [], ids, ids[39:]]
    ranges.copy_(torch.tensor([[-5, 2 ** 31 - 1], [10, 41], [7, 3], [40, 50], [-2 ** 31, 5], [2 ** 31 - 1, 2 ** 31 - 1], [0, 40], [39, 40]]))
    s.run().verify()


def test_a_long_history_and_a_listed_id_twice():
    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 5000))
    hist = [[17] * 70000 + [4999], list(rng.integers(0, 5000, 30000))]
    bias = [[(8, 1.0), (9, 2.0), (8, -3.0), (8, 5.0), (9, 7.0)], [(i % 50, float(i)) for i in range(3000)]]
    Step(x, "f32", hist, [(1.0, 0.001, 0.0)] * 2, bias).run().verify()


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("rows,vocab", [(3, 9001), (1040, 4096), (210, 20011)])
def test_lists_of_any_length_in_small_and_large_grids(io, rows, vocab):
    """Long lists (70,000 ids, some in each part of a workgroup's ids) beside short ones, few rows and many."""
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, vocab))
    hist, bias = _lists(rng, rows, vocab, 20), _biases(rng, rows, vocab, 5)
    hist[1] = [int(i) for i in rng.integers(0, vocab, 70000)]
    bias[rows - 1] = [(int(i), float(v)) for i, v in zip(rng.integers(0, vocab, 66000), rng.standard_normal(66000))]
    mask = rng.random((rows, vocab)) < 0.9
    Step(x, io, hist, [(1.2, 0.01, 0.1)] * rows, bias, mask).run().verify()
    Step(x, io, hist, [(1.2, 0.01, 0.1)] * rows).run().verify()
    Step(x, io, bias=bias).run().verify()


def test_a_workspace_of_any_content():
    """What lies in a fresh workspace, or another call's leavings, does not matter; again and again."""
    rng = np.random.default_rng(9)
    a, b = (Step(rng.standard_normal((rows, vocab)), "f32") for rows, vocab in ((4, 30000), (7, 9000)))
    assert a.d.workspace_bytes >= b.d.workspace_bytes
    b.d.workspace = a.d.workspace
    for fill in (0, 1, 127, 255):
        a.work.fill_(fill)
        for s in (a, b, a, a):
            s.choice.fill_(-1)
            s.run().verify()


def test_a_captured_call():
    """Captured on another stream, replayed with new logits and lists, eager calls between."""
    rng = np.random.default_rng(8)
    vocab, rows = 20000, 3
    hist = [list(rng.integers(0, vocab, 64)) for _ in range(rows)]
    s = Step(rng.standard_normal((rows, vocab)), "f32", hist, [(1.2, 0.1, 0.0)] * rows)
    other = Step(rng.standard_normal((rows, vocab)), "f32", hist, [(1.2, 0.1, 0.0)] * rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    s.run(side.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        check(mtg.lib().mtg_logits_step_dev(ctypes.byref(s.d), side.cuda_stream))
    for _ in range(4):
        s.x = rng.standard_normal((rows, vocab)).astype(np.float32)
        s.hist = [list(rng.integers(0, vocab, 64)) for _ in range(rows)]
        s.xd.copy_(torch.from_numpy(s.x))
        s.keep[0][:-1].copy_(torch.tensor([i for h in s.hist for i in h], dtype=torch.int32))
        s.choice.fill_(-1)
        other.run().verify()
        g.replay()
        torch.cuda.synchronize()
        s.verify()
