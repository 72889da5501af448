"""The serving operators one after the other, as a program runs them: a batch of recordings through a
prompt chunk, drafted tokens and single tokens over one paged cache. Each step's rows are turned and
stored, attend over the pages, are projected to logits and choose their next ids; the same program
in 64 bits, from the same rows, has to agree with what each operator gave."""
import ctypes

import numpy as np
import pytest

import mtg
from serve_ref import HALF, TYPES, Batch, attend, attend_tolerance, freqs, logits_row, first_max, rotate, rotate_tolerance

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import MTG, Attend, Cache, at, check, dev, stream  # noqa: E402


@pytest.mark.parametrize("io,kv", [("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
def test_chunk_then_drafts_then_tokens(io, kv):
    rng = np.random.default_rng(21)
    heads, hk, dim, page, vocab, seqs = 4, 2, 64, 16, 5003, 3
    wide = (heads + 2 * hk) * dim
    scale, f = dim ** -0.5, freqs(dim)
    lens = [0, 0, 0]
    history = [[], [], []]
    plan = [(70, 33, 1), (5, 8, 2), (1, 1, 1), (1, 0, 1)]
    total = [sum(p[b] for p in plan) for b in range(seqs)]
    b = Batch(rng, [(0, t) for t in total], hk, dim, page, kv, filled=False)
    cache = Cache(b)
    gain = (1 + 0.1 * rng.standard_normal(dim)).astype(np.float32)
    head = (rng.standard_normal((vocab, heads * dim)) * 0.2).astype(np.float32)
    gd, fd, wd = dev(gain), dev(f), dev(head)
    for new in plan:
        lens = [a + n for a, n in zip(lens, new)]
        b.lens = list(zip(new, lens))
        b.kv_len = np.array(lens, np.int32)
        b.q_start = np.cumsum([0] + list(new)).astype(np.int32)
        b.n_tokens = n = int(b.q_start[-1])
        cache.kv_len.copy_(torch.from_numpy(b.kv_len))
        cache.q_start.copy_(torch.from_numpy(b.q_start))
        x = rng.standard_normal((n, heads + 2 * hk, dim)).astype(TYPES[io])
        xd = dev(x)
        e = xd.element_size()
        q = torch.empty(n, heads, dim, dtype=xd.dtype, device="cuda")
        out = torch.empty_like(q)
        rope = mtg.RopeAppend(kv=cache.desc(), q=at(xd), k_new=at(xd) + heads * dim * e, v_new=at(xd) + (heads + hk) * dim * e,
                              q_out=at(q), freqs=at(fd), q_norm=at(gd), k_norm=at(gd), q_stride=wide, k_stride=wide, v_stride=wide,
                              q_out_stride=heads * dim, io_type=MTG[io], n_heads=heads, rot_dim=dim, eps=1e-6, mscale=1.0)
        check(mtg.lib().mtg_rope_append_dev(ctypes.byref(rope), stream()))
        Attend(cache, q, out, io, scale)()
        logits = (out.float().view(n, -1) @ wd.t()).contiguous()
        got_logits = logits.cpu().numpy()
        # the last row of each sequence chooses; its history is what its sequence chose before
        flat = np.array([i for h in history for i in h] + [0], np.int32)
        ends = np.cumsum([0] + [len(h) for h in history])
        seq_of = np.repeat(np.arange(seqs), new)
        ranges = np.array([[ends[s], ends[s + 1]] for s in seq_of], np.int32)
        allowed = rng.random((n, vocab)) < 0.5
        words = np.pad(np.packbits(allowed, axis=1, bitorder="little"), ((0, 0), (0, -((vocab + 7) // 8) % 4)))
        words = words.view(np.uint32)
        keep = [dev(flat), dev(ranges), dev(np.tile(np.float32([1.3, 0.1, 0.2]), (n, 1))), dev(words.view(np.int32))]
        shaped, choice = torch.empty_like(logits), torch.empty(n, dtype=torch.int32, device="cuda")
        step = mtg.LogitsStep(logits=at(logits), out=at(shaped), stride=vocab, out_stride=vocab, history=at(keep[0]),
                              hist_range=at(keep[1]), penalties=at(keep[2]), mask=at(keep[3]), mask_stride=words.shape[1],
                              choice=at(choice), io_type=mtg.TYPE_F32, rows=n, vocab=vocab, n_history=len(flat) - 1)
        size = mtg.lib().mtg_logits_step_workspace(ctypes.byref(step))
        work = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        step.workspace, step.workspace_bytes = at(work), size
        check(mtg.lib().mtg_logits_step_dev(ctypes.byref(step), stream()))
        torch.cuda.synchronize()

        # rows: rotated as in 64 bits, q and the new places of the cache
        gq = q.cpu().numpy()
        b.k, b.v = (a.copy() for a in cache.read())
        for t, (s, p) in b.positions().items():
            y, sz = rotate(x[t, :heads], p, f, dim, False, 1.0, gain)
            assert (np.abs(gq[t] - y) <= rotate_tolerance(y, sz, io)).all()
            y, sz = rotate(x[t, heads:heads + hk], p, f, dim, False, 1.0, gain)
            where = (b.page_of(s, p), slice(None), p % page)
            assert (np.abs(b.k[where] - y) <= rotate_tolerance(y, sz, kv)).all()
            v = x[t, heads + hk:].astype(np.float64)
            assert (np.abs(b.v[where] - v) <= np.abs(v) * HALF[kv]).all()
        # attention over all that was stored so far
        want, sz, sharp = attend(b, gq, scale)
        got = out.cpu().numpy()
        assert (np.abs(got - want) <= attend_tolerance(want, sz, sharp, io, max(lens), dim)).all()
        # logits and choices
        gs, gc = shaped.cpu().numpy(), choice.cpu().numpy()
        for t in range(n):
            y, sz = logits_row(got_logits[t], history[seq_of[t]], (1.3, 0.1, 0.2), [], allowed[t])
            fine = allowed[t]
            assert (gs[t][~fine] == -np.inf).all()
            assert (np.abs(gs[t][fine] - y[fine]) <= 5 * sz[fine] * 2.0 ** -24 + np.abs(y[fine]) * 2.0 ** -24).all()
            assert gc[t] == first_max(gs[t], allowed[t])
        for s in range(seqs):
            if new[s]:
                history[s] += [int(c) for c in gc[b.q_start[s]:b.q_start[s + 1]]]
