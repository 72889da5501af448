"""The serving operators over a cache in 8 bits, one after the other as a program runs them: rows are turned and stored as codes, attend
over the pages, are projected to logits, get their penalties and mask, and an id is drawn. Each step against 64 bits, from
what the steps before it gave. Also the calls on streams of their own, and codes beyond 32 bits."""
import ctypes

import numpy as np
import pytest

import mtg
import serve_ref_f8 as ref
from sample_ref import answers
from serve_ref import TYPES, freqs, logits_row, rotate, rotate_tolerance

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from serve_dev import MTG, TORCH, at, check, dev, stream  # noqa: E402
from serve_dev_f8 import Attend, Cache, append  # noqa: E402


@pytest.mark.parametrize("io", ["f32", "f16"])
@pytest.mark.parametrize("dim,window,sink", [(64, 0, 0), (128, 40, 4)])
def test_chunk_then_drafts_then_tokens(io, dim, window, sink):
    rng = np.random.default_rng(31 + dim)
    heads, hk, page, vocab, seqs = 4, 2, 16, 5003, 3
    scale, f = dim ** -0.5, freqs(dim)
    lens, history = [0] * seqs, [[] for _ in range(seqs)]
    plan = [(70, 33, 1), (5, 8, 2), (1, 1, 1), (1, 0, 1), (1, 1, 1)]
    b = ref.Batch(rng, [(0, sum(p[i] for p in plan)) for i in range(seqs)], hk, dim, page, filled=False)
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
        q = torch.empty(n, heads, dim, dtype=TORCH[io], device="cuda")
        out = torch.empty_like(q)
        append(cache, dev(x), heads, hk, dim, q, io, freqs=fd, rot=dim, norms=(gd, gd))
        Attend(cache, q, out, io, scale, window, sink=sink)()
        logits = (out.float().view(n, -1) @ wd.t()).contiguous()
        got_logits = logits.cpu().numpy()
        # penalties and a mask over each row, with what its sequence chose before
        flat = np.array([i for h in history for i in h] + [0], np.int32)
        ends = np.cumsum([0] + [len(h) for h in history])
        seq_of = np.repeat(np.arange(seqs), new)
        ranges = np.array([[ends[s], ends[s + 1]] for s in seq_of], np.int32)
        allowed = rng.random((n, vocab)) < 0.5
        words = np.pad(np.packbits(allowed, axis=1, bitorder="little"), ((0, 0), (0, -((vocab + 7) // 8) % 4))).view(np.uint32)
        keep = [dev(flat), dev(ranges), dev(np.tile(np.float32([1.3, 0.1, 0.2]), (n, 1))), dev(words.view(np.int32))]
        shaped = torch.empty_like(logits)
        step = mtg.LogitsStep(logits=at(logits), out=at(shaped), stride=vocab, out_stride=vocab, history=at(keep[0]), hist_range=at(keep[1]),
                              penalties=at(keep[2]), mask=at(keep[3]), mask_stride=words.shape[1], io_type=mtg.TYPE_F32, rows=n, vocab=vocab,
                              n_history=len(flat) - 1)
        size = mtg.lib().mtg_logits_step_workspace(ctypes.byref(step))
        work = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        step.workspace, step.workspace_bytes = at(work), size
        check(mtg.lib().mtg_logits_step_dev(ctypes.byref(step), stream()))
        settings = np.float32([[(0.8, 0.95, 0.01), (0.0, 1.0, 0.0), (3.0, 1.0, 0.0)][s] for s in seq_of])
        top_k, uniform = np.array([(50, 0, 0)[s] for s in seq_of], np.int32), rng.random(n).astype(np.float32)
        drawn = [dev(settings), dev(top_k), dev(uniform)]
        choice, prob = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")
        draw = mtg.Sample(logits=at(shaped), stride=vocab, settings=at(drawn[0]), top_k=at(drawn[1]), uniform=at(drawn[2]), choice=at(choice),
                          prob=at(prob), io_type=mtg.TYPE_F32, rows=n, vocab=vocab)
        size = mtg.lib().mtg_sample_workspace(ctypes.byref(draw))
        work2 = torch.empty(size, dtype=torch.uint8, device="cuda")
        draw.workspace, draw.workspace_bytes = at(work2), size
        check(mtg.lib().mtg_sample_dev(ctypes.byref(draw), stream()))
        torch.cuda.synchronize()

        gq = q.cpu().numpy()
        new_k, size_k = np.full((n, hk, dim), np.nan), np.zeros((n, hk, dim))
        for t, (s, p) in b.positions().items():
            y, sz = rotate(x[t, :heads], p, f, dim, False, 1.0, gain)
            assert (np.abs(gq[t] - y) <= rotate_tolerance(y, sz, io)).all()
            new_k[t], sz = rotate(x[t, heads:heads + hk], p, f, dim, False, 1.0, gain)
            size_k[t] = sz * 2.0 ** -18
        left = cache.read()
        ref.check_append(b, "k", left[0], left[2], new_k, size_k)
        ref.check_append(b, "v", left[1], left[3], x[:, heads + hk:].astype(np.float64), None)
        b.kc, b.vc, b.ks, b.vs = (a.copy() for a in left)
        b.values()
        form = ref.attend(b, gq, scale, window, sink)
        assert (np.abs(out.cpu().numpy() - form[0]) <= ref.attend_tolerance(b, gq, form, scale, io, max(lens))).all()
        gs, gc, gp = shaped.cpu().numpy(), choice.cpu().numpy(), prob.cpu().numpy().astype(np.float64)
        for t in range(n):
            y, sz = logits_row(got_logits[t], history[seq_of[t]], (1.3, 0.1, 0.2), [], allowed[t])
            fine = allowed[t]
            assert (gs[t][~fine] == -np.inf).all()
            assert (np.abs(gs[t][fine] - y[fine]) <= 5 * sz[fine] * 2.0 ** -24 + np.abs(y[fine]) * 2.0 ** -24).all()
            want = answers(gs[t], *settings[t], int(top_k[t]), uniform[t])
            assert int(gc[t]) in want and allowed[t][gc[t]]
            assert any(abs(gp[t] - w) <= w * 2.0 ** -23 for w in want[int(gc[t])])
        for s in range(seqs):
            history[s] += [int(c) for c in gc[b.q_start[s]:b.q_start[s + 1]]]


def test_two_batches_on_two_streams():
    """Each side's calls on a stream of its own, caches and workspaces apart, in turn; as the same calls one by one."""
    rng = np.random.default_rng(5)
    heads, hk, dim = 4, 2, 64
    f = dev(freqs(dim))
    sides = []
    for lens in ([(1, 700), (3, 90)], [(120, 500)]):
        b = ref.Batch(rng, lens, hk, dim, 16)
        x = dev(rng.standard_normal((b.n_tokens, heads + 2 * hk, dim)).astype(np.float16))
        caches = [Cache(b) for _ in range(2)]
        qs, outs = [[torch.empty(b.n_tokens, heads, dim, dtype=torch.float16, device="cuda") for _ in range(2)] for _ in range(2)]
        calls = [Attend(c, q, o, "f16", 0.1) for c, q, o in zip(caches, qs, outs)]
        sides.append((x, caches, qs, outs, calls, torch.cuda.Stream()))
    for x, caches, qs, outs, calls, _ in sides:
        for _ in range(3):
            append(caches[0], x, heads, hk, dim, qs[0], "f16", freqs=f, rot=dim)
            calls[0]()
    torch.cuda.synchronize()
    for _ in range(3):
        for x, caches, qs, outs, calls, s in sides:
            with torch.cuda.stream(s):
                append(caches[1], x, heads, hk, dim, qs[1], "f16", freqs=f, rot=dim)
                calls[1]()
    torch.cuda.synchronize()
    for x, caches, qs, outs, calls, _ in sides:
        assert torch.equal(qs[0], qs[1]) and torch.equal(outs[0], outs[1])
        assert all(np.array_equal(a, c) for a, c in zip(caches[0].read(), caches[1].read()))


@pytest.mark.parametrize("new", [1, 30])
def test_codes_beyond_32_bits(new):
    """Pages 2^32 bytes apart, and their scales."""
    rng = np.random.default_rng(12)
    far, heads, hk, dim = 1 << 32, 4, 2, 64
    b = ref.Batch(rng, [(new, 40)], hk, dim, 16, spare=0)
    b.table[0, :3] = [1, 0, 2]
    b.n_pages = 3
    for codes, scales in ((b.kc, b.ks), (b.vc, b.vs)):  # every place holds a number, for the pages are exchanged
        codes[:] = rng.integers(0, 127, codes.shape) + 128 * rng.integers(0, 2, codes.shape)
        scales[:] = rng.integers(110, 130, scales.shape)
    b.values()
    pools = [torch.empty(2 * far + 4096, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty(2 * far + 16, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for pool, host in zip(pools + scales, (b.kc, b.vc, b.ks, b.vs)):
        for p in range(3):
            pool[p * far:p * far + host[p].size] = dev(host[p]).view(-1)
    x = rng.standard_normal((new, heads + 2 * hk, dim)).astype(np.float32)
    qkv, out = dev(x), torch.empty(new, heads, dim, device="cuda")
    fd = dev(freqs(dim))
    d = append(Cache(b), qkv, heads, hk, dim, out, "f32", freqs=fd, rot=dim, call=False)
    d.a.kv.k, d.a.kv.v, d.a.kv.page_stride = at(pools[0]), at(pools[1]), far
    d.scales = mtg.F8Scales(k=at(scales[0]), v=at(scales[1]), page_stride=far, head_stride=1)
    check(mtg.lib().mtg_rope_append_f8_dev(ctypes.byref(d), stream()))
    torch.cuda.synchronize()
    got = [np.stack([pool[p * far:p * far + host[0].size].cpu().numpy().reshape(host[0].shape) for p in range(3)])
           for pool, host in zip(pools + scales, (b.kc, b.vc, b.ks, b.vs))]
    new_k, size_k = np.zeros((new, hk, dim)), np.zeros((new, hk, dim))
    for t, (_, p) in b.positions().items():
        new_k[t], s = rotate(x[t, heads:heads + hk], p, freqs(dim), dim, False, 1.0)
        size_k[t] = s * 2.0 ** -18
    ref.check_append(b, "k", got[0], got[2], new_k, size_k)
    ref.check_append(b, "v", got[1], got[3], x[:, heads + hk:].astype(np.float64), None)
