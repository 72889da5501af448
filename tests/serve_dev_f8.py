"""Calls of the operators over a cache in 8 bits on torch tensors, for the GPU tests (see serve_dev.py)."""
import ctypes

import torch

import mtg
from serve_dev import MTG, at, check, dev, stream  # noqa: F401


class Cache:
    """A serve_ref_f8.Batch's cache on the device. layout: how pages, heads and scales lie in memory."""

    def __init__(self, batch, layout="page"):
        self.batch, self.layout = batch, layout
        p, h, s, d = batch.kc.shape
        n = s // 16
        self.table, self.kv_len, self.q_start = dev(batch.table), dev(batch.kv_len), dev(batch.q_start)
        one = s * d
        if layout == "page":        # [page][head][place][dim], [page][head][block]
            self.k, self.v, self.ks, self.vs = (dev(x) for x in (batch.kc, batch.vc, batch.ks, batch.vs))
            self.page_stride, self.head_stride, self.scale_page, self.scale_head = h * one, one, h * n, n
            self.at = [at(x) for x in (self.k, self.v, self.ks, self.vs)]
        elif layout == "head":      # [head][page][place][dim], [head][page][block]
            self.k, self.v, self.ks, self.vs = (dev(x.swapaxes(0, 1)) for x in (batch.kc, batch.vc, batch.ks, batch.vs))
            self.page_stride, self.head_stride, self.scale_page, self.scale_head = one, p * one, n, p * n
            self.at = [at(x) for x in (self.k, self.v, self.ks, self.vs)]
        elif layout == "both":      # [page][k or v][head][place][dim] with a gap behind each page; scales likewise, odd gap
            gap = 48
            self.pool = torch.full((p, 2 * h * one + gap), 127, dtype=torch.uint8, device="cuda")
            self.pool[:, :h * one] = dev(batch.kc).view(p, -1)
            self.pool[:, h * one:2 * h * one] = dev(batch.vc).view(p, -1)
            self.scales = torch.full((p, 2 * h * n + 3), 255, dtype=torch.uint8, device="cuda")
            self.scales[:, :h * n] = dev(batch.ks).view(p, -1)
            self.scales[:, h * n:2 * h * n] = dev(batch.vs).view(p, -1)
            self.page_stride, self.head_stride, self.scale_page, self.scale_head = 2 * h * one + gap, one, 2 * h * n + 3, n
            self.at = [at(self.pool), at(self.pool) + h * one, at(self.scales), at(self.scales) + h * n]

    def read(self):
        """(k codes, v codes, k scales, v scales) on the host, as the batch has them."""
        b = self.batch
        shapes = [x.shape for x in (b.kc, b.vc, b.ks, b.vs)]
        if self.layout == "page":
            return tuple(x.cpu().numpy() for x in (self.k, self.v, self.ks, self.vs))
        if self.layout == "head":
            return tuple(x.cpu().numpy().swapaxes(0, 1) for x in (self.k, self.v, self.ks, self.vs))
        w, n = b.kc[0].size, b.ks[0].size
        assert (self.pool[:, 2 * w:] == 127).all() and (self.scales[:, 2 * n:] == 255).all()
        parts = [self.pool[:, :w], self.pool[:, w:2 * w], self.scales[:, :n], self.scales[:, n:2 * n]]
        return tuple(x.cpu().numpy().reshape(s) for x, s in zip(parts, shapes))

    def desc(self, **kw):
        b = self.batch
        f = dict(k=self.at[0], v=self.at[1], page_table=at(self.table), kv_len=at(self.kv_len), q_start=at(self.q_start),
                 page_stride=self.page_stride, head_stride=self.head_stride, kv_type=mtg.TYPE_F8_E4M3, n_pages=b.n_pages,
                 page_size=b.page, table_stride=b.table.shape[1], n_seqs=len(b.lens), n_tokens=b.n_tokens,
                 n_kv_heads=b.kv_heads, head_dim=b.dim)
        f.update(kw)
        return mtg.PagedKv(**f)

    def scale_desc(self):
        return mtg.F8Scales(k=self.at[2], v=self.at[3], page_stride=self.scale_page, head_stride=self.scale_head)


def append(cache, qkv, heads, kv_heads, dim, q_out, io, freqs=None, rot=0, positions=None, inter=False, norms=(None, None), mscale=1.0,
           eps=1e-6, with_q=True, with_kv=True, call=True):
    """mtg_rope_append_f8_dev on rows of q | k | v side by side."""
    x, eb, width = at(qkv), qkv.element_size(), qkv.stride(0)
    a = mtg.RopeAppend(kv=cache.desc(), freqs=at(freqs), positions=at(positions), q_norm=at(norms[0]), k_norm=at(norms[1]),
                       q_stride=width, k_stride=width, v_stride=width, io_type=MTG[io], rot_dim=rot, interleaved=int(inter), eps=eps,
                       mscale=mscale)
    if with_q:
        a.q, a.q_out, a.q_out_stride, a.n_heads = x, at(q_out), q_out.stride(0), heads
    if with_kv:
        a.k_new, a.v_new = x + heads * dim * eb, x + (heads + kv_heads) * dim * eb
    d = mtg.RopeAppendF8(a=a, scales=cache.scale_desc())
    if call:
        check(mtg.lib().mtg_rope_append_f8_dev(ctypes.byref(d), stream()))
    return d


class Attend:
    """A call of mtg_paged_attn_f8_dev with its buffers. q, out: [rows][heads][dim] views with one row stride."""

    def __init__(self, cache, q, out, io, scale, window=0, max_kv=0, sink=0):
        heads = q.shape[1]
        self.keep = (cache, q, out)
        a = mtg.PagedAttn(kv=cache.desc(), q=at(q), out=at(out), q_stride=q.stride(0), out_stride=out.stride(0),
                          io_type=MTG[io], n_heads=heads, max_kv=max_kv, window=window, scale=scale)
        self.d = mtg.PagedAttnF8(a=a, scales=cache.scale_desc(), sink=sink)
        size = mtg.lib().mtg_paged_attn_f8_workspace(ctypes.byref(self.d))
        if size:
            self.work = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN in every float
            self.d.a.workspace, self.d.a.workspace_bytes = at(self.work), size

    def __call__(self, s=None):
        check(mtg.lib().mtg_paged_attn_f8_dev(ctypes.byref(self.d), stream() if s is None else s))
