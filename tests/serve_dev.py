"""Calls of the serving operators on torch tensors, for the GPU tests: a description filled from a
serve_ref.Batch and device copies of its arrays."""
import ctypes

import numpy as np
import torch

import mtg

TORCH = {"f32": torch.float32, "f16": torch.float16}
MTG = {"f32": mtg.TYPE_F32, "f16": mtg.TYPE_F16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def at(t):
    return None if t is None else t.data_ptr()


class Cache:
    """A batch's cache on the device. layout: how pages and heads lie in memory."""

    def __init__(self, batch, layout="page"):
        self.batch, self.layout = batch, layout
        p, h, s, d = batch.k.shape
        self.table, self.kv_len, self.q_start = dev(batch.table), dev(batch.kv_len), dev(batch.q_start)
        one = s * d
        if layout == "page":        # [page][head][place][dim]
            self.k, self.v = dev(batch.k), dev(batch.v)
            self.page_stride, self.head_stride = h * one, one
            self.kp, self.vp = at(self.k), at(self.v)
        elif layout == "head":      # [head][page][place][dim]
            self.k, self.v = dev(batch.k.transpose(1, 0, 2, 3)), dev(batch.v.transpose(1, 0, 2, 3))
            self.page_stride, self.head_stride = one, p * one
            self.kp, self.vp = at(self.k), at(self.v)
        elif layout == "both":      # [page][k or v][head][place][dim], with a gap behind each page
            gap = 24
            self.pool = torch.full((p, 2 * h * one + gap), float("nan"), dtype=TORCH[batch.kv], device="cuda")
            self.pool[:, :h * one] = dev(batch.k).view(p, -1)
            self.pool[:, h * one:2 * h * one] = dev(batch.v).view(p, -1)
            self.page_stride, self.head_stride = 2 * h * one + gap, one
            self.kp = at(self.pool)
            self.vp = self.kp + h * one * self.pool.element_size()

    def read(self):
        """(k, v) as [page][head][place][dim] on the host."""
        b = self.batch
        if self.layout == "page":
            return self.k.cpu().numpy(), self.v.cpu().numpy()
        if self.layout == "head":
            return tuple(x.cpu().numpy().transpose(1, 0, 2, 3) for x in (self.k, self.v))
        w = b.kv_heads * b.page * b.dim
        return tuple(self.pool[:, i * w:(i + 1) * w].cpu().numpy().reshape(b.k.shape) for i in range(2))

    def desc(self, **kw):
        b = self.batch
        f = dict(k=self.kp, v=self.vp, page_table=at(self.table), kv_len=at(self.kv_len), q_start=at(self.q_start),
                 page_stride=self.page_stride, head_stride=self.head_stride, kv_type=MTG[b.kv], n_pages=b.n_pages,
                 page_size=b.page, table_stride=b.table.shape[1], n_seqs=len(b.lens), n_tokens=b.n_tokens,
                 n_kv_heads=b.kv_heads, head_dim=b.dim)
        f.update(kw)
        return mtg.PagedKv(**f)


def stream():
    return torch.cuda.current_stream().cuda_stream


def check(rc):
    assert rc == 0, (rc, mtg.lib().mtg_last_error(None))


class Attend:
    """A call of mtg_paged_attn_dev with its buffers. q, out: [rows][heads][dim] views with one row stride."""

    def __init__(self, cache, q, out, io, scale, window=0, max_kv=0):
        heads, dim = q.shape[1:]
        self.keep = (cache, q, out)
        self.d = mtg.PagedAttn(kv=cache.desc(), q=at(q), out=at(out), q_stride=q.stride(0), out_stride=out.stride(0),
                               io_type=MTG[io], n_heads=heads, max_kv=max_kv, window=window, scale=scale)
        size = mtg.lib().mtg_paged_attn_workspace(ctypes.byref(self.d))
        if size:
            self.work = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN in every float
            self.d.workspace, self.d.workspace_bytes = at(self.work), size

    def __call__(self, s=None):
        check(mtg.lib().mtg_paged_attn_dev(ctypes.byref(self.d), stream() if s is None else s))
