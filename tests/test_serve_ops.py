"""The serving operators on the CPU: what their entry points refuse before any GPU work, the sizes of
their workspaces, the rotary frequencies, the index rules of the paged cache, the struct layouts."""
import ctypes
import json
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

import mtg
import serve_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BASE = 1 << 40  # an address that nothing here reads: every refusal comes before the GPU is touched


def _kv(**kw):
    f = dict(k=BASE, v=BASE + (1 << 30), page_table=BASE + (2 << 30), kv_len=BASE + (3 << 30), q_start=BASE + (4 << 30),
             page_stride=8 * 16 * 128, head_stride=16 * 128, kv_type=mtg.TYPE_F16, n_pages=10, page_size=16,
             table_stride=5, n_seqs=2, n_tokens=4, n_kv_heads=8, head_dim=128)
    f.update(kw)
    return mtg.PagedKv(**f)


def _rope(kv=None, **kw):
    q = BASE + (8 << 30)
    f = dict(kv=_kv(**(kv or {})), q=q, k_new=q + 4 * 2048, v_new=q + 4 * 24 * 128, q_out=BASE + (9 << 30), freqs=BASE + (10 << 30),
             q_stride=4096, k_stride=4096, v_stride=4096, q_out_stride=2048, io_type=mtg.TYPE_F32, n_heads=16, rot_dim=128,
             eps=1e-6, mscale=1.0)
    f.update(kw)
    return mtg.RopeAppend(**f)


def _attn(kv=None, **kw):
    f = dict(kv=_kv(**(kv or {})), q=BASE + (8 << 30), out=BASE + (9 << 30), q_stride=2048, out_stride=2048,
             workspace=BASE + (11 << 30), workspace_bytes=1 << 30, io_type=mtg.TYPE_F32, n_heads=16, scale=0.1)
    f.update(kw)
    return mtg.PagedAttn(**f)


def _logits(**kw):
    f = dict(logits=BASE, out=BASE + (8 << 30), stride=1000, out_stride=1000, choice=BASE + (9 << 30), io_type=mtg.TYPE_F32,
             rows=3, vocab=1000)
    f.update(kw)
    return mtg.LogitsStep(**f)


BAD_CACHE = [
    (dict(n_seqs=-1), mtg.ERR_INVALID), (dict(n_tokens=-1), mtg.ERR_INVALID), (dict(n_kv_heads=0), mtg.ERR_INVALID),
    (dict(head_dim=96), mtg.ERR_UNSUPPORTED), (dict(head_dim=0), mtg.ERR_UNSUPPORTED),
    (dict(n_seqs=1 << 21), mtg.ERR_UNSUPPORTED), (dict(n_tokens=1 << 23), mtg.ERR_UNSUPPORTED),
    (dict(kv_len=None), mtg.ERR_INVALID), (dict(q_start=None), mtg.ERR_INVALID), (dict(page_table=None), mtg.ERR_INVALID),
    (dict(k=None), mtg.ERR_INVALID), (dict(v=None), mtg.ERR_INVALID), (dict(q_start=BASE + 2), mtg.ERR_INVALID),
    (dict(kv_type=mtg.TYPE_Q8_0), mtg.ERR_UNSUPPORTED), (dict(n_pages=0), mtg.ERR_INVALID), (dict(table_stride=0), mtg.ERR_INVALID),
    (dict(page_size=8), mtg.ERR_UNSUPPORTED), (dict(page_size=24), mtg.ERR_UNSUPPORTED),
    (dict(page_size=1 << 17), mtg.ERR_UNSUPPORTED), (dict(page_size=1 << 16, table_stride=1 << 15), mtg.ERR_UNSUPPORTED),
    (dict(k=BASE + 8), mtg.ERR_UNSUPPORTED), (dict(page_stride=8 * 16 * 128 + 4), mtg.ERR_UNSUPPORTED),
    (dict(page_stride=16 * 128), mtg.ERR_INVALID), (dict(head_stride=-16 * 128), mtg.ERR_INVALID),
]


@pytest.mark.parametrize("bad,status", BAD_CACHE, ids=lambda x: str(x)[:40])
def test_bad_caches_are_refused(bad, status):
    L = mtg.lib()
    r, a = _rope(kv=bad), _attn(kv=bad)
    assert L.mtg_rope_append_dev(ctypes.byref(r), None) == status
    assert b"rope_append" in L.mtg_last_error(None)
    assert L.mtg_paged_attn_dev(ctypes.byref(a), None) == status
    assert b"paged_attn" in L.mtg_last_error(None)


@pytest.mark.parametrize("bad,status", [
    (dict(q=None), mtg.ERR_INVALID), (dict(q_out=None), mtg.ERR_INVALID), (dict(k_new=None), mtg.ERR_INVALID),
    (dict(v_new=None), mtg.ERR_INVALID), (dict(q=None, q_out=None, k_new=None, v_new=None), mtg.ERR_INVALID),
    (dict(rot_dim=130), mtg.ERR_INVALID), (dict(rot_dim=63), mtg.ERR_INVALID), (dict(rot_dim=-2), mtg.ERR_INVALID),
    (dict(n_heads=0), mtg.ERR_INVALID), (dict(freqs=None), mtg.ERR_INVALID), (dict(freqs=BASE + 4), mtg.ERR_INVALID),
    (dict(io_type=mtg.TYPE_Q4_K), mtg.ERR_UNSUPPORTED), (dict(q_stride=2000), mtg.ERR_INVALID),
    (dict(k_stride=1000), mtg.ERR_INVALID), (dict(q_stride=4098), mtg.ERR_UNSUPPORTED), (dict(q=BASE + 8), mtg.ERR_UNSUPPORTED),
    (dict(q_norm=BASE + 4), mtg.ERR_UNSUPPORTED), (dict(kv=dict(kv_type=mtg.TYPE_F32), io_type=mtg.TYPE_F16), mtg.ERR_UNSUPPORTED),
    # q_out one element into q; over k_new; in place with another stride; inside the pages; k and v in one pool
    (dict(q_out=BASE + (8 << 30) + 16), mtg.ERR_INVALID), (dict(q_out=BASE + (8 << 30) + 4 * 1024, q_out_stride=4096), mtg.ERR_INVALID),
    (dict(q_out=BASE + (8 << 30)), mtg.ERR_INVALID), (dict(q_out=BASE + 160), mtg.ERR_INVALID),
    (dict(kv=dict(v=BASE)), mtg.ERR_INVALID),
], ids=lambda x: str(x)[:40])
def test_bad_rotary_calls_are_refused(bad, status):
    r = _rope(**bad)
    assert mtg.lib().mtg_rope_append_dev(ctypes.byref(r), None) == status, mtg.lib().mtg_last_error(None)


@pytest.mark.parametrize("bad,status", [
    (dict(q=None), mtg.ERR_INVALID), (dict(out=None), mtg.ERR_INVALID), (dict(n_heads=12), mtg.ERR_INVALID),
    (dict(n_heads=0), mtg.ERR_INVALID), (dict(io_type=mtg.TYPE_Q8_0), mtg.ERR_UNSUPPORTED),
    (dict(kv=dict(kv_type=mtg.TYPE_F32), io_type=mtg.TYPE_F16), mtg.ERR_UNSUPPORTED), (dict(max_kv=-1), mtg.ERR_INVALID),
    (dict(window=-1), mtg.ERR_INVALID), (dict(scale=float("nan")), mtg.ERR_INVALID), (dict(scale=float("inf")), mtg.ERR_INVALID),
    (dict(q_stride=1024), mtg.ERR_INVALID), (dict(out_stride=2050), mtg.ERR_UNSUPPORTED), (dict(out=BASE + (9 << 30) + 8), mtg.ERR_UNSUPPORTED),
    (dict(out=BASE + (8 << 30) + 32), mtg.ERR_INVALID), (dict(out=BASE + (8 << 30), out_stride=4096), mtg.ERR_INVALID),
    (dict(out=BASE + 4096), mtg.ERR_INVALID),
    (dict(kv=dict(table_stride=4096), workspace=None), mtg.ERR_INVALID),
    (dict(kv=dict(table_stride=4096), workspace=BASE + (11 << 30) + 8), mtg.ERR_INVALID),
    (dict(kv=dict(table_stride=4096), workspace_bytes=64), mtg.ERR_CAPACITY),
    (dict(kv=dict(table_stride=4096), workspace=BASE + (9 << 30)), mtg.ERR_INVALID),
    (dict(kv=dict(n_tokens=1 << 22, table_stride=2), n_heads=1024), mtg.ERR_UNSUPPORTED),
], ids=lambda x: str(x)[:40])
def test_bad_attention_calls_are_refused(bad, status):
    a = _attn(**bad)
    assert mtg.lib().mtg_paged_attn_dev(ctypes.byref(a), None) == status, mtg.lib().mtg_last_error(None)


@pytest.mark.parametrize("bad,status", [
    (dict(rows=-1), mtg.ERR_INVALID), (dict(rows=65536), mtg.ERR_INVALID), (dict(vocab=0), mtg.ERR_INVALID),
    (dict(vocab=(1 << 24) + 1), mtg.ERR_INVALID), (dict(n_history=-1), mtg.ERR_INVALID), (dict(n_bias=-1), mtg.ERR_INVALID),
    (dict(io_type=mtg.TYPE_Q8_0), mtg.ERR_UNSUPPORTED), (dict(logits=None), mtg.ERR_INVALID), (dict(out=None, choice=None), mtg.ERR_INVALID),
    (dict(stride=999), mtg.ERR_INVALID), (dict(out_stride=10), mtg.ERR_INVALID), (dict(history=BASE), mtg.ERR_INVALID),
    (dict(history=BASE, hist_range=BASE), mtg.ERR_INVALID), (dict(bias=BASE), mtg.ERR_INVALID),
    (dict(bias=BASE, bias_ids=BASE), mtg.ERR_INVALID), (dict(mask=BASE, mask_stride=31), mtg.ERR_INVALID),
    (dict(logits=BASE + 2), mtg.ERR_INVALID), (dict(choice=BASE + 2), mtg.ERR_INVALID), (dict(out=BASE + 4), mtg.ERR_INVALID),
    (dict(out=BASE, out_stride=1001), mtg.ERR_INVALID),
    (dict(vocab=4097, stride=4097, out_stride=4097), mtg.ERR_INVALID),
    (dict(vocab=4097, stride=4097, out_stride=4097, workspace=BASE + (10 << 30), workspace_bytes=95), mtg.ERR_CAPACITY),
    (dict(vocab=4097, stride=4097, out_stride=4097, workspace=BASE, workspace_bytes=96), mtg.ERR_INVALID),
], ids=lambda x: str(x)[:40])
def test_bad_logits_calls_are_refused(bad, status):
    a = _logits(**bad)
    assert mtg.lib().mtg_logits_step_dev(ctypes.byref(a), None) == status, mtg.lib().mtg_last_error(None)


@pytest.mark.parametrize("bad", [dict(n_history=(1 << 30) + 1), dict(n_bias=2 ** 31 - 1)], ids=str)
def test_lists_whose_steps_would_pass_31_bits_are_refused(bad):
    a = _logits(history=BASE, hist_range=BASE, penalties=BASE, bias=BASE, bias_ids=BASE, bias_range=BASE, **bad)
    assert mtg.lib().mtg_logits_step_dev(ctypes.byref(a), None) == mtg.ERR_INVALID
    assert mtg.lib().mtg_logits_step_workspace(ctypes.byref(a)) == 0


def test_calls_without_rows_do_nothing():
    L = mtg.lib()
    for kv in (dict(n_seqs=0), dict(n_tokens=0), dict(n_seqs=0, n_tokens=0, k=None, v=None, page_table=None, q_start=None, kv_len=None)):
        r, a = _rope(kv=kv), _attn(kv=kv)
        assert L.mtg_rope_append_dev(ctypes.byref(r), None) == mtg.OK
        assert L.mtg_paged_attn_workspace(ctypes.byref(a)) == 0
        assert L.mtg_paged_attn_dev(ctypes.byref(a), None) == mtg.OK
    empty = _logits(rows=0)
    assert L.mtg_logits_step_dev(ctypes.byref(empty), None) == mtg.OK
    assert L.mtg_rope_append_dev(None, None) == L.mtg_paged_attn_dev(None, None) == L.mtg_logits_step_dev(None, None) == mtg.ERR_INVALID
    assert L.mtg_paged_attn_workspace(None) == L.mtg_logits_step_workspace(None) == 0


def test_workspaces():
    L = mtg.lib()
    size = lambda **kw: L.mtg_paged_attn_workspace(ctypes.byref(_attn(**kw)))  # noqa: E731
    assert size() == 0                                     # 80 positions: one split
    assert size(kv=dict(head_dim=96)) == 0                 # refused
    long = size(kv=dict(table_stride=4096))
    assert long and long % 16 == 0
    # sizes alone decide: no pointer is looked at, and a small max_kv needs no splits
    assert size(kv=dict(table_stride=4096, k=None, v=None, kv_len=None, q_start=None, page_table=None), q=None, out=None) == long
    assert size(kv=dict(table_stride=4096), max_kv=100) == 0
    words = lambda **kw: L.mtg_logits_step_workspace(ctypes.byref(_logits(**kw)))  # noqa: E731
    assert words() == 0 and words(vocab=151936, choice=None) == 0
    assert words(vocab=151936) == 3 * 38 * 16             # a key and marks
    assert words(vocab=151936, rows=33) == (33 * 38 * 8 + 15) // 16 * 16


def test_frequencies():
    for rot in (2, 64, 96, 128):
        f, m = mtg.rope_freqs(rot, 1e6)
        assert m == 1.0 and np.array_equal(f, [1e6 ** (-2.0 * i / rot) for i in range(rot // 2)])
        g, m = mtg.rope_freqs(rot, 1e6, mtg.ROPE_LINEAR, factor=4.0)
        assert m == 1.0 and np.array_equal(g, f / 4)
    f, _ = mtg.rope_freqs(64, 1e4)
    g, m = mtg.rope_freqs(64, 1e4, mtg.ROPE_NTK, factor=8.0)
    # the fastest pair keeps its turns, the slowest is slowed by the whole factor
    assert m == 1.0 and g[0] == f[0] and abs(g[-1] * 8 / f[-1] - 1) < 1e-12 and (np.diff(f / g) > 0).all()
    g, m = mtg.rope_freqs(64, 1e4, mtg.ROPE_YARN, factor=8.0, orig_ctx=4096)
    turns = f * 4096 / (2 * math.pi)
    assert m == np.float32(0.1 * math.log(8.0) + 1)
    assert np.array_equal(g[turns > 40], f[turns > 40])     # a whole pair index outside the ramp at least
    assert np.allclose(g[turns < 0.7], f[turns < 0.7] / 8, rtol=1e-15)
    between = (turns < 30) & (turns > 1.1)
    assert between.any() and (g[between] < f[between]).all() and (g[between] > f[between] / 8).all()
    g, m = mtg.rope_freqs(64, 1e4, mtg.ROPE_YARN, factor=1.0, orig_ctx=4096)
    assert m == 1.0 and np.allclose(g, f, rtol=1e-15)
    for bad in (dict(rot_dim=63, base=1e4), dict(rot_dim=0, base=1e4), dict(rot_dim=64, base=1.0), dict(rot_dim=64, base=float("inf")),
                dict(rot_dim=64, base=1e4, factor=0.5), dict(rot_dim=64, base=1e4, factor=float("nan")), dict(rot_dim=64, base=1e4, kind=4),
                dict(rot_dim=64, base=1e4, kind=mtg.ROPE_YARN, orig_ctx=0.0), dict(rot_dim=2, base=1e4, kind=mtg.ROPE_NTK),
                dict(rot_dim=64, base=1e4, kind=mtg.ROPE_YARN, orig_ctx=4096, beta_fast=1.0)):
        with pytest.raises(mtg.MtgError):
            mtg.rope_freqs(**bad)


def test_paged_index_rules():
    exe = os.path.join(ROOT, "tests", "cpp", "bin", "test_paged_kv")
    if not os.path.exists(exe):
        import build
        build.build_cpp_tests()
    p = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=60)
    assert p.returncode == 0, p.stderr
    assert json.loads(p.stdout) == {"record": "pagedKv", "failures": 0}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layouts(tmp_path):
    structs = {"mtg_paged_kv": mtg.PagedKv, "mtg_rope_append": mtg.RopeAppend, "mtg_paged_attn": mtg.PagedAttn,
               "mtg_logits_step": mtg.LogitsStep}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "%s/include/mtg_verify.h"' % ROOT, "int main(void){"]
    for name, s in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f, name, f) for f, _ in s._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout
    got = dict(line.split() for line in out.strip().splitlines())
    for name, s in structs.items():
        assert int(got[name]) == ctypes.sizeof(s), name
        for f, _ in s._fields_:
            assert int(got["%s.%s" % (name, f)]) == getattr(s, f).offset, (name, f)


def test_the_plain_forms_against_the_library_where_it_has_them():
    """serve_ref on cases whose answer the library's host functions give: the greedy choice with a
    repetition penalty over up to 100 ids, and the rotation of one pair by hand."""
    rng = np.random.default_rng(5)
    for n in (1, 7, 300):
        x = rng.standard_normal(n).astype(np.float32)
        hist = rng.integers(-2, n + 2, 60)
        y, _ = serve_ref.logits_row(x, hist, (1.3, 0, 0), [], None)
        assert serve_ref.first_max(y, None) == mtg.greedy_choice(x, hist, 1.3)
    y, size = serve_ref.rotate(np.array([[3.0, 4.0, 5.0, 6.0]]), 2.0, np.array([math.pi / 4]), 2, True, 1.0)
    assert np.allclose(y, [[-4.0, 3.0, 5.0, 6.0]]) and np.array_equal(size, [[7, 7, 5, 6]])
