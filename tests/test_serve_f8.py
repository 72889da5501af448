"""The operators over a cache in 8 bits on the CPU: what their entry points refuse before any GPU work, the index rules,
the struct layouts, and the plain forms against themselves."""
import ctypes
import shutil
import subprocess

import numpy as np
import pytest

import mtg
import serve_ref_f8 as ref
from test_cpp_interfaces import _run
from test_serve_ops import BAD_CACHE, BASE, ROOT, _attn, _rope

SCALES = dict(k=BASE + (16 << 30) + 1, v=BASE + (17 << 30) + 3, page_stride=8, head_stride=1)


def _rope_f8(kv=None, scales=None, **kw):
    kv = {"kv_type": mtg.TYPE_F8_E4M3, **(kv or {})}
    return mtg.RopeAppendF8(a=_rope(kv=kv, **kw), scales=mtg.F8Scales(**{**SCALES, **(scales or {})}))


def _attn_f8(kv=None, scales=None, sink=0, **kw):
    kv = {"kv_type": mtg.TYPE_F8_E4M3, **(kv or {})}
    return mtg.PagedAttnF8(a=_attn(kv=kv, **kw), scales=mtg.F8Scales(**{**SCALES, **(scales or {})}), sink=sink)


def _append(d):
    return mtg.lib().mtg_rope_append_f8_dev(ctypes.byref(d), None)


def _attend(d):
    return mtg.lib().mtg_paged_attn_f8_dev(ctypes.byref(d), None)


BAD_F8 = [(b, s) for b, s in BAD_CACHE if "kv_type" not in b and b != dict(page_stride=8 * 16 * 128 + 4)] + [
    (dict(kv_type=mtg.TYPE_F16), mtg.ERR_UNSUPPORTED), (dict(kv_type=mtg.TYPE_F32), mtg.ERR_UNSUPPORTED),
    (dict(kv_type=mtg.TYPE_Q8_0), mtg.ERR_UNSUPPORTED), (dict(page_stride=8 * 16 * 128 + 8), mtg.ERR_UNSUPPORTED)]


@pytest.mark.parametrize("bad,status", BAD_F8, ids=lambda x: str(x)[:40])
def test_bad_caches_are_refused(bad, status):
    assert _append(_rope_f8(kv=bad)) == status
    assert b"rope_append_f8" in mtg.lib().mtg_last_error(None)
    assert _attend(_attn_f8(kv=bad)) == status
    assert b"paged_attn_f8" in mtg.lib().mtg_last_error(None)


@pytest.mark.parametrize("call", ["rope", "attn"])
def test_the_other_operators_do_not_take_codes(call):
    L = mtg.lib()
    d = (_rope if call == "rope" else _attn)(kv=dict(kv_type=mtg.TYPE_F8_E4M3))
    f = L.mtg_rope_append_dev if call == "rope" else L.mtg_paged_attn_dev
    assert f(ctypes.byref(d), None) == mtg.ERR_UNSUPPORTED


# where the calls' other arrays lie, from test_serve_ops._rope
ARRAYS = dict(k=(BASE, 10 * 8 * 16 * 128), v=(BASE + (1 << 30), 10 * 8 * 16 * 128), page_table=(BASE + (2 << 30), 40), kv_len=(BASE + (3 << 30), 8),
              q_start=(BASE + (4 << 30), 12), q=(BASE + (8 << 30), 4 * 4 * 4096), q_out=(BASE + (9 << 30), 4 * 4 * 2048),
              freqs=(BASE + (10 << 30), 4 * 128))


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("other", ARRAYS)
def test_scales_that_share_a_byte_with_another_array_are_refused(which, other):
    at, size = ARRAYS[other]
    for place in (at - 79, at + size - 1):
        assert _append(_rope_f8(scales={which: place})) == mtg.ERR_INVALID, mtg.lib().mtg_last_error(None)
        assert b"scales" in mtg.lib().mtg_last_error(None)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(v=SCALES["k"]), dict(v=SCALES["k"] + 79), dict(page_stride=-8),
                                 dict(head_stride=-1), dict(page_stride=4), dict(head_stride=0), dict(page_stride=1 << 41)], ids=str)
def test_bad_scales_are_refused(bad):
    assert _append(_rope_f8(scales=bad)) == mtg.ERR_INVALID


@pytest.mark.parametrize("bad,status", [
    (dict(io_type=mtg.TYPE_F8_E4M3), mtg.ERR_UNSUPPORTED), (dict(io_type=mtg.TYPE_Q8_0), mtg.ERR_UNSUPPORTED), (dict(rot_dim=63), mtg.ERR_INVALID),
    (dict(q=None), mtg.ERR_INVALID), (dict(v_new=None), mtg.ERR_INVALID), (dict(q_out=BASE + (8 << 30)), mtg.ERR_INVALID),
    (dict(q_out=BASE + 160), mtg.ERR_INVALID), (dict(kv=dict(v=BASE)), mtg.ERR_INVALID), (dict(freqs=None), mtg.ERR_INVALID),
    (dict(n_heads=0), mtg.ERR_INVALID), (dict(q_stride=4098), mtg.ERR_UNSUPPORTED)], ids=lambda x: str(x)[:40])
def test_bad_rotary_calls_are_refused(bad, status):
    assert _append(_rope_f8(**bad)) == status


@pytest.mark.parametrize("bad,status", [
    (dict(q=None), mtg.ERR_INVALID), (dict(out=None), mtg.ERR_INVALID), (dict(n_heads=12), mtg.ERR_INVALID), (dict(n_heads=0), mtg.ERR_INVALID),
    (dict(io_type=mtg.TYPE_Q8_0), mtg.ERR_UNSUPPORTED), (dict(io_type=mtg.TYPE_F8_E4M3), mtg.ERR_UNSUPPORTED), (dict(max_kv=-1), mtg.ERR_INVALID),
    (dict(window=-1), mtg.ERR_INVALID), (dict(sink=-1), mtg.ERR_INVALID), (dict(window=5, sink=2 ** 30 + 1), mtg.ERR_INVALID),
    (dict(scale=float("nan")), mtg.ERR_INVALID), (dict(scale=3e38), mtg.ERR_INVALID), (dict(out_stride=2050), mtg.ERR_UNSUPPORTED),
    (dict(out=BASE + (8 << 30) + 32), mtg.ERR_INVALID), (dict(out=BASE + 4096), mtg.ERR_INVALID),
    (dict(kv=dict(table_stride=4096), workspace=None), mtg.ERR_INVALID), (dict(kv=dict(table_stride=4096), workspace_bytes=64), mtg.ERR_CAPACITY),
    (dict(kv=dict(table_stride=4096), workspace=BASE + (9 << 30)), mtg.ERR_INVALID),
    # scales: missing, in the pages, under out, under the workspace
    (dict(scales=dict(k=None)), mtg.ERR_INVALID), (dict(scales=dict(v=BASE + 100)), mtg.ERR_INVALID),
    (dict(scales=dict(page_stride=1)), mtg.ERR_INVALID), (dict(scales=dict(v=BASE + (9 << 30) + 4 * 4 * 2048 - 1)), mtg.ERR_INVALID),
    (dict(scales=dict(k=BASE + (9 << 30) - 79)), mtg.ERR_INVALID), (dict(kv=dict(table_stride=4096), scales=dict(k=BASE + (11 << 30))), mtg.ERR_INVALID),
], ids=lambda x: str(x)[:40])
def test_bad_attention_calls_are_refused(bad, status):
    assert _attend(_attn_f8(**bad)) == status, mtg.lib().mtg_last_error(None)


def test_attention_workspaces():
    size = lambda **kw: mtg.lib().mtg_paged_attn_f8_workspace(ctypes.byref(_attn_f8(**kw)))  # noqa: E731
    assert size() == 0 and size(kv=dict(head_dim=96)) == 0 and size(kv=dict(table_stride=4096), sink=-1) == 0
    long = size(kv=dict(table_stride=4096))
    assert long and long % 16 == 0
    assert size(kv=dict(table_stride=4096, k=None, v=None, kv_len=None, q_start=None, page_table=None), q=None, out=None,
                scales=dict(k=None, v=None)) == long
    assert size(kv=dict(table_stride=4096), max_kv=100) == 0
    # a window bounds what is gone over; the first positions add to it, but say nothing without a window
    assert size(kv=dict(table_stride=4096), window=40) == 0 and size(kv=dict(table_stride=4096), window=40, sink=4000) > 0
    assert size(kv=dict(table_stride=4096), sink=4000) == long


def test_calls_without_rows_do_nothing():
    for kv in (dict(n_seqs=0), dict(n_tokens=0), dict(n_seqs=0, n_tokens=0, k=None, v=None, page_table=None, q_start=None, kv_len=None)):
        assert _attend(_attn_f8(kv=kv, scales=dict(k=None, v=None))) == mtg.OK
        assert mtg.lib().mtg_paged_attn_f8_workspace(ctypes.byref(_attn_f8(kv=kv))) == 0
    assert mtg.lib().mtg_paged_attn_f8_dev(None, None) == mtg.ERR_INVALID
    assert mtg.lib().mtg_paged_attn_f8_workspace(None) == 0
    for kv in (dict(n_seqs=0), dict(n_tokens=0), dict(n_seqs=0, n_tokens=0, k=None, v=None, page_table=None, q_start=None, kv_len=None)):
        assert _append(_rope_f8(kv=kv, scales=dict(k=None, v=None))) == mtg.OK
    assert mtg.lib().mtg_rope_append_f8_dev(None, None) == mtg.ERR_INVALID


def test_index_rules():
    assert _run("test_paged_f8", 60) == {"record": "pagedF8", "failures": 0}


STRUCTS = {"mtg_f8_scales": mtg.F8Scales, "mtg_rope_append_f8": mtg.RopeAppendF8, "mtg_paged_attn_f8": mtg.PagedAttnF8}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("name", STRUCTS)
def test_struct_layouts(tmp_path, name):
    s = STRUCTS[name]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "%s/include/mtg_verify.h"' % ROOT, "int main(void){",
             'printf("%%zu\\n", sizeof(%s));' % name]
    lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for f, _ in s._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()]
    assert got == [ctypes.sizeof(s)] + [getattr(s, f).offset for f, _ in s._fields_]


def test_the_plain_codes():
    """Against torch's e4m3 numbers, and what rounds to even by hand."""
    import torch
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.VALUES, want, equal_nan=True)
    x = np.random.default_rng(1).standard_normal(5000) * 2.0 ** np.random.default_rng(2).integers(-14, 7, 5000)
    x = x[np.abs(x) <= 448]
    assert np.array_equal(ref.codes(x), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert ref.VALUES[ref.codes([17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10, 448.0, -0.0])].tolist() == [16.0, 20.0, 0.0, 2.0 ** -8, 448.0, 0.0]
    assert ref.is_nan(ref.codes([np.nan, np.inf, -np.inf])).all()
    assert [ref.exponent(t) for t in (0.0, 448.0, 448.1, 224.0, 2.0 ** -120)] == [-100, 0, 1, -1, -100]


def test_the_plain_append():
    """By hand: two rows behind one earlier row of a block, whose scale has to grow by 2^3."""
    rng = np.random.default_rng(3)
    b = ref.Batch(rng, [(2, 3)], 1, 64, 16, filled=False)
    page = b.table[0, 0]
    b.kc[page, 0, 0], b.ks[page, 0, 0] = ref.codes([448.0, 1.0 / 64, 1.0 / 128, 0.0] * 16), 127
    new = np.zeros((2, 1, 64))
    new[0, 0, 0], new[1, 0, 1] = 3584.0, -16.0
    _, low, high, _, _, kind = ref.append(b, "k", new, None)
    assert low[page, 0, 0] == high[page, 0, 0] == 130 and kind[page].tolist() == [1, 2, 2] + [0] * 13
    c, s = b.kc.copy(), b.ks.copy()
    s[page, 0, 0] = 130
    c[page, 0, 0] = ref.codes([56.0, 2.0 ** -9, 0.0, 0.0] * 16)  # 2^-10 lies between 0 and 2^-9: to the even one
    c[page, 0, 1], c[page, 0, 2] = ref.codes(new[0, 0] / 8), ref.codes(new[1, 0] / 8)
    ref.check_append(b, "k", c, s, new, None)
    c[page, 0, 0, 1] += 1
    with pytest.raises(AssertionError):
        ref.check_append(b, "k", c, s, new, None)
