"""What the serving operators' host code has to hold beyond test_serve_ops.py, on the CPU."""
import ctypes
import math
import os
import re
import subprocess

import numpy as np
import pytest

import mtg
import paged_routes
from test_cpp_interfaces import BIN, _run
from test_serve_ops import BASE, _attn, _logits, _rope


def _refused(call, description, word):
    assert call(ctypes.byref(description), None) == mtg.ERR_INVALID
    assert word in mtg.lib().mtg_last_error(None).decode(), mtg.lib().mtg_last_error(None)


def test_marks_of_calls_have_no_half_of_zero():
    assert _run("test_call_marks", 60) == {"record": "callMarks", "failures": 0}


LISTS = dict(history=BASE + (20 << 30), hist_range=BASE + (21 << 30), penalties=BASE + (22 << 30), n_history=50,
             bias_ids=BASE + (23 << 30), bias=BASE + (24 << 30), bias_range=BASE + (25 << 30), n_bias=70,
             mask=BASE + (26 << 30), mask_stride=200, vocab=5000, stride=5000, out_stride=5000, rows=3,
             workspace=BASE + (27 << 30), workspace_bytes=96)
SIZES = dict(history=200, hist_range=24, penalties=36, bias_ids=280, bias=280, bias_range=24, mask=4 * (2 * 200 + 157),
             logits=3 * 5000 * 4, out=3 * 5000 * 4, choice=12, workspace=96)


@pytest.mark.parametrize("written,other", [(w, x) for w in ("out", "choice", "workspace") for x in SIZES if x != w])
@pytest.mark.parametrize("end", ["first", "last"])
def test_logits_arrays_that_share_a_byte_are_refused(written, other, end):
    """The written array's first bytes on the other's last ones, or its last on the other's first."""
    d = _logits(**LISTS)
    unit = 16   # the coarsest alignment asked for
    at = getattr(d, other)
    if end == "first":
        at += (SIZES[other] - 1) // unit * unit
    else:
        at -= (SIZES[written] - 1) // unit * unit
    setattr(d, written, at)
    _refused(mtg.lib().mtg_logits_step_dev, d, "overlaps")


INDEX = dict(page_table=4 * 2 * 5, kv_len=8, q_start=12)                     # of 2 sequences, 5 pages a table row
ROWS = dict(positions=16, freqs=512, q_norm=512, k_norm=512, q=4 * (3 * 4096 + 2048), k_new=4 * (3 * 4096 + 1024),
            v_new=4 * (3 * 4096 + 1024))                                     # of 4 rows
POOL = 2 * (9 * 8 * 16 * 128 + 7 * 16 * 128 + 16 * 128)                      # of 10 pages of 8 heads, f16


def _set(d, name, at):
    setattr(d.kv if hasattr(mtg.PagedKv, name) else d, name, at)


def _get(d, name):
    return getattr(d.kv if hasattr(mtg.PagedKv, name) else d, name)


@pytest.mark.parametrize("written,size", [("q_out", 4 * (4 * 2048)), ("k", POOL), ("v", POOL)])
@pytest.mark.parametrize("other", [*INDEX, *ROWS])
@pytest.mark.parametrize("end", ["first", "last"])
def test_rotary_arrays_that_share_a_byte_are_refused(written, size, other, end):
    """An array that is read, its last bytes on the first ones of q_out or of the pages, or its first on their last."""
    apart = BASE + (30 << 30)
    d = _rope(positions=apart, q_norm=apart + 4096, k_norm=apart + 8192, k_new=apart + (1 << 30), v_new=apart + (2 << 30))
    n = {**INDEX, **ROWS}[other]
    unit = 16
    _set(d, other, _get(d, written) + ((size - 1) // unit * unit if end == "first" else -((n - 1) // unit * unit)))
    _refused(mtg.lib().mtg_rope_append_dev, d, "overlaps" if written == "q_out" else "in the pages")


@pytest.mark.parametrize("written,size", [("out", 4 * 4 * 2048), ("workspace", 1 << 12)])
@pytest.mark.parametrize("other", list(INDEX))
@pytest.mark.parametrize("end", ["first", "last"])
def test_attention_arrays_that_share_a_byte_are_refused(written, size, other, end):
    d = _attn(kv=dict(table_stride=4096, page_table=BASE + (30 << 30)))
    need = mtg.lib().mtg_paged_attn_workspace(ctypes.byref(d))
    assert need
    n = dict(INDEX, page_table=4 * 2 * 4096)[other]
    size = need if written == "workspace" else size
    _set(d, other, _get(d, written) + ((size - 1) // 16 * 16 if end == "first" else -((n - 1) // 16 * 16)))
    _refused(mtg.lib().mtg_paged_attn_dev, d, "overlaps")


def test_sizes_whose_extent_passes_63_bits_are_refused():
    """2^22 rows 2^40 elements apart are 2^64 bytes of f32: an extent that wraps to a few would hide every overlap."""
    L = mtg.lib()
    many = dict(n_tokens=1 << 22)
    for wide in (dict(q_stride=1 << 40), dict(out_stride=1 << 40)):
        _refused(L.mtg_paged_attn_dev, _attn(kv=many, **wide), "2^46")
    for wide in (dict(q_stride=1 << 40), dict(q_out_stride=1 << 40), dict(k_stride=1 << 40), dict(v_stride=1 << 40)):
        _refused(L.mtg_rope_append_dev, _rope(kv=many, **wide), "2^46")
    for kv in (dict(n_pages=2 ** 31 - 1, page_stride=1 << 40), dict(n_pages=2 ** 23 + 2, page_stride=1 << 40),
               dict(n_kv_heads=1024, head_stride=1 << 40, n_pages=1, n_heads=1024)):
        heads = dict(n_heads=kv.pop("n_heads")) if "n_heads" in kv else {}
        _refused(L.mtg_paged_attn_dev, _attn(kv=kv, **heads), "stride")
        _refused(L.mtg_rope_append_dev, _rope(kv=kv, **heads), "stride")


@pytest.mark.parametrize("scale", [2.5e38, -3.4e38])
def test_a_scale_that_is_infinite_as_a_power_of_two_is_refused(scale):
    """The kernels take scale * log2(e): beyond 2.36e38 that is infinite, and a score of 0 would become NaN."""
    d = _attn(scale=scale)
    _refused(mtg.lib().mtg_paged_attn_dev, d, "scale")
    assert mtg.lib().mtg_paged_attn_workspace(ctypes.byref(_attn(kv=dict(table_stride=4096), scale=scale))) == 0


@pytest.mark.parametrize("rot,base", [(2, 1e4), (64, 1e4), (128, 1e6), (6, 1.5)])
@pytest.mark.parametrize("orig_ctx,fast,slow", [(4.0, 32.0, 1.0), (4096.0, 2000.0, 700.0), (6.0, 0.99, 0.96), (4096.0, 32.0, 1.0),
                                                (1e9, 32.0, 1.0), (1e-3, 32.0, 1.0)])
def test_yarn_divides_all_pairs_that_turn_too_seldom(rot, base, orig_ctx, fast, slow):
    """Pairs of more than beta_fast turns (and a whole index further) as PLAIN, of fewer than beta_slow as LINEAR, the
    first pair among them."""
    f, _ = mtg.rope_freqs(rot, base)
    g, _ = mtg.rope_freqs(rot, base, mtg.ROPE_YARN, factor=8.0, orig_ctx=orig_ctx, beta_fast=fast, beta_slow=slow)
    turns = f * orig_ctx / (2 * math.pi)
    step = base ** (2.0 / rot)   # the turns of neighbouring pairs
    few, many = turns * step < slow, turns / step > fast
    assert np.allclose(g[few], f[few] / 8, rtol=1e-14)
    assert np.array_equal(g[many], f[many])
    assert ((g <= f * (1 + 1e-14)) & (g >= f / 8 * (1 - 1e-14))).all()


def _routes(calls):
    """The route of each call, in the words of paged_routes.py."""
    exe = os.path.join(BIN, "test_serve_calls")
    lines = "".join(" ".join(map(str, c)) + "\n" for c in calls)
    p = subprocess.run([exe], input=lines, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=60)
    assert p.returncode == 0, p.stderr
    out = []
    for line in p.stdout.splitlines()[:-1]:
        size, kernel, *join = line.split()
        kind, args = re.search(r"k_paged_(rows|chunk)I(.*)EEv", kernel).groups()
        if kind == "rows":
            _, tiles, _, waves = map(int, re.findall(r"Li(\d+)E", args + "E"))
            kind = "rows%d%s" % (16 * tiles, "x8" if waves == 8 else "")
        how = "join" + re.search(r"k_paged_joinI.*Li(\d+)EEEv", join[0]).group(1) if join else "marks" if int(size) else "alone"
        out.append(kind + " " + how)
    return out


@pytest.mark.parametrize("case", paged_routes.CASES, ids=lambda c: c[0])
def test_attention_calls_take_the_route_that_their_gpu_test_is_for(case):
    kinds = [(io, kv, dim) for io, kv in (("f32", "f16"), ("f16", "f16"), ("f32", "f32")) for dim in (64, 128)]
    assert _routes([paged_routes.call(case, *k) for k in kinds]) == [paged_routes.route(case, kv) for _, kv, _ in kinds]


def test_routes_are_all_there():
    """Each kernel with each way to join that it has."""
    routes = {paged_routes.route(c, kv) for c in paged_routes.CASES for kv in ("f16", "f32")}
    joins = ("alone", "join1", "join4", "join16")
    assert routes == {k + " " + j for k in ("rows16", "rows32") for j in (*joins, "marks")} | {"chunk " + j for j in joins} | {"rows16x8 alone"}


def test_calls_that_stay_allowed():
    """Arrays side by side, in place, slices of one product, and arrays that are not read wherever they are."""
    assert _run("test_serve_calls", 60) == {"record": "serveCalls", "failures": 0}


def test_the_search_of_a_row_s_sequence():
    assert _run("test_seq_search", 60) == {"record": "seqSearch", "failures": 0}
