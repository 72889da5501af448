"""mtg_sample_dev on the CPU: what it refuses before any GPU work, its workspace, its struct, and the plain form by hand."""
import ctypes
import shutil
import subprocess

import numpy as np
import pytest

import mtg
from sample_ref import answers
from test_serve_ops import BASE, ROOT

AT = dict(logits=BASE, settings=BASE + (1 << 30), top_k=BASE + (2 << 30), uniform=BASE + (3 << 30), choice=BASE + (4 << 30),
          prob=BASE + (5 << 30), workspace=BASE + (6 << 30))


def _sample(**kw):
    f = dict(AT, stride=1000, io_type=mtg.TYPE_F32, rows=3, vocab=1000, workspace_bytes=1 << 30)
    f.update(kw)
    return mtg.Sample(**f)


def _call(**kw):
    return mtg.lib().mtg_sample_dev(ctypes.byref(_sample(**kw)), None)


def _size(**kw):
    return mtg.lib().mtg_sample_workspace(ctypes.byref(_sample(**kw)))


@pytest.mark.parametrize("bad,status", [
    (dict(rows=-1), mtg.ERR_INVALID), (dict(rows=65536), mtg.ERR_INVALID), (dict(vocab=0), mtg.ERR_INVALID), (dict(vocab=-5), mtg.ERR_INVALID),
    (dict(vocab=(1 << 24) + 1), mtg.ERR_INVALID), (dict(io_type=mtg.TYPE_Q8_0), mtg.ERR_UNSUPPORTED), (dict(io_type=mtg.TYPE_F8_E4M3), mtg.ERR_UNSUPPORTED),
    (dict(logits=None), mtg.ERR_INVALID), (dict(settings=None), mtg.ERR_INVALID), (dict(uniform=None), mtg.ERR_INVALID),
    (dict(choice=None), mtg.ERR_INVALID), (dict(workspace=None), mtg.ERR_INVALID), (dict(workspace=AT["workspace"] + 8), mtg.ERR_INVALID),
    (dict(workspace_bytes=64), mtg.ERR_CAPACITY), (dict(stride=999), mtg.ERR_INVALID), (dict(stride=1 << 41), mtg.ERR_INVALID),
    (dict(stride=-1000), mtg.ERR_INVALID), (dict(logits=BASE + 2), mtg.ERR_INVALID), (dict(io_type=mtg.TYPE_F16, logits=BASE + 1), mtg.ERR_INVALID),
    (dict(settings=AT["settings"] + 2), mtg.ERR_INVALID), (dict(top_k=AT["top_k"] + 1), mtg.ERR_INVALID), (dict(uniform=AT["uniform"] + 3), mtg.ERR_INVALID),
    (dict(choice=AT["choice"] + 2), mtg.ERR_INVALID), (dict(prob=AT["prob"] + 2), mtg.ERR_INVALID)], ids=lambda x: str(x)[:40])
def test_bad_calls_are_refused(bad, status):
    assert _call(**bad) == status
    assert b"sample" in mtg.lib().mtg_last_error(None)


SIZES = dict(logits=12000, settings=36, top_k=12, uniform=12, choice=12, prob=12)


@pytest.mark.parametrize("written", ["choice", "prob", "workspace"])
@pytest.mark.parametrize("end", ["first", "last"])
def test_arrays_that_share_a_byte_are_refused(written, end):
    sizes = dict(SIZES, workspace=_size())
    unit = 16 if written == "workspace" else 4
    for other in sizes:
        if other == written:
            continue
        at = AT[other] + (sizes[other] - 1) // unit * unit if end == "first" else AT[other] - (sizes[written] - 1) // unit * unit
        assert _call(**{written: at}) == mtg.ERR_INVALID, other
        assert b"overlap" in mtg.lib().mtg_last_error(None)


def test_calls_without_rows_and_workspaces():
    assert _call(rows=0, logits=None, workspace=None) == mtg.OK and _size(rows=0) == 0
    assert mtg.lib().mtg_sample_dev(None, None) == mtg.ERR_INVALID and mtg.lib().mtg_sample_workspace(None) == 0
    assert _size(vocab=0) == _size(rows=65536) == _size(rows=-1) == 0
    for rows in (1, 7, 61, 256, 5000):
        for vocab in (1, 257, 4097, 50257, 151936, 1 << 20):
            n = _size(rows=rows, vocab=vocab, logits=None, choice=None)
            # the units' maxima and a histogram for each workgroup, of which a row has one per 32,768 ids or more
            assert n % 16 == 0 and n >= rows * (-(-vocab // 256) * 4 + -(-vocab // 32768) * 8192)
            assert n <= rows * (-(-vocab // 256) * 4 + 4096 + (vocab // 4096 + 1) * 8300) + 4096


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layout(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "%s/include/mtg_verify.h"' % ROOT, "int main(void){", 'printf("%zu\\n", sizeof(mtg_sample));']
    lines += ['printf("%%zu\\n", offsetof(mtg_sample, %s));' % f for f, _ in mtg.Sample._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-o", str(exe), str(src)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()]
    assert got == [ctypes.sizeof(mtg.Sample)] + [getattr(mtg.Sample, f).offset for f, _ in mtg.Sample._fields_]


def test_the_plain_form():
    x = np.log([0.1, 0.4, 0.2, 0.25, 0.05])  # in order: ids 1, 3, 2, 0, 4
    none = dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)

    def one(u, **kw):
        (i, p), = answers(x, uniform=u, **{**none, **kw}).items()
        return i, round(p[0], 6)
    assert [one(u)[0] for u in (0.0, 0.39, 0.41, 0.64, 0.66, 0.84, 0.86, 0.94, 0.96, 2.0, float("nan"))] == [1, 1, 3, 3, 2, 2, 0, 0, 4, 4, 1]
    assert one(0.7, top_k=2) == (3, round(0.25 / 0.65, 6)) and one(0.5, top_k=1) == (1, 1.0)
    assert one(0.9, top_p=0.7) == (2, round(0.2 / 0.85, 6)) and one(0.9, top_p=0.01) == (1, 1.0) and one(0.9, top_p=-1) == (1, 1.0)
    assert one(0.99, min_p=0.3) == (2, round(0.25, 2) and round(0.2 / 0.85, 6)) and one(0.9, min_p=2.0) == (1, 1.0)
    assert one(0.9, temperature=0.0) == (1, 1.0) and one(0.99, top_k=3, top_p=0.6) == (3, round(0.25 / 0.65, 6))
    assert one(0.2, temperature=0.5) == (1, round(0.16 / (0.16 + 0.0625 + 0.04 + 0.01 + 0.0025), 6))
    assert answers([np.nan, -np.inf], 1.0, 1.0, 0.0, 0, 0.5) == {-1: [0.0]}
    assert answers([1.0, np.inf, 3.0, np.inf], 1.0, 1.0, 0.0, 0, 0.75) == {3: [0.5]}
    assert answers([2.0, 2.0, 2.0], 1.0, 1.0, 0.0, 2, 0.6) == {1: [0.5]}
