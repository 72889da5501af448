"""The routes that the operators over a cache in 8 bits take, on the fake HIP runtime: tests/cpp/test_serve_f8_calls.cpp."""
import os
import re
import subprocess

import pytest

import paged_f8_routes
from test_cpp_interfaces import BIN, _run


def routes(calls):
    """The route of each call, in the words of paged_f8_routes.py, and the dynamic LDS of its first kernel."""
    lines = "".join(" ".join(map(str, c)) + "\n" for c in calls)
    p = subprocess.run([os.path.join(BIN, "test_serve_f8_calls")], input=lines, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True,
                       timeout=60)
    assert p.returncode == 0, p.stderr
    out = []
    for line in p.stdout.splitlines()[:-1]:
        size, kernel, lds, *join = line.split()
        kind, args = re.search(r"k_paged_(rows|chunk)_f8I(.*)EEv", kernel).groups()
        numbers = list(map(int, re.findall(r"Li(\d+)E", args + "E")))
        if kind == "rows":
            _, tiles, waves = numbers
            kind = "rows%d%s" % (16 * tiles, "x8" if waves == 8 else "")
        else:
            kind = {4: "chunk", 8: "wide"}[numbers[1]]
        how = "join" + re.search(r"k_paged_join_sinkI.*Li(\d+)EEEv", join[0]).group(1) if join else "marks" if int(size) else "alone"
        out.append((kind + " " + how, int(lds)))
    return out


@pytest.mark.parametrize("case", paged_f8_routes.CASES, ids=lambda c: c[0])
def test_attention_calls_take_the_route_that_their_gpu_test_is_for(case):
    got = routes([paged_f8_routes.call(case, io, dim) for io in ("f32", "f16") for dim in (64, 128)])
    assert [r for r, _ in got] == [case[-1]] * 4
    for r, lds in got:  # workgroups kept apart: by LDS that is never used, all of it under what a launch may have
        assert lds in ((0, 21 << 10, 37 << 10) if r.startswith("rows16 ") else (0,))


def test_routes_are_all_there():
    taken = {c[-1] for c in paged_f8_routes.CASES}
    joins = ("alone", "join1", "join4", "join16")
    assert taken == {k + " " + j for k in ("rows16", "rows32") for j in (*joins, "marks")} | {k + " " + j for k in ("chunk", "wide") for j in joins} | {"rows16x8 alone"}


def test_calls_and_their_launches():
    assert _run("test_serve_f8_calls", 60) == {"record": "serveF8Calls", "failures": 0}
