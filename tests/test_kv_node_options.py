"""The Node shim's rope refuses options that it does not know, as the Python binding does, before anything reaches the library."""
import json
import os
import subprocess

import numpy as np
import pytest

import p0k
from test_kv_node import ADDON, NODE, ROOT

pytestmark = [pytest.mark.skipif(NODE is None, reason="node is not installed"),
              pytest.mark.skipif(not os.path.exists(ADDON), reason="p0k.node is not built")]

CASES = [({"mode": "neox"}, "rope: unknown mode neox"), ({"mode": "Half"}, "rope: unknown mode Half"),
         ({"mode": "toString"}, "rope: unknown mode toString"),
         ({"scaling": {"kind": "yarn", "factor": 8}}, "rope: unknown scaling kind yarn"),
         ({"scaling": {"factor": 8}}, "rope: unknown scaling kind undefined"),
         ({"mode": "half", "scaling": {"kind": "bands"}}, "NULL context"), ({"mode": "interleaved", "scaling": {"kind": "plain"}}, "NULL context"),
         ({"scaling": {"kind": "linear"}}, "NULL context"), ({}, "NULL context")]


def test_rope_options():
    src = ("import('%s/p0pc0rn-kernels_amd/node/index.mjs').then((m) => console.log(JSON.stringify(%s.map((o) => {"
           "try { m.rope({ ctx: null }, { x: { buf: { ptr: 16n, size: 4096 } }, H: 1, batch: { pos: { ptr: 16n, size: 16 }, rows: 1 }, ...o }); return null; }"
           " catch (e) { return e.message; } }))))" % (ROOT, json.dumps([o for o, _ in CASES])))
    r = subprocess.run([NODE, "-e", src], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    for (o, want), got in zip(CASES, json.loads(r.stdout)):
        assert got and want in got, (o, got)


@pytest.mark.parametrize("o", [o for o, m in CASES if "unknown" in m], ids=str)
def test_rope_options_of_the_python_binding(o):
    x = np.zeros(128, np.float16)
    with pytest.raises(KeyError):
        p0k.rope_args({"x": x, "H": 1, "batch": {"pos": np.zeros(1, np.int32), "rows": 1}, **o}, p0k.numpy_resolve)


NEEDED = [("rope", {"H": None}, "rope: H is"), ("rope", {"batch": {"rows": None}}, "batch: rows is"), ("rope", {"batch": {"B": None}}, "batch: B is"),
          ("kvAppend", {"batch": {"rows": None}}, "batch: rows is"), ("kvRead", {"batch": {"B": None}}, "batch: B is"),
          ("kvAttention", {"batch": {"rows": "many"}}, "batch: rows is many"), ("kvAttention", {}, "NULL context")]


def test_numbers_that_are_left_out():
    """rows, sequences and heads that are not given are not taken as none"""
    src = ("import('%s/p0pc0rn-kernels_amd/node/index.mjs').then((m) => console.log(JSON.stringify(%s.map(([f, o]) => {"
           "const u = (x) => Object.fromEntries(Object.entries(x).map(([k, v]) => [k, v === null ? undefined : v]));"
           "const b = { ptr: 16n, size: 4096 }, batch = { pos: b, cu: b, B: 1, rows: 1, ...u(o.batch || {}) };"
           "try { m[f]({ ctx: null }, { cache: {}, x: b, k: b, v: b, q: b, o: b, len: b, Hq: 1, H: 1, ...u(o), batch }); return null; }"
           " catch (e) { return e.message; } }))))" % (ROOT, json.dumps([c[:2] for c in NEEDED])))
    r = subprocess.run([NODE, "-e", src], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    for c, got in zip(NEEDED, json.loads(r.stdout)):
        assert got and c[2] in got, (c, got)


def test_numbers_that_are_left_out_of_the_python_binding():
    x, i = np.zeros(128, np.float16), np.zeros(2, np.int32)
    for a in ({"H": 1, "batch": {"pos": i, "cu": i, "rows": 1}}, {"H": 1, "batch": {"pos": i, "cu": i, "B": 1}}, {"batch": {"pos": i, "rows": 1}}):
        with pytest.raises(KeyError):
            p0k.rope_args({"x": x, **a}, p0k.numpy_resolve)
