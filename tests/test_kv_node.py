"""Rotary positions and the 8-bit key / value cache through the Node shim (p0pc0rn-kernels_amd/node/index.mjs), against the
definitions and with the tolerances of test_kv_cache.py."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from test_kv_cache import D, Ref, attend_ref, rope_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")
ADDON = os.path.join(ROOT, "p0pc0rn-kernels_amd", "node", "p0k.node")
pytestmark = [pytest.mark.skipif(NODE is None, reason="node is not installed"),
              pytest.mark.skipif(not os.path.exists(ADDON), reason="p0k.node is not built")]


def test_exports():
    src = ("import('%s/p0pc0rn-kernels_amd/node/index.mjs').then((m) => console.log(JSON.stringify("
           "['rope', 'kvCache', 'kvAppend', 'kvRead', 'kvAttention'].map((n) => typeof m[n]))))" % ROOT)
    r = subprocess.run([NODE, "-e", src], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert json.loads(r.stdout) == ["function"] * 5


@pytest.mark.gpu
def test_shim_cache(tmp_path):
    rng = np.random.default_rng(40)
    n, Hq, Hkv, rd = 150, 4, 2, 32
    x = rng.standard_normal((Hq + 2 * Hkv, n, D)).astype(np.float16)
    freqs = 1.0 / (1.0 + np.arange(rd // 2))
    x.tofile(str(tmp_path / "qkv.bin"))
    (tmp_path / "spec.json").write_text(json.dumps({"n": n, "Hq": Hq, "Hkv": Hkv, "rd": rd, "freqs": list(freqs), "maxPages": 4,
                                                    "window": 70, "sinks": 2}))
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "node", "kv.mjs"), str(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    rot = np.fromfile(str(tmp_path / "rot.bin"), np.float16).reshape(Hq + Hkv, n, D).transpose(1, 0, 2)
    want, tol = rope_ref(x[:Hq + Hkv].transpose(1, 0, 2), np.arange(n), freqs, True)
    assert np.all(np.abs(rot.astype(np.float64) - want) <= tol)
    ref = Ref(1, Hkv)
    ref.append(0, 0, rot[:, Hq:], x[Hq + Hkv:].transpose(1, 0, 2))
    wk, wv = ref.held(0)
    for name, w in (("k.bin", wk), ("v.bin", wv)):
        got = np.fromfile(str(tmp_path / name), np.uint16).reshape(Hkv, n, D).transpose(1, 0, 2)
        np.testing.assert_array_equal(got, w.view(np.uint16))
    o = np.fromfile(str(tmp_path / "o.bin"), np.float16).reshape(n, Hq, D).astype(np.float64)
    w, tol = attend_ref(rot[:, :Hq], 0, *ref.held(0, read=False), Hq // Hkv, window=70, sinks=2)
    assert np.all(np.abs(o - w) <= tol)
    e = json.loads((tmp_path / "errors.json").read_text())
    assert "sinks without" in e["sinks"] and "needs" in e["rows"] and "freqs" in e["freqs"] and "live buffer" in e["freed"]
