"""A cache of which not all buffers can be had: those that were are given back (no GPU: the buffers are counted on the host)."""
import json
import os
import subprocess

import pytest

import p0k
from test_kv_node import ADDON, NODE, ROOT


class Counting(p0k.Device):
    """a device whose n-th allocation fails"""

    def __init__(self, fails):
        self.live, self.left = {}, fails

    def buffer(self, nbytes):
        if self.left == 0:
            raise p0k.P0kError(3, "no memory")
        self.left -= 1
        b = p0k.Buffer(len(self.live) + 1, nbytes, self)
        self.live[b.ptr] = b
        return b

    def upload(self, arr, dst=None, dst_off=0):
        return self.buffer(arr.nbytes)

    def free(self, buf):
        if buf is not None and buf.ptr:
            del self.live[buf.ptr]
            buf.ptr = None


@pytest.mark.parametrize("own", [True, False])
def test_python(own):
    for n in range(6):
        d = Counting(n)
        table = None if own else p0k.Buffer(99, 64, d)
        if n < (5 if own else 4):
            with pytest.raises(p0k.P0kError):
                d.kv_cache(2, 5, 2, 4, table)
        else:
            d.kv_cache_free(d.kv_cache(2, 5, 2, 4, table))
        assert not d.live and (own or table.ptr == 99)


@pytest.mark.skipif(NODE is None, reason="node is not installed")
@pytest.mark.skipif(not os.path.exists(ADDON), reason="p0k.node is not built")
def test_node():
    src = """import('%s/p0pc0rn-kernels_amd/node/index.mjs').then((m) => {
      const out = [];
      for (const table of [undefined, { given: true }]) for (let n = 0; n < 6; n++) {
        let left = n; const live = new Set();
        const buffer = () => { if (left-- === 0) throw new Error('no memory'); const b = {}; live.add(b); return b; };
        let c = null, e = '';
        try { c = m.kvCache({ buffer, upload: buffer, free: (b) => live.delete(b) }, { Hkv: 2, pages: 5, slots: 2, maxPages: 4, table }); }
        catch (x) { e = x.message; }
        out.push([!!c, e, live.size]);
      }
      console.log(JSON.stringify(out));
    })""" % ROOT
    r = subprocess.run([NODE, "-e", src], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    for i, (made, e, live) in enumerate(json.loads(r.stdout)):
        need = 5 if i < 6 else 4
        assert (made, e, live) == ((True, "", need) if i % 6 >= need else (False, "no memory", 0))
