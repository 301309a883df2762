"""kv_attention's limits: what the header allows is taken, whatever kernel can count it."""
import ctypes as C

import numpy as np
import pytest

import p0k
from test_kv_cache import CALLS, Cache, Ref, _host_batch, _host_cache, fill


def check(Hkv, Hq, B, rows, max_pages):
    """the check's answer for sizes of which no memory is touched"""
    make, args, fn = CALLS["attend"]
    s = args(make(), p0k.numpy_resolve)
    s.cache.Hkv, s.cache.slots, s.cache.max_pages, s.cache.pages = Hkv, B, max_pages, 5
    for n in ("code", "scale", "tail", "table"):
        setattr(s.cache, n + "_size", 1 << 60)
    s.batch.B, s.batch.rows = B, rows
    s.batch.pos_size = s.batch.cu_size = s.o_size = s.q_size = 1 << 55
    s.Hq = Hq
    s.o_buf = 1 << 56                                        # (far from the queries)
    r = getattr(p0k.lib(), fn)(C.byref(s))
    assert r in (p0k.OK, p0k.E_ARG) and (r == p0k.OK or "too many for one call" in p0k.lib().p0k_last_error().decode())
    return r == p0k.OK


def test_limits():
    assert check(8, 128, 1, 131072, 2048)                    # a prompt of 131072 tokens of 128 heads over its own cache
    assert check(8, 64, 1, 1 << 17, 16384)                   # the same in a table for a million tokens
    assert check(8, 64, 8192, 8192, 16384)                   # a decode step of 8192 such sequences
    assert check(1, 1, 1, 1 << 24, 1 << 18)
    assert check(8, 32, 1 << 20, 1 << 20, 100)               # the most sequences there are
    assert not check(8, 32, 1 << 20, 1 << 20, 205)
    assert check(4, 128, 1, (1 << 24) - 16, 1 << 18)
    assert not check(8, 128, 1, 1 << 24, 1 << 18)            # 2^31 rows of heads
    # the bounds themselves: rows * Hq / 256 + B * Hkv < 2^23, (rows * Hq / 16 + B * Hkv) * max_pages < 2^31
    assert check(1, 256, 255, (1 << 23) - 256, 1 << 18) and not check(1, 256, 256, (1 << 23) - 256, 1 << 18)
    assert check(16, 16, 1 << 19, 1 << 19, 240) and not check(16, 16, 1 << 19, 1 << 19, 256)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 40])
def test_long_tables(dev, n):
    """few tokens in tables of four million blocks: the units that there could be pass 32 bits"""
    rng = np.random.default_rng(80)
    Hkv, slots, mp = 64, 8, 1 << 22
    lens = [n + x for x in (0, 1, 63, 64, 100, 150, 200, 7)]
    c = Cache.__new__(Cache)
    c.dev, c.Hkv, c.slots, c.mp, c.bufs, c.ref = dev, Hkv, slots, mp, [], Ref(slots, Hkv)
    table = np.full((slots, mp), -1, np.int32)
    table[:, :4] = rng.permutation(slots * 4).reshape(slots, 4)
    c.tb = dev.upload(table)
    c.c = dev.kv_cache(Hkv, slots * 4, slots, mp, c.tb)
    try:
        fill(c, lens, rng)
        c.attend([(s, x - n, n) for s, x in enumerate(lens)], Hkv, rng)
        c.attend([(s, x - n, n) for s, x in enumerate(lens)], 2 * Hkv, rng, window=70, sinks=3, cap=20.0)
    finally:
        c.free()
        dev.drain_pool()
