"""Offsets that decrease, on the attention's kernel for many queries: rows that no workgroup takes stay as they are."""
import numpy as np
import pytest

from test_kv_cache import D, cache, fill  # noqa: F401


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[800, 0, 400, 800], [0, 800, 0, 800], [0, 500, 300, 800], [300, 800, 0, 800]], ids=str)
def test_decreasing_offsets_leave_rows(cache, cu):  # noqa: F811
    """keys in several runs, whose partial results meet in the workspace: with offsets that decrease there is nothing to join,
    and the results of an earlier call, which lie there, are not written"""
    rng = np.random.default_rng(60)
    Hkv, Hq, n = 2, 16, 800
    c = cache(Hkv, 3, 40)
    fill(c, [1100, 1000, 1100], rng)
    assert n * Hq // Hkv > 256 * 3 and n * Hq > 20 * c.dev.cus()       # (the kernel over blocks of rows)
    c.attend([(0, 800, 300), (1, 800, 200), (2, 800, 300)], Hq, rng)   # leaves its parts in the workspace
    b = {"pos": c.up(np.full(3, 800, np.int32)), "cu": c.up(np.array(cu, np.int32)), "B": 3, "rows": n}
    q = c.up(rng.standard_normal((Hq, n, D)).astype(np.float16))
    o = c.up(np.full((n, Hq * D), 0x1234, np.uint16))
    for _ in range(2):
        c.dev.kv_attention({"cache": c.c, "batch": b, "q": q, "o": o, "Hq": Hq})
    assert np.all(c.dev.read(o, np.uint16) == 0x1234)
