"""Outputs that overlap other operands of the same call are refused, parts of the same rows and heads are not: the host's rule
against every value's address."""
import ctypes as C

import numpy as np
import pytest

import p0k
from test_kv_cache import D, _host, _host_batch, refused


def places(o, rows, H):
    """addresses of an operand's values, in halves"""
    rs, hs = o.get("rs") or D, o.get("hs") or (o.get("rs") or D) * rows
    r, h, d = np.arange(rows)[:, None, None], np.arange(H)[None, :, None], np.arange(D)[None, None, :]
    return set(((o["buf"].ctypes.data + o.get("off", 0)) // 2 + rs * r + hs * h + d).ravel().tolist())


def test_attention_in_place_is_refused():
    big = _host(1 << 15, np.float16)
    q = {"buf": big, "rs": 4 * D, "hs": D}
    refused("attend", "q and o overlap", q=q, o={"buf": big})
    refused("attend", "q and o overlap", q=q, o={"buf": big, "off": 8})
    refused("attend", "q and o overlap", q={"buf": big}, o={"buf": big})                       # head-major queries
    refused("attend", "q and o overlap", q={"buf": big}, o={"buf": big, "off": 6 * 4 * D * 2 - 16})
    refused("attend", q={"buf": big}, o={"buf": big, "off": 6 * 4 * D * 2})                    # behind them
    refused("attend", q={"buf": big, "off": 6 * 4 * D * 2}, o={"buf": big})                    # before them
    wide = {"buf": big, "rs": 8 * D, "hs": D}                                                  # parts of the same rows
    refused("attend", q=wide, o={"buf": big, "off": 4 * D * 2, "ld": 8 * D})
    refused("attend", q={**wide, "off": 4 * D * 2}, o={"buf": big, "ld": 8 * D})
    refused("attend", "q and o overlap", q=wide, o={"buf": big, "off": 4 * D * 2 - 16, "ld": 8 * D})
    refused("attend", q=wide, o={"buf": big, "ld": 8 * D}, batch=_host_batch(rows=0))          # no rows: nothing overlaps


def test_rope_and_read_overlap():
    big = _host(1 << 16, np.float16)
    x = {"buf": big, "rs": 4 * D, "hs": D}
    refused("rope", x=x)                                                                       # in place
    refused("rope", x=x, y=x)
    refused("rope", "x and y overlap", x=x, y={**x, "off": 16})
    refused("rope", "x and y overlap", x=x, y={**x, "off": 4 * D * 2})                         # one row on
    refused("rope", "x and y overlap", x=x, y={**x, "off": 4 * D * 2 * 5 + 3 * D * 2})         # the last head of the last row
    refused("rope", x=x, y={**x, "off": 4 * D * 2 * 6})
    refused("rope", x={**x, "rs": 8 * D}, y={**x, "rs": 8 * D, "off": 4 * D * 2})              # parts of the same rows
    refused("rope", x={**x, "rs": 8 * D, "hs": 2 * D}, y={**x, "rs": 8 * D, "hs": 2 * D, "off": D * 2})   # heads in turn
    refused("read", "k and v overlap", k={"buf": big}, v={"buf": big})
    refused("read", "k and v overlap", k={"buf": big}, v={"buf": big, "off": 2 * 6 * D * 2 - 16})
    refused("read", k={"buf": big}, v={"buf": big, "off": 2 * 6 * D * 2})
    refused("read", k={"buf": big, "hs": 12 * D}, v={"buf": big, "hs": 12 * D, "off": 6 * D * 2})         # K and V of a head in turn
    refused("read", k={"buf": big, "rs": 4 * D, "hs": D}, v={"buf": big, "rs": 4 * D, "hs": D, "off": 2 * D * 2})


def test_overlap_against_all_addresses():
    """with the same strides the rule is exact; without them it never lets an overlap through"""
    rng = np.random.default_rng(70)
    big = _host(1 << 18, np.float16)
    seen = [0, 0]
    for _ in range(4000):
        rows, H = int(rng.integers(1, 5)), 4
        st = [int(rng.choice([128, 136, 256, 512, 520, 1024, 2048])) for _ in range(2)]
        k = {"buf": big, "off": 16 * int(rng.integers(0, 300)), "rs": max(st), "hs": min(st)} if rng.random() < 0.5 else \
            {"buf": big, "off": 16 * int(rng.integers(0, 300)), "rs": min(st), "hs": max(st)}
        same = rng.random() < 0.7
        o = dict(k) if same else {**k, "rs": k["hs"], "hs": k["rs"]}
        o["off"] = k["off"] if rng.random() < 0.05 else 16 * int(rng.integers(0, 300))
        s = p0k.rope_args({"x": k, "y": o, "H": H, "batch": {"pos": _host(rows, np.int32), "rows": rows}}, p0k.numpy_resolve)
        r = p0k.lib().p0k_rope_check(C.byref(s))
        msg = p0k.lib().p0k_last_error().decode() if r else ""
        if "rows or heads overlap" in msg or "same strides" in msg:
            continue
        meet = bool(places(k, rows, H) & places(o, rows, H)) and not (k["off"] == o["off"])
        assert r == 0 or "x and y overlap" in msg, msg
        if same:
            assert bool(r) == meet, (k, o, rows)
        else:
            assert r or not meet, (k, o, rows)
        seen[meet] += 1
    assert min(seen) > 200
