"""Rotary positions (p0k_rope) and the 8-bit key / value cache (p0k_kv_append, p0k_kv_read, p0k_kv_attention).

CPU: the refusals, the struct layouts and the buffers' sizes. GPU: each call against its definition in 64 bits (numpy).

Tolerances. Read-back is exact: every value is f16(fp32(code * scale)), and the codes are those of the exact quotient.
rope: |y| is rounded once (2^-11 |y|, 2^-25 below the normal range); sine, cosine, products and sum are fp32 with a few units
of 2^-24 each of |x1| + |x2|: 2^-20 (|x1| + |x2|) covers them.
attention: with A = sum p |v| / sum p of a row and head, the result is rounded once (2^-11 |o|), the probabilities once before
the products (2^-11 A, and 2^-25 of the largest each, times max |v|, where they fall below f16's normal range: their sum is
at least 1), a score is off by at most 2^-24 x 130 x sum |q k| scale (fp32 sums of 128 exact products and two roundings),
which changes a probability by that factor, twice (numerator and sum), and fp32 sums over n keys add n 2^-24 A."""
import ctypes as C

import numpy as np
import pytest

import p0k

T, D = 64, 128


# ------------------------------------------------------------------------------------------------ the definition
def finite16(x):
    x = np.asarray(x, np.float16)
    return np.where(np.isnan(x), np.float16(0), np.clip(x, np.float16(-65504), np.float16(65504))).astype(np.float16)


def quantised(x):
    """a whole block [64][head][128] f16 -> (codes * scale in 64 bits, what is read back in f16)"""
    x = finite16(x).astype(np.float64)
    a = np.abs(x).max((0, 2), keepdims=True).astype(np.float32)
    s = np.where(a > 0, a / np.float32(127), np.float32(1)).astype(np.float32)
    c = np.rint(x / s.astype(np.float64)) + 0.0          # (an integer code has no negative zero)
    return c * s.astype(np.float64), (c.astype(np.float32) * s).astype(np.float16)


class Ref:
    """what a cache holds: the tokens of each slot, f16 [token][head][128]"""

    def __init__(self, slots, Hkv):
        self.k = [np.zeros((0, Hkv, D), np.float16) for _ in range(slots)]
        self.v = [np.zeros((0, Hkv, D), np.float16) for _ in range(slots)]

    def append(self, slot, pos, k, v):
        assert pos <= len(self.k[slot])
        self.k[slot] = np.concatenate([self.k[slot][:pos], finite16(k)])
        self.v[slot] = np.concatenate([self.v[slot][:pos], finite16(v)])

    def values(self, x, read):
        full = len(x) // T
        out = [quantised(x[b * T:(b + 1) * T])[1 if read else 0] for b in range(full)]
        return np.concatenate(out + [x[full * T:]]) if out else x

    def held(self, slot, read=True):
        k, v = self.values(self.k[slot], read), self.values(self.v[slot], read)
        return (k, v) if read else (k.astype(np.float64), v.astype(np.float64))


def attend_ref(q, pos, k, v, rep, window=0, sinks=0, cap=0.0, scale=None, gone=()):
    """q [row][Hq][128], k / v [token][Hkv][128] in 64 bits; gone: blocks that are not there -> (o, tolerance)"""
    n, Hq, L = q.shape[0], q.shape[1], len(k)
    q = q.astype(np.float64)
    sc = np.float64(np.float32(0.08838834764831845)) if scale is None else scale
    o, tol = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    j, t = np.arange(L)[None, :], (pos + np.arange(n))[:, None]
    see = j <= t
    if window:
        see &= (j > t - window) | (j < sinks)
    for b in gone:
        see &= j // T != b
    for h in range(Hq):
        kk, vv = k[:, h // rep], v[:, h // rep]
        s = q[:, h] @ kk.T * sc
        mag = (np.abs(q[:, h]) @ np.abs(kk).T * sc) if L else s
        if cap:
            s = cap * np.tanh(s / cap)
        s = np.where(see, s, -np.inf)
        m = s.max(1, keepdims=True, initial=-np.inf)
        p = np.where(see, np.exp(s - np.where(np.isfinite(m), m, 0)), 0)
        l = p.sum(1, keepdims=True)
        some = l > 0
        l = np.where(some, l, 1)
        o[:, h] = p @ vv / l
        A = p @ np.abs(vv) / l
        ds = 130 * 2.0 ** -24 * np.where(see, mag, 0).max(1, keepdims=True, initial=0)
        if cap:
            ds = ds + 2.0 ** -20 * cap                      # tanh on the hardware's exp2 and reciprocal
        vmax = np.where(see[..., None], np.abs(vv)[None], 0).max((1, 2), initial=0)[:, None]
        nv = see.sum(1, keepdims=True)
        tol[:, h] = 2.0 ** -11 * np.abs(o[:, h]) + 2.0 ** -25 + A * (2.0 ** -11 + 2 * ds + nv * 2.0 ** -24) + nv * 2.0 ** -25 * vmax
    return o, tol


# ------------------------------------------------------------------------------------------------ on the device
class Cache:
    """a cache on the device with scrambled pages, beside what it should hold"""

    def __init__(self, dev, Hkv, slots, max_pages, extra=3, seed=0, bad=()):
        rng = np.random.default_rng(seed)
        self.dev, self.Hkv, self.slots, self.mp, self.bufs = dev, Hkv, slots, max_pages, []
        pages = slots * max_pages + extra
        self.table = rng.permutation(pages)[:slots * max_pages].astype(np.int32).reshape(slots, max_pages)
        for s, b, page in bad:
            self.table[s, b] = page
        self.tb = dev.upload(self.table)
        self.c = dev.kv_cache(Hkv, pages, slots, max_pages, self.tb)
        # what no call has written must not matter: NaN everywhere
        for n in ("code", "scale", "tail"):
            dev.upload(np.full(self.c[n].size // 4, 0x7fc07e01, np.uint32), self.c[n])
        self.ref = Ref(slots, Hkv)

    def up(self, x):
        b = self.dev.upload(np.ascontiguousarray(x))
        self.bufs.append(b)
        return b

    def rows(self, x, token, pad=0):
        """[row][head][128] -> operand, head-major or token-major, with `pad` unused halves behind each row"""
        n, h = x.shape[:2]
        if token:
            w = np.full((n, h * D + pad), np.nan, x.dtype)
            w[:, :h * D] = x.reshape(n, -1)
            return {"buf": self.up(w), "rs": h * D + pad, "hs": D}
        w = np.full((h, n + 1, D + pad), np.nan, x.dtype)
        w[:, :n, :D] = x.transpose(1, 0, 2)
        return {"buf": self.up(w), "rs": D + pad, "hs": (n + 1) * (D + pad)}

    def batch(self, pos, n, slot=None, lead=0, tail=0):
        cu = np.concatenate([[lead], lead + np.cumsum(n)]).astype(np.int32)
        b = {"pos": self.up(np.array(pos, np.int32)), "cu": self.up(cu), "B": len(n), "rows": int(cu[-1]) + tail}
        if slot is not None:
            b["slot"] = self.up(np.array(slot, np.int32))
        return b, cu

    def append(self, seqs, rng, token=False, pad=0, lead=0, tail=0, make=None, skip=()):
        """seqs: (slot, pos, n)"""
        b, cu = self.batch([p for _, p, _ in seqs], [n for _, _, n in seqs], [s for s, _, _ in seqs], lead, tail)
        make = make or (lambda *s: (rng.standard_normal(s) * np.exp(rng.standard_normal((s[0], 1, 1)))).astype(np.float16))
        k, v = make(b["rows"], self.Hkv, D), make(b["rows"], self.Hkv, D)
        self.dev.kv_append({"cache": self.c, "batch": b, "k": self.rows(k, token, pad), "v": self.rows(v, token, pad)})
        for i, (s, p, n) in enumerate(seqs):
            if i not in skip:
                self.ref.append(s, p, k[cu[i]:cu[i + 1]], v[cu[i]:cu[i + 1]])

    def read(self, seqs, token=False, lead=0, tail=0, lens=None):
        """seqs: (slot, pos, n) -> K, V [row][head][128] as bits (rows outside the batch: 0x1234)"""
        b, cu = self.batch([p for _, p, _ in seqs], [n for _, _, n in seqs], [s for s, _, _ in seqs], lead, tail)
        held = self.up(np.array([len(self.ref.k[s]) for s, _, _ in seqs] if lens is None else lens, np.int32))
        R, H = b["rows"], self.Hkv
        out = [self.up(np.full(R * H * D + 64, 0x1234, np.uint16)) for _ in range(2)]
        st = {"rs": H * D, "hs": D} if token else {"rs": D, "hs": R * D}
        self.dev.kv_read({"cache": self.c, "batch": b, "len": held, "k": {"buf": out[0], "off": 32, **st}, "v": {"buf": out[1], "off": 32, **st}})
        got = []
        for o in out:
            x = self.dev.read(o, np.uint16, R * H * D + 64)
            assert np.all(x[:16] == 0x1234) and np.all(x[16 + R * H * D:] == 0x1234)
            x = x[16:16 + R * H * D]
            got.append(x.reshape(R, H, D) if token else x.reshape(H, R, D).transpose(1, 0, 2))
        return got[0], got[1], cu

    def check_all(self, token=False):
        """every slot's tokens against the reference, bit for bit"""
        seqs = [(s, 0, len(self.ref.k[s])) for s in range(self.slots)]
        k, v, cu = self.read(seqs, token)
        for i, (s, _, n) in enumerate(seqs):
            wk, wv = self.ref.held(s)
            np.testing.assert_array_equal(k[cu[i]:cu[i + 1]], wk.view(np.uint16))
            np.testing.assert_array_equal(v[cu[i]:cu[i + 1]], wv.view(np.uint16))

    def attend(self, seqs, Hq, rng, token=False, pad=0, lead=0, tail=0, ldo=0, gone=(), qscale=1.0, nokeys=(), **kw):
        """queries (slot, pos, n), whose tokens the cache holds, against the definition"""
        b, cu = self.batch([p for _, p, _ in seqs], [n for _, _, n in seqs], [s for s, _, _ in seqs], lead, tail)
        q = (rng.standard_normal((b["rows"], Hq, D)) * qscale).astype(np.float16)
        ld = ldo or Hq * D
        o = self.up(np.full(b["rows"] * ld + 8, 0x1234, np.uint16))
        self.dev.kv_attention({"cache": self.c, "batch": b, "q": self.rows(q, token, pad), "o": {"buf": o, "off": 8, "ld": ldo},
                               "Hq": Hq, **kw})
        got = self.dev.read(o, np.uint16, b["rows"] * ld + 8)
        assert np.all(got[:4] == 0x1234)
        got = got[4:4 + b["rows"] * ld].reshape(b["rows"], ld)
        assert np.all(got[:cu[0]] == 0x1234) and np.all(got[cu[-1]:] == 0x1234) and np.all(got[:, Hq * D:] == 0x1234)
        got = got[:, :Hq * D].copy().view(np.float16).astype(np.float64)
        for i, (s, p, n) in enumerate(seqs):
            g = got[cu[i]:cu[i + 1]].reshape(n, Hq, D)
            if i in nokeys:
                assert np.all(g == 0)
                continue
            k, v = self.ref.held(s, read=False)
            w, tol = attend_ref(q[cu[i]:cu[i + 1]], p, k[:p + n], v[:p + n], Hq // self.Hkv, gone=[g_[1] for g_ in gone if g_[0] == s], **kw)
            err = np.abs(g - w)
            assert np.all(np.isfinite(g)), f"sequence {i} {(s, p, n)}"
            worst = np.unravel_index(np.argmax(err / np.maximum(tol, 1e-30)), err.shape)
            assert np.all(err <= tol), f"sequence {i} {(s, p, n)}: {err[worst]} > {tol[worst]} at {worst}"
        return got

    def free(self):
        self.dev.done()
        for b in self.bufs + [self.tb]:
            self.dev.free(b)
        self.dev.kv_cache_free(self.c)


@pytest.fixture
def cache(dev):
    made = []

    def make(*a, **k):
        made.append(Cache(dev, *a, **k))
        return made[-1]
    yield make
    for c in made:
        c.free()


# ------------------------------------------------------------------------------------------------ CPU: refusals
def _host(n, dtype=np.uint8):
    return np.zeros(n, dtype)


def _host_cache(**kw):
    L, c = p0k.lib(), {"pages": 5, "slots": 2, "max_pages": 4, "Hkv": 2, **kw}
    c.setdefault("code", _host(L.p0k_kv_code_bytes(5, 2)))
    c.setdefault("scale", _host(L.p0k_kv_scale_bytes(5, 2)))
    c.setdefault("tail", _host(L.p0k_kv_tail_bytes(2, 2)))
    c.setdefault("table", _host(2 * 4, np.int32))
    return c


def _host_batch(**kw):
    return {"pos": _host(2, np.int32), "cu": _host(3, np.int32), "B": 2, "rows": 6, **kw}


def _row_op(heads=2, rows=6):
    return {"buf": _host(heads * rows * D, np.float16)}


CALLS = {
    "append": (lambda **kw: {"cache": _host_cache(), "batch": _host_batch(), "k": _row_op(), "v": _row_op(), **kw},
               p0k.kv_append_args, "p0k_kv_append_check"),
    "read": (lambda **kw: {"cache": _host_cache(), "batch": _host_batch(), "len": _host(2, np.int32), "k": _row_op(), "v": _row_op(), **kw},
             p0k.kv_read_args, "p0k_kv_read_check"),
    "attend": (lambda **kw: {"cache": _host_cache(), "batch": _host_batch(), "q": _row_op(4), "o": {"buf": _host(6 * 4 * D, np.float16)}, "Hq": 4, **kw},
               p0k.kv_attention_args, "p0k_kv_attention_check"),
    "rope": (lambda **kw: {"x": _row_op(4), "batch": _host_batch(), "H": 4, **kw}, p0k.rope_args, "p0k_rope_check"),
}


def refused(call, pattern=None, **kw):
    make, args, check = CALLS[call]
    s = args(make(**kw), p0k.numpy_resolve)
    r = getattr(p0k.lib(), check)(C.byref(s))
    msg = p0k.lib().p0k_last_error().decode()
    if pattern is None:
        assert r == p0k.OK, msg
    else:
        assert r == p0k.E_ARG and pattern in msg, (r, msg)


@pytest.mark.parametrize("call", list(CALLS))
def test_valid_and_struct(call):
    refused(call)
    make, args, check = CALLS[call]
    s = args(make(), p0k.numpy_resolve)
    s.struct_size = 7
    assert getattr(p0k.lib(), check)(C.byref(s)) == p0k.E_ARG
    assert f"expects {C.sizeof(type(s))}" in p0k.lib().p0k_last_error().decode()
    assert getattr(p0k.lib(), check)(None) == p0k.E_ARG


@pytest.mark.parametrize("call", ["append", "read", "attend"])
def test_cache_refusals(call):
    for n, size in (("code", 5 * 2 * 2 * 8192), ("scale", 5 * 2 * 8), ("tail", 2 * 2 * 8 * 8192), ("table", 32)):
        refused(call, f"{n} needs", cache=_host_cache(**{n: _host(size - 4)}))
        refused(call, cache=_host_cache(**{n: _host(size)}))
    refused(call, "scale needs", cache=_host_cache(scale={"buf": _host(80), "off": 8}))
    refused(call, "16-byte aligned", cache=_host_cache(tail={"buf": _host(300000), "off": 8}))
    refused(call, "multiple of 4", cache=_host_cache(table={"buf": _host(80), "off": 2}))
    for n in ("pages", "slots", "max_pages", "Hkv"):
        refused(call, "must be positive", cache=_host_cache(**{n: 0}))
    refused(call, "3 sequences on a cache of 2", batch=_host_batch(B=3, pos=_host(3, np.int32), cu=_host(4, np.int32)))
    refused(call, "cu needs", batch=_host_batch(cu=_host(2, np.int32)))
    refused(call, "pos needs", batch=_host_batch(pos=_host(1, np.int32)))
    refused(call, "slot needs", batch=_host_batch(slot=_host(1, np.int32)))
    refused(call, "too many", batch=_host_batch(rows=(1 << 24) + 1))
    b = _host_batch(B=0)
    refused(call, batch=b)                                   # no sequences: nothing to do


@pytest.mark.parametrize("call,names", [("append", "kv"), ("read", "kv"), ("attend", "q"), ("rope", "x")])
def test_row_refusals(call, names):
    heads = {"attend": 4, "rope": 4}.get(call, 2)
    for n in names:
        refused(call, f"{n} needs", **{n: _row_op(heads, 5)})
        refused(call, "16-byte aligned", **{n: {**_row_op(heads, 8), "off": 8}})
        refused(call, "multiples of 8", **{n: {**_row_op(heads, 8), "rs": 132}})
        refused(call, "stride too large", **{n: {**_row_op(heads, 8), "rs": 1 << 40}})
        refused(call, "needs", **{n: {**_row_op(heads, 8), "hs": (1 << 32) - 8}})
    if call in ("read", "rope"):
        n = "k" if call == "read" else "y"
        big = {"buf": _host(1 << 16, np.float16)}
        refused(call, "overlap", **{n: {**big, "rs": 64, "hs": 2048}})
        refused(call, "overlap", **{n: {**big, "rs": 128, "hs": 640}})
        refused(call, **{n: {**big, "rs": 128 * heads, "hs": 128}})


def test_attention_and_rope_refusals():
    refused("attend", "multiple of Hkv", Hq=3, q=_row_op(3))
    refused("attend", "sinks without", sinks=4)
    refused("attend", "scale", scale=-1.0)
    refused("attend", "cap", cap=float("nan"))
    refused("attend", "cap", cap=1e-30)
    refused("attend", "scale", scale=1e-20)
    refused("attend", "scale", scale=float("inf"))
    refused("attend", "o needs", o={"buf": _host(6 * 4 * D - 1, np.float16)})
    refused("attend", "covering", o={"buf": _host(6 * 4 * D, np.float16), "ld": 508})
    refused("rope", "even and at most", rd=130)
    refused("rope", "even and at most", rd=7)
    refused("rope", "theta", theta=-1.0)
    refused("rope", "factor", scaling={"kind": "linear"})
    refused("rope", "bands need", scaling={"kind": "bands", "factor": 2.0, "orig": 100.0, "low": 1.0, "high": 1.0})
    refused("rope", "not finite", rd=4, freqs=[1.0, float("inf")])
    refused("rope", "mscale", mscale=float("nan"))
    x = _row_op(4)
    refused("rope", "same strides", x=x, y={**x, "rs": 512, "hs": 128})
    refused("rope", "pos needs", batch={"pos": _host(5, np.int32), "rows": 6})
    refused("rope", batch={"pos": _host(6, np.int32), "rows": 6})


def test_sizes():
    L = p0k.lib()
    assert L.p0k_kv_code_bytes(3, 8) == 3 * 8 * 2 * 64 * 128
    assert L.p0k_kv_scale_bytes(3, 8) == 3 * 8 * 2 * 4
    assert L.p0k_kv_tail_bytes(5, 8) == 5 * 8 * 2 * 2 * 64 * 128 * 2
    assert L.p0k_kv_code_bytes(1 << 20, 16) == 1 << 38


# ------------------------------------------------------------------------------------------------ GPU: rotary positions
def rope_freqs(rd, theta, sc):
    f = theta ** (-2.0 * np.arange(rd // 2) / rd)
    if sc and sc["kind"] == "linear":
        f = f / sc["factor"]
    if sc and sc["kind"] == "bands":
        u = np.clip((sc["orig"] * f / (2 * np.pi) - sc["low"]) / (sc["high"] - sc["low"]), 0, 1)
        f = f * (u + (1 - u) / sc["factor"])
    return f


def rope_ref(x, t, f, half, m=1.0):
    """-> (y, tolerance); angles reduced in extended precision so that far positions stay exact"""
    rd = 2 * len(f)
    a = np.asarray(t, np.longdouble)[:, None] * (f.astype(np.longdouble))
    a = np.remainder(a, 2 * np.longdouble("3.14159265358979323846264338327950288")).astype(np.float64)[:, None]
    x = x.astype(np.float64)
    i = np.arange(rd // 2)
    i1, i2 = (i, i + rd // 2) if half else (2 * i, 2 * i + 1)
    y, mag = x.copy(), np.zeros_like(x)
    y[..., i1] = m * (x[..., i1] * np.cos(a) - x[..., i2] * np.sin(a))
    y[..., i2] = m * (x[..., i2] * np.cos(a) + x[..., i1] * np.sin(a))
    mag[..., i1] = mag[..., i2] = abs(m) * (np.abs(x[..., i1]) + np.abs(x[..., i2]))
    # frequencies and positions are 64-bit numbers: an angle of a turns is off by a 2^-52 of them
    far = np.zeros_like(x)
    far[..., i1] = far[..., i2] = (np.abs(np.asarray(t, np.float64))[:, None] * np.abs(f))[:, None] * 2.0 ** -51
    return y, np.where(mag > 0, 2.0 ** -11 * np.abs(y) + 2.0 ** -25 + (2.0 ** -20 + far) * mag, 0)


ROPES = [dict(rd=rd, half=half, sc=sc) for rd in (2, 6, 32, 64, 100, 128) for half in (False, True)
         for sc in (None, {"kind": "linear", "factor": 4.0}, {"kind": "bands", "factor": 8.0, "orig": 8192.0, "low": 1.0, "high": 4.0})
         if rd in (64, 100) or sc is None]


@pytest.mark.gpu
@pytest.mark.parametrize("c", ROPES, ids=lambda c: f"rd{c['rd']}-{'half' if c['half'] else 'pairs'}-{c['sc']['kind'] if c['sc'] else 'plain'}")
@pytest.mark.parametrize("form", ["heads", "token", "inplace", "rows"])
def test_rope(dev, c, form):
    rng = np.random.default_rng(5)
    H, n, pos = (3, [1, 40, 0, 7], [0, 1000003, 9, 2 ** 31 - 8])
    lead, tail = (2, 3) if form != "rows" else (0, 0)
    cu = np.concatenate([[lead], lead + np.cumsum(n)]).astype(np.int32)
    R = int(cu[-1]) + tail
    t = np.concatenate([p + np.arange(m) for p, m in zip(pos, n)])
    theta, m = 500000.0, 1.25
    f = rope_freqs(c["rd"], theta, c["sc"])
    x = rng.standard_normal((R, H, D)).astype(np.float16)
    token = form == "token"
    bx = dev.upload(x if token else np.ascontiguousarray(x.transpose(1, 0, 2)))
    by = dev.upload(np.full((R, H, D), 0x1234, np.uint16))
    st = {"rs": H * D, "hs": D} if token else {}
    t32 = np.resize(t, R)
    if form == "rows":
        t32 = t32 - 5                                                      # (negative positions turn backwards)
        b = {"pos": dev.upload(t32.astype(np.int32)), "rows": R}
    else:
        b = {"pos": dev.upload(np.array(pos, np.int32)), "cu": dev.upload(cu), "B": 4, "rows": R}
    a = {"x": {"buf": bx, **st}, "H": H, "batch": b, "rd": c["rd"], "mode": "half" if c["half"] else "interleaved",
         "theta": theta, "scaling": c["sc"], "mscale": m}
    if form != "inplace":
        a["y"] = {"buf": by, **st}
    try:
        dev.rope(a)
        raw = dev.read(bx if form == "inplace" else by, np.uint16, R * H * D)
        raw = raw.reshape(R, H, D) if token else raw.reshape(H, R, D).transpose(1, 0, 2)
        keep = x.view(np.uint16) if form == "inplace" else np.full((R, H, D), 0x1234, np.uint16)
        np.testing.assert_array_equal(raw[:lead], keep[:lead])
        np.testing.assert_array_equal(raw[R - tail:], keep[R - tail:])
        got = raw[lead:R - tail].copy().view(np.float16).astype(np.float64)
        want, tol = rope_ref(x[lead:R - tail], t32[:R] if form == "rows" else t, f, c["half"], m)
        assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) - tol)
    finally:
        for o in [bx, by] + [v for v in b.values() if isinstance(v, p0k.Buffer)]:
            dev.free(o)


@pytest.mark.gpu
def test_rope_given_frequencies(dev):
    """freqs in host memory, one of them negative; rows of one token at many positions"""
    rng = np.random.default_rng(6)
    R, H, rd = 50, 5, 12
    f = np.array([1.0, -0.37, 0.1, 3.3, 1e-9, 0.0])
    x = rng.standard_normal((H, R, D)).astype(np.float16)
    t = rng.integers(0, 10 ** 6, R).astype(np.int32)
    bx, bt = dev.upload(x), dev.upload(t)
    by = dev.buffer(x.nbytes)
    try:
        dev.rope({"x": {"buf": bx}, "y": {"buf": by}, "H": H, "batch": {"pos": bt, "rows": R}, "rd": rd, "freqs": list(f)})
        got = dev.read(by, np.float16, x.size).reshape(x.shape).transpose(1, 0, 2).astype(np.float64)
        want, tol = rope_ref(x.transpose(1, 0, 2), t, f, False)
        assert np.all(np.abs(got - want) <= tol)
    finally:
        for o in (bx, bt, by):
            dev.free(o)


# ------------------------------------------------------------------------------------------------ GPU: writing, reading
@pytest.mark.gpu
@pytest.mark.parametrize("token,pad", [(False, 0), (True, 0), (False, 8), (True, 24)])
@pytest.mark.parametrize("steps", [[1] * 70, [63, 1, 1], [64], [65, 63, 128], [7] * 30, [200, 1, 55, 64], [130, 300]], ids=str)
def test_append_reads_back(cache, steps, token, pad):
    """whatever the calls' sizes, the cache holds the same values; rows outside the batch take no part"""
    rng = np.random.default_rng(len(steps))
    c = cache(3, 3, 9, seed=1)
    pos = 0
    for n in steps:
        # slot 2 lags behind by one token, slot 0 is not in the batch
        seqs = [(2, max(0, pos - 1), n if pos else n - 1), (1, pos, n)]
        c.append([s for s in seqs if s[2]], rng, token, pad, lead=3, tail=2)
        pos += n
    c.check_all(token)


@pytest.mark.gpu
def test_append_special_values(cache):
    """infinities to the largest value, NaN to 0, blocks of zeros, the smallest values, values on a rounding border"""
    rng = np.random.default_rng(9)
    c = cache(2, 1, 8)

    def special(n, h, d):
        x = rng.standard_normal((n, h, d)).astype(np.float16)
        x[:64] = 0                                                   # a block of zeros
        x[64:128] = rng.integers(0, 5, (64, h, d)) * np.float16(6e-8)    # subnormal
        x[128:192, :, ::3] = np.inf
        x[130:192:7, :, 1] = np.nan
        x[192:256] = (rng.integers(-254, 255, (64, h, d)) * 0.5).astype(np.float16)   # scale 1: every other value a tie
        x[192, :, 0] = 127
        x[256:320] = -np.inf
        x[330, :, 5] = np.nan
        x[331, :, 6] = -np.inf
        return x
    c.append([(0, 0, 340)], rng, make=special)
    c.check_all()
    k, _, _ = c.read([(0, 192, 64)])
    assert np.all(k.view(np.float16)[0, :, 0] == 127)


@pytest.mark.gpu
def test_append_goes_back(cache):
    """rejected tokens: the sequence goes back up to 64 tokens, over the border of a block and to its start"""
    rng = np.random.default_rng(10)
    c = cache(2, 2, 12)
    c.append([(0, 0, 130), (1, 0, 70)], rng)
    for a, b in [((0, 125, 9), (1, 64, 3)), ((0, 130, 70), (1, 67, 61)), ((0, 190, 5), (1, 120, 100)), ((0, 131, 200), (1, 128, 1)),
                 ((0, 331, 21), (1, 129, 130)), ((0, 288, 1), (1, 195, 66))]:
        c.append([a, b], rng)
        c.check_all()


@pytest.mark.gpu
def test_append_long_over_an_open_block(cache):
    """a call over many blocks whose first was open: what it held is read before its place in the tail is written again"""
    rng = np.random.default_rng(11)
    for n in (64 * 2, 64 * 2 + 5, 64 * 3 + 1, 64 * 4 + 63, 64 * 5):
        for first in (1, 33, 63):
            c = cache(4, 5, 12, seed=n)
            c.append([(s, 0, first) for s in range(5)], rng)
            c.append([(s, first, n + s) for s in range(5)], rng)
            c.check_all()


@pytest.mark.gpu
def test_append_bad_pages_and_ends(cache):
    """no page: not written and read as zeros; the table's end; slots and positions outside: nothing is written"""
    rng = np.random.default_rng(12)
    c = cache(2, 3, 4, bad=[(0, 1, -1), (1, 0, 10 ** 6), (1, 2, 2 ** 31 - 1)])
    before = c.dev.read(c.c["code"])
    c.append([(0, 0, 200), (1, 0, 300), (2, 0, 256)], rng)
    assert np.any(before != c.dev.read(c.c["code"]))
    for s in range(3):
        n = min(len(c.ref.k[s]), 256)
        c.ref.k[s], c.ref.v[s] = c.ref.k[s][:n], c.ref.v[s][:n]
    k, v, cu = c.read([(0, 0, 200), (1, 0, 300), (2, 0, 256)], lens=[200, 300, 256])
    for i, gone in enumerate([(1,), (0, 2), ()]):
        wk, wv = (w.copy() for w in c.ref.held(i))
        for b in gone:
            wk[b * T:(b + 1) * T] = wv[b * T:(b + 1) * T] = 0
        n = len(wk)
        np.testing.assert_array_equal(k[cu[i]:cu[i] + n], wk.view(np.uint16))
        np.testing.assert_array_equal(v[cu[i]:cu[i] + n], wv.view(np.uint16))
        assert np.all(k[cu[i] + n:cu[i + 1]] == 0) and np.all(v[cu[i] + n:cu[i + 1]] == 0)
    state = [c.dev.read(c.c[n]) for n in ("code", "scale", "tail")]
    c.append([(7, 0, 100), (-1, 0, 64), (1, -5, 100), (2, 256, 70), (0, 2 ** 31 - 1, 9)], rng, skip=range(5))
    for n, w in zip(("code", "scale", "tail"), state):
        np.testing.assert_array_equal(c.dev.read(c.c[n]), w)
    k, v, cu = c.read([(7, 0, 10), (0, 190, 20), (1, -3, 5), (2, 2 ** 31 - 4, 6)], lens=[10, 200, 300, 256], lead=1, tail=1)
    assert np.all(k[0] == 0x1234) and np.all(k[-1] == 0x1234)
    assert np.all(k[cu[0]:cu[1]] == 0) and np.all(k[cu[1] + 10:cu[4]] == 0) and np.any(k[cu[1]:cu[1] + 10] != 0)


@pytest.mark.gpu
def test_batch_offsets_are_held_to_the_rows(cache):
    """cu beyond the tensors' rows, negative or decreasing: nothing outside the buffers is touched"""
    rng = np.random.default_rng(13)
    c = cache(2, 4, 4)
    x = rng.standard_normal((2, 40, D)).astype(np.float16)
    for cu in ([0, 30, 1000, 2000, 2 ** 31 - 1], [-7, 5, 3, 40, 40], [40, 30, 20, 10, 0], [2 ** 31 - 1] * 5, [-1] * 5):
        b = {"pos": c.up(np.zeros(4, np.int32)), "cu": c.up(np.array(cu, np.int32)), "B": 4, "rows": 40}
        k = {"buf": c.up(x)}
        c.dev.kv_append({"cache": c.c, "batch": b, "k": k, "v": k})
        o = c.up(np.zeros((40, 2 * D), np.float16))
        c.dev.kv_attention({"cache": c.c, "batch": b, "q": k, "o": {"buf": o}, "Hq": 2})
        c.dev.rope({"x": k, "H": 2, "batch": b})
        c.dev.kv_read({"cache": c.c, "batch": b, "len": b["pos"], "k": k, "v": {"buf": c.up(x)}})
        c.dev.done()
    assert np.all(np.isfinite(c.dev.read(o, np.float16)))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 600])
def test_decreasing_offsets_end(cache, n):
    """offsets that go up and down, so that sequences would share all rows: the calls end, inside their buffers"""
    rng = np.random.default_rng(15)
    B = 200
    c = cache(2, B, 12)
    x = c.up(rng.standard_normal((8, n, D)).astype(np.float16))
    o = c.up(np.zeros((n, 8 * D), np.float16))
    cu = np.where(np.arange(B + 1) % 2, n, 0).astype(np.int32)
    for pos in (0, 700):
        b = {"pos": c.up(np.full(B, pos, np.int32)), "cu": c.up(cu), "B": B, "rows": n}
        c.dev.kv_append({"cache": c.c, "batch": b, "k": x, "v": x})
        c.dev.kv_attention({"cache": c.c, "batch": b, "q": x, "o": o, "Hq": 8})
        c.dev.kv_attention({"cache": c.c, "batch": b, "q": x, "o": o, "Hq": 8, "window": 70, "sinks": 3})
        c.dev.rope({"x": x, "H": 8, "batch": b})
        c.dev.done()


@pytest.mark.gpu
def test_nothing_to_do(cache):
    """no sequences, no rows: the calls are accepted and write nothing"""
    c = cache(2, 2, 4)
    x, o = c.up(np.full((8, 6, D), 0x1234, np.uint16)), c.up(np.full((6, 8 * D), 0x1234, np.uint16))
    cu = c.up(np.zeros(3, np.int32))
    for B, rows in ((0, 6), (2, 0), (2, 6)):
        b = {"pos": cu, "cu": cu, "B": B, "rows": rows}
        c.dev.kv_append({"cache": c.c, "batch": b, "k": x, "v": x})
        c.dev.kv_read({"cache": c.c, "batch": b, "len": cu, "k": x, "v": o})
        c.dev.kv_attention({"cache": c.c, "batch": b, "q": x, "o": o, "Hq": 8})
        c.dev.rope({"x": x, "H": 8, "batch": b})
    assert np.all(c.dev.read(x, np.uint16) == 0x1234) and np.all(c.dev.read(o, np.uint16) == 0x1234)


@pytest.mark.gpu
def test_many_sequences(cache):
    """more sequences than one step of the search over the batch takes, most of them without rows"""
    rng = np.random.default_rng(14)
    c = cache(1, 150, 2)
    c.append([(s, 0, int(n)) for s, n in enumerate(rng.integers(0, 4, 150) * rng.integers(0, 40, 150))], rng)
    c.check_all()
    c.append([(s, len(c.ref.k[s]), 1) for s in rng.permutation(150)], rng)
    c.check_all()
    c.attend([(s, len(c.ref.k[s]) - 1, 1) for s in rng.permutation(150)], 2, rng)


# ------------------------------------------------------------------------------------------------ GPU: attention
def fill(c, lens, rng):
    c.append([(s, 0, n) for s, n in enumerate(lens) if n], rng)


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,rep", [(1, 1), (2, 2), (3, 4), (2, 5), (1, 8), (2, 16), (1, 24), (1, 40)])
def test_attend_decode(cache, Hkv, rep):
    """one query per sequence, lengths around the blocks' borders"""
    rng = np.random.default_rng(20)
    lens = [1, 2, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 191, 200, 320]
    c = cache(Hkv, len(lens), 5)
    fill(c, lens, rng)
    c.attend([(s, n - 1, 1) for s, n in enumerate(lens)], Hkv * rep, rng)
    c.attend([(s, n - 1, 1) for s, n in reversed(list(enumerate(lens)))], Hkv * rep, rng, token=True, pad=8, lead=2, tail=3,
             ldo=Hkv * rep * D + 4)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 3, 5, 8, 16, 17, 33, 64, 65, 100, 130, 300])
@pytest.mark.parametrize("Hkv,rep", [(2, 1), (1, 3), (2, 4), (1, 16)])
def test_attend_several_queries(cache, Hkv, rep, n):
    """drafts, chunks and whole prompts: causal within the rows"""
    rng = np.random.default_rng(n)
    before = [0, 1, 63, 64, 200]
    c = cache(Hkv, len(before), 9)
    fill(c, [p + n for p in before], rng)
    c.attend([(s, p, n) for s, p in enumerate(before)], Hkv * rep, rng, token=n % 2 == 1)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 70), (63, 4), (64, 0), (65, 64), (100, 4), (128, 130), (1000, 4), (2 ** 32 - 1, 2 ** 32 - 1), (77, 2 ** 32 - 1)])
@pytest.mark.parametrize("n", [1, 6, 90, 260])
def test_attend_window(cache, window, sinks, n):
    """a window of every relation to the blocks, sinks inside and behind the first block, queries that straddle blocks"""
    rng = np.random.default_rng(22)
    before = [0, 3, 64, 150, 401]
    c = cache(2, len(before), 12)
    fill(c, [p + n for p in before], rng)
    c.attend([(s, p, n) for s, p in enumerate(before)], 8, rng, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 7, 150])
@pytest.mark.parametrize("kw", [dict(cap=2.0), dict(cap=30.0, window=90, sinks=4), dict(scale=0.5), dict(scale=2.0 ** -6, cap=1.0)], ids=str)
def test_attend_cap_and_scale(cache, n, kw):
    rng = np.random.default_rng(23)
    c = cache(2, 2, 9)
    fill(c, [n + 200, n], rng)
    c.attend([(0, 200, n), (1, 0, n)], 6, rng, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20, 140])
def test_attend_missing_pages(cache, n):
    """blocks without a page are not seen, also where a row then sees nothing; slots and positions outside see nothing"""
    rng = np.random.default_rng(24)
    c = cache(2, 3, 8, bad=[(0, 0, -1), (0, 2, 999), (1, 0, -7), (1, 1, -1), (1, 2, 2 ** 31 - 1), (1, 3, -2 ** 31)])
    fill(c, [400, 256, 100 + n], rng)
    c.attend([(0, 400 - n, n), (1, 256 - n, n), (2, 100, n)], 4, rng, gone=[(0, 0), (0, 2), (1, 0), (1, 1), (1, 2), (1, 3)])
    c.attend([(9, 0, n), (2, 100, n), (-1, 5, n), (1, -1, n)], 4, rng, nokeys=(0, 2, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20, 140])
def test_attend_large_values(cache, n):
    """scores far apart, values of very different size from block to block, the type's largest"""
    rng = np.random.default_rng(25)
    c = cache(2, 2, 9)
    size = np.repeat(np.float64(10.0) ** rng.integers(-4, 5, 12), 64)

    def make(m, h, d):
        return finite16(rng.standard_normal((m, h, d)) * size[:m, None, None])
    c.append([(0, 0, 300 + n)], rng, make=make)
    c.append([(1, 0, n)], rng, make=lambda m, h, d: finite16(np.full((m, h, d), np.inf)))
    c.attend([(0, 300, n)], 4, rng, qscale=0.01)
    c.attend([(0, 300, n)], 4, rng, qscale=30.0, scale=1.0)
    c.attend([(1, 0, n)], 4, rng)


@pytest.mark.gpu
def test_attend_same_sequence_twice_and_behind(cache):
    """a slot twice in one call, and queries that stand before the cache's end (their own later tokens are there already)"""
    rng = np.random.default_rng(26)
    c = cache(2, 1, 8)
    fill(c, [330], rng)
    c.attend([(0, 320, 10), (0, 329, 1), (0, 329, 1)], 8, rng)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[5000], [3777] * 3, [9000, 1, 700, 64, 4097]], ids=str)
@pytest.mark.parametrize("n", [1, 5, 30])
def test_attend_long(cache, lens, n):
    """long caches, whose keys several workgroups share"""
    rng = np.random.default_rng(27)
    c = cache(2, len(lens), max(lens) // T + 2)
    fill(c, [max(x, n) for x in lens], rng)
    seqs = [(s, max(x, n) - n, n) for s, x in enumerate(lens)]
    a = c.attend(seqs, 8, np.random.default_rng(1))
    b = c.attend(seqs, 8, np.random.default_rng(1))
    np.testing.assert_array_equal(a, b)                              # the same bits again
    c.attend(seqs, 8, rng, window=2000, sinks=4)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(dev):
    """pages whose codes lie beyond 4 GiB of the pool, and behind an offset"""
    rng = np.random.default_rng(28)
    Hkv, pages = 8, 33500
    c = Cache.__new__(Cache)
    c.dev, c.Hkv, c.slots, c.mp, c.bufs, c.ref = dev, Hkv, 2, 4, [], Ref(2, Hkv)
    c.tb = dev.upload(np.array([[33499, 5, 33000, 1], [32768, 33498, 0, 16384]], np.int32))
    c.c = dev.kv_cache(Hkv, pages, 2, 4, c.tb)
    assert c.c["code"].size > 2 ** 32
    try:
        fill(c, [250, 200], rng)
        c.check_all()
        c.attend([(0, 249, 1), (1, 190, 10)], 32, rng)
        c.attend([(0, 100, 150)], 16, rng)
    finally:
        c.free()
        dev.drain_pool()


# ------------------------------------------------------------------------------------------------ GPU: as they are used
@pytest.mark.gpu
def test_decode_loop_in_a_graph(dev):
    """positions rotated, keys and values appended, attention over the cache: captured once, replayed for every token with the
    positions changed in between, against the same steps in 64 bits"""
    rng = np.random.default_rng(30)
    B, Hq, Hkv, steps = 3, 8, 2, 140
    start = np.array([0, 61, 130], np.int32)
    c = Cache(dev, Hkv, B, 6)
    fill(c, start, rng)
    H = Hq + Hkv
    qkv, rot = dev.buffer((H + Hkv) * B * D * 2), dev.buffer((H + Hkv) * B * D * 2)
    pos, cu = dev.upload(start), dev.upload(np.arange(B + 1, dtype=np.int32))
    o = dev.buffer(B * Hq * D * 2)
    batch = {"pos": pos, "cu": cu, "B": B, "rows": B}
    kbytes = Hq * B * D * 2

    def step():
        dev.rope({"x": qkv, "y": rot, "H": H, "batch": batch, "mode": "half"})
        dev.kv_append({"cache": c.c, "batch": batch, "k": {"buf": rot, "off": kbytes}, "v": {"buf": qkv, "off": H * B * D * 2}})
        dev.kv_attention({"cache": c.c, "batch": batch, "q": rot, "o": o, "Hq": Hq, "window": 100, "sinks": 3})
    f = rope_freqs(128, 10000.0, None)
    try:
        dev.graph_begin()
        step()
        g = dev.graph_end()
        for i in range(steps):
            x = rng.standard_normal((H + Hkv, B, D)).astype(np.float16)
            dev.upload(x, qkv)
            dev.upload(start + i, pos)
            if i % 10 == 3:
                step()                                               # (an eager step between the replays)
            dev.graph_launch(g)
            r = dev.read(rot, np.float16, (H + Hkv) * B * D).reshape(H + Hkv, B, D).transpose(1, 0, 2)
            want, tol = rope_ref(x[:H].transpose(1, 0, 2), start + i, f, True)
            assert np.all(np.abs(r[:, :H].astype(np.float64) - want) <= tol)
            got = dev.read(o, np.float16, B * Hq * D).reshape(B, 1, Hq, D).astype(np.float64)
            for b in range(B):
                c.ref.append(b, int(start[b]) + i, r[b:b + 1, Hq:H], x[H:, b][None])
                k, v = c.ref.held(b, read=False)
                w, tol = attend_ref(r[b:b + 1, :Hq], int(start[b]) + i, k, v, Hq // Hkv, window=100, sinks=3)
                assert np.all(np.abs(got[b] - w) <= tol), (i, b)
        dev.done()
        dev.graph_destroy(g)
        c.check_all()
    finally:
        for b in (qkv, rot, pos, cu, o):
            dev.free(b)
        c.free()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 700])
def test_capture_begun_by_the_caller(cache, n):
    """in a capture that the caller began the attention does without workspaces (whole groups, one run of keys): the same
    values, with the context's own calls between the replays"""
    hip = C.CDLL("libamdhip64.so")
    rng = np.random.default_rng(31)
    c = cache(2, 2, 40)
    dev = c.dev
    fill(c, [1500 + n, 200 + n], rng)
    b, cu = c.batch([1500, 200], [n, n], [0, 1])
    q = rng.standard_normal((b["rows"], 8, D)).astype(np.float16)
    qb, o = c.rows(q, False), c.up(np.zeros((b["rows"], 8 * D), np.float16))
    a = {"cache": c.c, "batch": b, "q": qb, "o": o, "Hq": 8}
    stream = C.c_void_p(p0k.lib().p0k_ctx_stream(dev.ctx))
    graph, exe = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 1) == 0                 # thread-local capture mode
    try:
        dev.kv_attention(a)
    finally:
        assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
    try:
        for i in range(3):
            dev.upload(np.zeros((b["rows"], 8 * D), np.float16), o)
            assert hip.hipGraphLaunch(exe, stream) == 0
            dev.done()
            got = dev.read(o, np.float16, b["rows"] * 8 * D).reshape(-1, 8, D).astype(np.float64)
            for s, p in enumerate((1500, 200)):
                k, v = c.ref.held(s, read=False)
                w, tol = attend_ref(q[cu[s]:cu[s + 1]], p, k, v, 4)
                assert np.all(np.abs(got[cu[s]:cu[s + 1]] - w) <= tol)
            dev.kv_attention(a)
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.gpu
def test_two_graphs_share_the_workspaces(cache):
    """graphs of the two kernels and of both block sizes, replayed in turn with eager calls in between and positions changed"""
    rng = np.random.default_rng(32)
    c = cache(4, 6, 70)
    dev = c.dev
    fill(c, [4400] * 6, rng)
    calls, graphs = [], []
    for n in (1, 6, 300):                                            # one of each: 16 rows, 32 rows, blocks of 256
        b, cu = c.batch([4400 - n] * 6, [n] * 6, range(6))
        q = rng.standard_normal((b["rows"], 16, D)).astype(np.float16)
        o = c.up(np.zeros((b["rows"], 16 * D), np.float16))
        a = {"cache": c.c, "batch": b, "q": c.rows(q, False), "o": o, "Hq": 16}
        dev.kv_attention(a)
        want = dev.read(o, np.uint16)
        k, v = c.ref.held(2, read=False)
        w, tol = attend_ref(q[cu[2]:cu[3]], 4400 - n, k, v, 4)
        got = want.view(np.float16)[:b["rows"] * 16 * D].reshape(-1, 16, D)[cu[2]:cu[3]].astype(np.float64)
        assert np.all(np.abs(got - w) <= tol)
        dev.graph_begin()
        dev.kv_attention(a)
        graphs.append(dev.graph_end())
        calls.append((a, b, o, want, n))
    try:
        for i in (0, 1, 2, 1, 0, 2, 2, 0, 1):
            a, b, o, want, n = calls[i]
            dev.upload(np.zeros_like(want), o)
            dev.upload(np.full(6, 1000 - n, np.int32), b["pos"])
            dev.graph_launch(graphs[i])                              # (another length: the plan is made on the device)
            dev.kv_attention(calls[(i + 1) % 3][0])
            dev.upload(np.full(6, 4400 - n, np.int32), b["pos"])
            dev.graph_launch(graphs[i])
            np.testing.assert_array_equal(dev.read(o, np.uint16), want)
    finally:
        for g in graphs:
            dev.graph_destroy(g)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 300])
def test_graph_through_another_context(dev, n):
    """a graph whose attention uses its context's workspaces: launched through another context it is ordered with the calls of
    its own, and refused once that is gone"""
    rng = np.random.default_rng(33)
    own = p0k.Device(0)
    g = None
    try:
        c = Cache(own, 4, 3, 40)
        fill(c, [2300] * 3, rng)
        calls = []
        for m in (n, n + 1):
            b, _ = c.batch([2300 - m] * 3, [m] * 3, range(3))
            q = rng.standard_normal((b["rows"], 16, D)).astype(np.float16)
            o = c.up(np.zeros((b["rows"], 16 * D), np.float16))
            calls.append(({"cache": c.c, "batch": b, "q": c.rows(q, False), "o": o, "Hq": 16}, o))
            own.kv_attention(calls[-1][0])
        want = [own.read(o, np.uint16) for _, o in calls]
        own.graph_begin()
        own.kv_attention(calls[0][0])
        g = own.graph_end()
        for _ in range(4):
            for (_, o), w in zip(calls, want):
                own.upload(np.zeros_like(w), o)
            dev.graph_launch(g)
            own.kv_attention(calls[1][0])
            dev.graph_launch(g)
            dev.done()
            for (_, o), w in zip(calls, want):
                np.testing.assert_array_equal(own.read(o, np.uint16), w)
        c.free()
        own.close()
        with pytest.raises(p0k.P0kError, match="destroyed"):
            dev.graph_launch(g)
    finally:
        own.close()
        if g is not None:
            dev.graph_destroy(g)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 90, 400])
def test_layers_in_one_buffer(dev, n):
    """two layers' caches behind offsets of the same buffers, with one page table behind an offset too, and Q, K, V as parts of
    the same rows ([row][Hq + 2 Hkv][128]); the attention's rows into a part of wider ones"""
    rng = np.random.default_rng(34)
    L, Hq, Hkv, pages, mp = p0k.lib(), 6, 2, 14, 13
    bufs = []

    def up(x):
        bufs.append(dev.upload(np.ascontiguousarray(x)))
        return bufs[-1]
    size = {"code": L.p0k_kv_code_bytes(pages, Hkv), "scale": L.p0k_kv_scale_bytes(pages, Hkv), "tail": L.p0k_kv_tail_bytes(1, Hkv)}
    mem = {k: up(np.zeros(32 + 2 * v, np.uint8)) for k, v in size.items()}
    table = up(np.concatenate([[7], rng.permutation(pages)[:mp]]).astype(np.int32))
    layers = [{**{k: {"buf": mem[k], "off": 16 + i * size[k]} for k in size}, "table": {"buf": table, "off": 4}, "pages": pages, "slots": 1,
               "max_pages": mp, "Hkv": Hkv} for i in range(2)]
    W = Hq + 2 * Hkv
    st = {"rs": W * D, "hs": D}
    try:
        refs = [Ref(1, Hkv) for _ in layers]
        for p, m in ((0, 333), (333, n)):
            b = {"pos": up(np.array([p], np.int32)), "cu": up(np.array([0, m], np.int32)), "B": 1, "rows": m}
            for c, ref in zip(layers, refs):
                x = rng.standard_normal((m, W, D)).astype(np.float16)
                row = up(x)
                dev.kv_append({"cache": c, "batch": b, "k": {"buf": row, "off": Hq * 256, **st}, "v": {"buf": row, "off": (Hq + Hkv) * 256, **st}})
                ref.append(0, p, x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:])
                ref.last = x, row
        for c, ref in zip(layers, refs):
            x, row = ref.last
            o = up(np.full((n, 8 * D), 0x1234, np.uint16))
            dev.kv_attention({"cache": c, "batch": b, "q": {"buf": row, **st}, "o": {"buf": o, "off": D * 2, "ld": 8 * D}, "Hq": Hq})
            got = dev.read(o, np.uint16, n * 8 * D).reshape(n, 8, D)
            assert np.all(got[:, 0] == 0x1234) and np.all(got[:, 7] == 0x1234)
            w, tol = attend_ref(x[:, :Hq], 333, *ref.held(0, read=False), Hq // Hkv)
            assert np.all(np.abs(got[:, 1:7].copy().view(np.float16).astype(np.float64) - w) <= tol)
        for k in size:
            assert np.all(dev.read(mem[k], np.uint8, 16) == 0) and np.all(dev.read(mem[k], np.uint8, 16, 16 + 2 * size[k]) == 0)
    finally:
        dev.done()
        for x in bufs:
            dev.free(x)


@pytest.mark.gpu
def test_prompt_then_gemm_heads(dev):
    """the cache takes Q, K, V as the gemm's `heads` epilogue lays them out, and the attention's rows go on as gemm input"""
    from cases import make_case
    case = make_case(epi="heads", M=70, N=128 * 6, K=256, Hq=4, Hkv=1)
    y = case.run_device(dev)
    y = np.ascontiguousarray(y).view(np.uint16).reshape(6, -1, D)
    M = y.shape[1]
    c = Cache(dev, 1, 1, 3)
    try:
        b, _ = c.batch([0], [M])
        buf = c.up(y)
        size = M * D * 2
        c.dev.kv_append({"cache": c.c, "batch": b, "k": {"buf": buf, "off": 4 * size}, "v": {"buf": buf, "off": 5 * size}})
        h = y.view(np.float16)
        c.ref.append(0, 0, h[4][:, None], h[5][:, None])
        o = c.up(np.zeros((M, 4 * D), np.float16))
        dev.kv_attention({"cache": c.c, "batch": b, "q": buf, "o": o, "Hq": 4})
        got = dev.read(o, np.float16, M * 4 * D).reshape(M, 4, D).astype(np.float64)
        k, v = c.ref.held(0, read=False)
        w, tol = attend_ref(h[:4].transpose(1, 0, 2), 0, k, v, 4)
        assert np.all(np.abs(got - w) <= tol)
    finally:
        c.free()
