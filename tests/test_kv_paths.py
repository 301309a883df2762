"""kv_attention on each of its kernels, against the definition in 64 bits: the runs of keys with blocks of 16 rows and of 32, and
the blocks of 256 rows with the keys in one run and in several. Each test says which one its calls take, from the rules at
the kernels (p0k_kvattn.hip) and the device's CU count, so that it cannot come to test another one unnoticed.

Tolerance as in test_kv_cache.py, except that what the probabilities lose below f16's normal range (2^-25 of the largest each) counts
against their sum, as the result is divided by it: with many keys of like scores a lost key shows."""
import ctypes as C

import numpy as np
import pytest

import p0k
from test_kv_cache import D, T, cache, finite16  # noqa: F401


def plan(c, seqs, Hq, window=0, sinks=0):
    """which kernel takes the call: 'runs16', 'runs32', 'block' (the keys in one run) or 'blocks' (several)"""
    cus, rep, B, rows = c.dev.cus(), Hq // c.Hkv, len(seqs), sum(n for _, _, n in seqs)
    if rows * rep > 256 * B and rows * Hq > 20 * cus:
        groups = (rows * rep // 256 + B) * c.Hkv
        return "block" if c.mp < 8 or groups >= 2 * cus else "blocks"

    def units(rb):
        t = 0
        for s, p, n in seqs:
            ok = p >= 0 and 0 <= s < c.slots
            end = min(p + n, c.mp * T) if ok else 0
            every, lo, su = -(-end // 32), 0, 0
            if ok and window and p >= window:
                lo = min((p + 1 - window) // 32, every)
                su = min(-(-sinks // 32), lo)
            t += (max(su + every - lo, 1) if n else 0) * -(-n * rep // rb) * c.Hkv
        return t
    t, t2 = units(16), units(32)
    return "runs32" if t > 64 * cus and t2 <= t - t // 4 else "runs16"


def reference(q, pos, k, v, rep, window=0, sinks=0, cap=0.0, scale=None, gone=()):
    """q [row][Hq][128], k / v [token][Hkv][128] in 64 bits -> (o, tolerance)"""
    n, Hq, L = q.shape[0], q.shape[1], len(k)
    q = q.astype(np.float64)
    sc = np.float64(np.float32(0.08838834764831845)) if scale is None else scale
    o, tol = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    j, t = np.arange(L)[None, :], (pos + np.arange(n))[:, None]
    see = (j <= t) & ~np.isin(j // T, list(gone))
    if window:
        see &= (j > t - window) | (j < sinks)
    nv = see.sum(1, keepdims=True)
    for h in range(Hq):
        kk, vv = k[:, h // rep], v[:, h // rep]
        s, mag = q[:, h] @ kk.T * sc, np.abs(q[:, h]) @ np.abs(kk).T * sc
        if cap:
            s = cap * np.tanh(s / cap)
        s = np.where(see, s, -np.inf)
        m = s.max(1, keepdims=True, initial=-np.inf)
        p = np.exp(s - np.where(np.isfinite(m), m, 0))
        l = np.maximum(p.sum(1, keepdims=True), 1e-300)
        o[:, h] = p @ vv / l
        A = p @ np.abs(vv) / l
        ds = 130 * 2.0 ** -24 * np.where(see, mag, 0).max(1, keepdims=True, initial=0)
        if cap:
            ds = ds + 2.0 ** -20 * cap
        vmax = np.where(see, np.abs(vv).max(1, initial=0)[None], 0).max(1, keepdims=True, initial=0)
        tol[:, h] = 2.0 ** -11 * np.abs(o[:, h]) + 2.0 ** -25 + A * (2.0 ** -11 + 2 * ds + nv * 2.0 ** -24) + np.where(nv, nv * 2.0 ** -25 * vmax / l, 0)
    return o, tol


def attend(c, route, seqs, Hq, rng, qscale=1.0, gone=(), empty=(), token=False, lead=1, tail=2, call=None, **kw):
    """queries (slot, pos, n) of sequences that hold pos + n tokens, on the kernel `route`; empty: sequences that see nothing"""
    assert plan(c, seqs, Hq, kw.get("window", 0), kw.get("sinks", 0)) == route
    b, cu = c.batch([p for _, p, _ in seqs], [n for _, _, n in seqs], [s for s, _, _ in seqs], lead, tail)
    q = (rng.standard_normal((b["rows"], Hq, D)) * qscale).astype(np.float16)
    o = c.up(np.full((b["rows"], Hq * D), 0x1234, np.uint16))
    a = {"cache": c.c, "batch": b, "q": c.rows(q, token), "o": o, "Hq": Hq, **kw}
    call(a) if call else c.dev.kv_attention(a)
    raw = c.dev.read(o, np.uint16, b["rows"] * Hq * D).reshape(b["rows"], Hq, D)
    assert np.all(raw[:cu[0]] == 0x1234) and np.all(raw[cu[-1]:] == 0x1234)
    got = raw.view(np.float16).astype(np.float64)
    for i, (s, p, n) in enumerate(seqs):
        g = got[cu[i]:cu[i + 1]]
        if i in empty:
            assert np.all(g == 0)
            continue
        if n == 0:
            continue
        k, v = c.ref.held(s, read=False)
        assert len(k) == p + n
        w, tol = reference(q[cu[i]:cu[i + 1]], p, k, v, Hq // c.Hkv, gone=[x for y, x in gone if y == s], **kw)
        err = np.abs(g - w)
        at = np.unravel_index(np.argmax(np.where(np.isfinite(err), err / tol, np.inf)), err.shape)
        assert np.all(err <= tol), f"sequence {i} {(s, p, n)}: {err[at]} > {tol[at]} at {at}"
    return raw, a, o


def fill(c, lens, rng, make=None):
    c.append([(s, 0, n) for s, n in enumerate(lens) if n], rng, make=make)


# ------------------------------------------------------------------------------------------------ blocks of 256 rows
BLOCKS = [("block", 7, [(0, 17, 431), (1, 0, 400)]), ("blocks", 30, [(0, 1100, 420), (1, 3, 390), (2, 900, 2)]),
          ("blocks", 40, [(0, 2000, 500), (1, 2, 0), (2, 0, 1), (3, 700, 0), (4, 60, 333), (5, 299, 1)])]


@pytest.mark.gpu
@pytest.mark.parametrize("route,mp,seqs", BLOCKS, ids=["one-run", "runs", "unequal"])
@pytest.mark.parametrize("kw", [{}, dict(cap=30.0), dict(cap=1.5), dict(cap=4.0, window=200, sinks=70), dict(window=64), dict(scale=0.3)], ids=str)
def test_blocks(cache, route, mp, seqs, kw):  # noqa: F811
    """plain, scores far below the cap and beyond it, windows; sequences of very different row counts, some of no rows"""
    rng = np.random.default_rng(90)
    c = cache(2, len(seqs), mp)
    fill(c, [p + n for _, p, n in seqs], rng)
    attend(c, route, seqs, 16, rng, token=bool(kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("route,mp,seqs", [("block", 7, [(0, 0, 448), (1, 5, 400), (2, 20, 3)]), ("blocks", 24, [(0, 1000, 420), (1, 0, 400), (2, 800, 65)])])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_blocks_missing_pages(cache, route, mp, seqs, cap):  # noqa: F811
    """blocks without a page, at a sequence's start so that its first rows see nothing, in its middle and at its end"""
    rng = np.random.default_rng(91)
    gone = [(0, 0), (0, 1), (0, 5), (1, 0), (1, 1), (1, 2), (2, 0)] + ([(0, 16), (2, 12)] if mp > 7 else [])
    c = cache(2, 3, mp, bad=[(s, b, (-1, 10 ** 6, -2 ** 31)[b % 3]) for s, b in gone])
    fill(c, [p + n for _, p, n in seqs], rng)
    # (the block that a sequence is still filling lies in its tail: its page does not matter)
    attend(c, route, seqs, 16, rng, gone=[(s, b) for s, b in gone if (b + 1) * T <= len(c.ref.k[s])], cap=cap)


@pytest.mark.gpu
@pytest.mark.parametrize("mp,route", [(7, "block"), (30, "blocks")])
def test_blocks_nothing_to_see(cache, mp, route):  # noqa: F811
    """slots and positions outside the cache between sequences that have tokens: zeros, and the others as ever"""
    rng = np.random.default_rng(92)
    c = cache(2, 2, mp)
    fill(c, [430, 300], rng)
    attend(c, route, [(2, 10, 300), (0, 30, 400), (-1, 0, 40), (1, -1, 290), (1, 295, 5), (2 ** 31 - 1, 2 ** 31 - 1, 300)], 16, rng, empty=(0, 2, 3, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("qscale,kw", [(0.01, {}), (30.0, dict(scale=1.0)), (0.02, dict(cap=3.0)), (0.01, dict(window=333, sinks=64))], ids=str)
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_blocks_values_of_different_size(cache, order, qscale, kw):  # noqa: F811
    """keys and values whose size goes from block to block over the type's whole range, up, down and to and fro"""
    rng = np.random.default_rng(93)
    c = cache(2, 2, 30)
    e = {"up": np.linspace(-6, 4.5, 30), "down": np.linspace(4.5, -6, 30), "mixed": rng.uniform(-6, 4.5, 30)}[order]
    size = np.repeat(10.0 ** e, T)

    def make(m, h, d):
        return finite16(np.clip(rng.standard_normal((m, h, d)) * size[np.arange(m) % 1500, None, None], -65504, 65504))
    seqs = [(0, 1100, 400), (1, 1000, 500)]
    fill(c, [1500, 1500], rng, make)
    attend(c, "blocks", seqs, 16, rng, qscale=qscale, **kw)


# ------------------------------------------------------------------------------------------------ runs of keys
def marked(unit):
    """values by which each unit of 32 tokens shows, in one of 128 places of a head"""
    def make(m, h, d):
        if make.v:
            x = np.zeros((m, h, d), np.float16)
            at = make.token[:m]
            x[np.arange(m), :, (at // unit) % d] = 1.0 + (at % 7)[:, None] / 8.0
        else:
            x = (0.5 * np.random.default_rng(94).standard_normal((m, h, d))).astype(np.float16)
        make.v = not make.v
        return x
    make.v = False
    return make


@pytest.mark.gpu
@pytest.mark.parametrize("route,lens,Hkv,Hq,n", [("runs16", [5000], 2, 8, 1), ("runs16", [3777, 9000, 1, 700, 64, 4097], 2, 8, 1),
                                                 ("runs16", [9000, 2000], 1, 16, 5), ("runs32", [5000, 4000, 6001, 5003], 1, 16, 29),
                                                 ("blocks", [3000, 2600], 2, 16, 330)], ids=str)
@pytest.mark.parametrize("kw", [{}, dict(window=1900, sinks=40)], ids=["all", "window"])
def test_every_key_counts(cache, route, lens, Hkv, Hq, n, kw):  # noqa: F811
    """flat scores over long caches: one unit of 32 keys lost or taken twice would be far outside the tolerance (checked here)"""
    rng = np.random.default_rng(95)
    lens = [max(x, n) for x in lens]
    c = cache(Hkv, len(lens), max(lens) // T + 2)
    make = marked(32)
    make.token = np.concatenate([np.arange(x) for x in lens])
    fill(c, lens, rng, make)
    seqs = [(s, x - n, n) for s, x in enumerate(lens)]
    if kw and route == "runs32":
        kw = dict(window=4900, sinks=40)
    attend(c, route, seqs, Hq, rng, qscale=0.2, **kw)
    k, v = c.ref.held(0, read=False)
    k, v, q = k[:, :1], v[:, :1], 0.2 * rng.standard_normal((1, 1, D))
    w, tol = reference(q, lens[0] - 1, k, v, 1, **kw)
    see = [u for u in range(-(-lens[0] // 32)) if not kw or u == 0 or u * 32 > lens[0] - kw["window"]]
    for u in see:
        less = v.copy()
        less[u * 32:(u + 1) * 32] = 0
        w2, _ = reference(q, lens[0] - 1, k, less, 1, **kw)
        assert np.any(np.abs(w2 - w) > 3 * tol)


RUNS32 = [dict(), dict(cap=30.0), dict(cap=1.5), dict(window=4700, sinks=70), dict(window=4600, sinks=4, cap=10.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", RUNS32, ids=str)
def test_runs_of_32_rows(cache, kw):  # noqa: F811
    """blocks of 32 rows: the last one partial, sequences of other lengths and of none between them; the same bits again"""
    rng = np.random.default_rng(96)
    lens = [5000, 5600, 64, 5001, 0, 4800, 4999]
    c = cache(1, len(lens), 90)
    fill(c, lens, rng)
    seqs = [(s, x - n, n) for s, (x, n) in enumerate(zip(lens, [29, 29, 1, 30, 0, 29, 3]))]
    a, call, o = attend(c, "runs32", seqs, 16, rng, **kw)
    c.dev.upload(np.zeros_like(a), o)
    c.dev.kv_attention(call)
    b = c.dev.read(o, np.uint16, a.size).reshape(a.shape)
    np.testing.assert_array_equal(a[1:-2], b[1:-2])


@pytest.mark.gpu
def test_runs_of_32_rows_missing_pages(cache):  # noqa: F811
    rng = np.random.default_rng(97)
    gone = [(0, 0), (0, 40), (0, 77), (1, 1)] + [(2, b) for b in range(78)]
    c = cache(1, 4, 80, bad=[(s, b, -1) for s, b in gone])
    fill(c, [5001, 5000, 78 * T, 5000], rng)
    # (the third sequence has no pages at all and nothing in its tail)
    attend(c, "runs32", [(0, 4972, 29), (1, 4971, 29), (2, 78 * T - 29, 29), (3, 4971, 29), (9, 100, 29)], 16, rng, gone=gone, empty=(2, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("route", ["runs16", "runs32", "blocks"])
def test_captured_by_the_caller(cache, route):  # noqa: F811
    """without the context's workspaces (a capture that the caller began), each form, several replays; a wave's units and a
    workgroup's tiles are more than the 64 whose pages it looks up at once"""
    hip = C.CDLL("libamdhip64.so")
    rng = np.random.default_rng(98)
    n, lens = {"runs16": (5, [21000, 300, 2500]), "runs32": (29, [5000, 4800, 5100, 4900]), "blocks": (400, [6000, 900])}[route]
    Hkv = 2 if route == "blocks" else 1
    c = cache(Hkv, len(lens), 330)
    fill(c, lens, rng)
    stream = C.c_void_p(p0k.lib().p0k_ctx_stream(c.dev.ctx))
    graph, exe = C.c_void_p(), C.c_void_p()

    def call(a):
        c.dev.done()
        assert hip.hipStreamBeginCapture(stream, 1) == 0             # thread-local capture mode
        try:
            c.dev.kv_attention(a)
        finally:
            assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
        assert hip.hipGraphLaunch(exe, stream) == 0
        c.dev.done()
    seqs = [(s, x - n, n) for s, x in enumerate(lens)]
    try:
        raw, a, o = attend(c, route, seqs, 16, rng, call=call, window=4700 if route == "runs32" else 0)
        for _ in range(3):
            c.dev.kv_attention(a)                                    # the context's own, with workspaces
            c.dev.upload(np.full_like(raw, 0x1234), o)
            assert hip.hipGraphLaunch(exe, stream) == 0
            c.dev.done()
            np.testing.assert_array_equal(c.dev.read(o, np.uint16, raw.size).reshape(raw.shape), raw)
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


# ------------------------------------------------------------------------------------------------ mixed batches
@pytest.mark.gpu
@pytest.mark.parametrize("route,seqs", [
    ("blocks", [(0, 2999, 1), (1, 500, 700), (2, 100, 6)]), ("blocks", [(0, 0, 600), (1, 2000, 1), (2, 63, 1), (3, 1500, 900), (4, 0, 1)]),
    ("runs16", [(s, 200 + 37 * s, 1) for s in range(11)] + [(11, 640, 300)] + [(s, 900, 1) for s in range(12, 16)])], ids=["draft", "chunks", "runs"])
def test_decode_rows_beside_chunks(cache, route, seqs):  # noqa: F811
    """rows mixed as they come: the kernel is chosen for the call, every sequence is right on it"""
    rng = np.random.default_rng(99)
    c = cache(2, len(seqs), 50)
    fill(c, [p + n for _, p, n in seqs], rng)
    attend(c, route, seqs, 16, rng)
    attend(c, route, seqs, 16, rng, cap=5.0, window=450, sinks=3, token=True)
