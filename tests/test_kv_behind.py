"""Reading and attending over a part of what a sequence holds: the tokens behind the call's last one are there already (a prompt that
was written at once and whose queries come in chunks, a prefix of a sequence). The block in which the call ends is taken from the
tail in f16 while that holds it, else from its codes."""
import numpy as np
import pytest

from test_kv_back import TailRef
from test_kv_cache import D, T, cache, quantised  # noqa: F401
from test_kv_paths import plan, reference


class Part(TailRef):
    def part(self, slot, end):
        """keys and values of tokens 0 .. end - 1 in 64 bits, as a call that ends there takes them"""
        out = []
        for x in (self.k[slot], self.v[slot]):
            y = x.astype(np.float64)
            for b in range(min(len(x), end) // T + 1):
                whole = (b + 1) * T <= len(x)
                if whole and (b < end // T or self.tail[slot][b % 2] != b):
                    y[b * T:(b + 1) * T] = quantised(x[b * T:(b + 1) * T])[0]
            out.append(y[:end])
        return out


def attend(c, route, seqs, Hq, rng, **kw):
    assert plan(c, seqs, Hq, kw.get("window", 0), kw.get("sinks", 0)) == route
    b, cu = c.batch([p for _, p, _ in seqs], [n for _, _, n in seqs], [s for s, _, _ in seqs])
    q = rng.standard_normal((b["rows"], Hq, D)).astype(np.float16)
    o = c.up(np.zeros((b["rows"], Hq * D), np.float16))
    c.dev.kv_attention({"cache": c.c, "batch": b, "q": c.rows(q, False), "o": o, "Hq": Hq, **kw})
    got = c.dev.read(o, np.float16, b["rows"] * Hq * D).reshape(b["rows"], Hq, D).astype(np.float64)
    for i, (s, p, n) in enumerate(seqs):
        w, tol = reference(q[cu[i]:cu[i + 1]], p, *c.ref.part(s, p + n), Hq // c.Hkv, **kw)
        err = np.abs(got[cu[i]:cu[i + 1]] - w)
        assert np.all(err <= tol), (i, s, p, n, np.nanmax(err - tol))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(window=300, sinks=70), dict(cap=8.0)], ids=str)
def test_attend_a_part(cache, kw):  # noqa: F811
    """every place at which a call can end: inside the first blocks, the two that the tail holds, those whose places were taken"""
    rng = np.random.default_rng(110)
    c = cache(2, 3, 30)
    c.ref = Part(3, 2)
    c.append([(0, 0, 1500), (1, 0, 330), (2, 0, 128)], rng)
    ends = [(0, 1500), (0, 1450), (0, 1408), (0, 1400), (0, 1300), (0, 1), (0, 63), (0, 64), (0, 65), (0, 700), (1, 329), (1, 319), (1, 255), (1, 250),
            (1, 33), (2, 128), (2, 127), (2, 64), (2, 63), (2, 5)]
    attend(c, "runs16", [(s, e - 1, 1) for s, e in ends], 8, rng, **kw)
    attend(c, "runs16", [(s, e - min(e, 7), min(e, 7)) for s, e in ends], 8, rng, **kw)
    attend(c, "blocks", [(0, 100, 450), (1, 10, 280), (0, 1000, 401)], 16, rng, **kw)
    attend(c, "blocks", [(0, 0, 777)], 16, rng, **kw)


@pytest.mark.gpu
def test_attend_a_part_in_blocks_of_32_rows(cache):  # noqa: F811
    rng = np.random.default_rng(111)
    c = cache(1, 4, 90)
    c.ref = Part(4, 1)
    c.append([(s, 0, 5600) for s in range(4)], rng)
    attend(c, "runs32", [(0, 5000, 29), (1, 5300, 29), (2, 5571, 29), (3, 5503, 29)], 16, rng)


@pytest.mark.gpu
def test_prompt_in_chunks(cache):  # noqa: F811
    """a prompt written by one call and attended in chunks of odd sizes"""
    rng = np.random.default_rng(112)
    c = cache(2, 1, 40)
    c.ref = Part(1, 2)
    c.append([(0, 0, 2000)], rng)
    at = 0
    for n in (333, 1, 400, 64, 65, 380, 500, 257):
        attend(c, "blocks" if n * 8 > 256 and n * 16 > 20 * c.dev.cus() else "runs16", [(0, at, n)], 16, rng)
        at += n
    assert at == 2000


@pytest.mark.gpu
def test_read_a_part(cache):  # noqa: F811
    """kv_read of a sequence's first tokens: those behind them are zeros"""
    rng = np.random.default_rng(113)
    c = cache(2, 2, 12)
    c.ref = Part(2, 2)
    c.append([(0, 0, 700), (1, 0, 129)], rng)
    for s, ln in [(0, 700), (0, 650), (0, 600), (0, 577), (0, 512), (0, 300), (0, 1), (0, 0), (1, 129), (1, 128), (1, 127), (1, 60)]:
        k, v, _ = c.read([(s, 0, len(c.ref.k[s]))], lens=[ln], token=ln % 2 == 1)
        for x, w in zip((k, v), c.ref.part(s, ln)):
            x = x.view(np.float16)
            whole = c.ref.held(s)[0 if x.base is k.base else 1]
            assert np.all(x[ln:].view(np.uint16) == 0)
            np.testing.assert_array_equal(x[:ln], w.astype(np.float32).astype(np.float16))
            np.testing.assert_array_equal(x[:ln // T * T], whole[:ln // T * T])


@pytest.mark.gpu
def test_slot_taken_over(cache):  # noqa: F811
    """a slot that held a sequence goes to one whose first blocks are another sequence's pages: nothing of the old one shows"""
    rng = np.random.default_rng(114)
    c = cache(2, 2, 12)
    c.ref = Part(2, 2)
    c.append([(0, 0, 150), (1, 0, 700)], rng)
    c.table[0, :2] = c.table[1, :2]
    c.dev.upload(c.table, c.tb)
    c.dev.upload(np.zeros(8, np.int32), c.c["held"], 0)
    c.ref.k[0], c.ref.v[0], c.ref.tail[0] = c.ref.k[1][:128], c.ref.v[1][:128], [None, None]
    for seqs in ([(0, 50, 1), (0, 120, 8), (0, 63, 1)], [(0, 99, 2)]):
        attend(c, "runs16", seqs, 8, rng)
    c.append([(0, 128, 30)], rng)
    c.check_all()
    attend(c, "runs16", [(0, 157, 1), (0, 140, 3), (0, 100, 5), (0, 3, 40), (1, 699, 1), (1, 100, 5)], 8, rng)
    c.append([(0, 158, 200)], rng)
    c.check_all()
    attend(c, "runs16", [(0, 357, 1), (0, 157, 1), (0, 100, 5), (1, 699, 1)], 8, rng)
    assert c.ref.lost == 0


@pytest.mark.gpu
def test_sequence_copied_to_another_slot(cache):  # noqa: F811
    """a sequence goes on in two slots that share its whole pages: the second has a copy of the first one's parts of tail and held"""
    rng = np.random.default_rng(115)
    c = cache(2, 3, 12)
    c.ref = Part(3, 2)
    c.append([(0, 0, 500), (1, 0, 205), (2, 0, 400)], rng)
    for n, size in (("tail", 2 * 65536), ("held", 32)):
        c.dev.copy(c.c[n], 2 * size, c.c[n], size, size)
    c.table[2, :3] = c.table[1, :3]
    c.dev.upload(c.table, c.tb)
    for x in (c.ref.k, c.ref.v, c.ref.tail):
        x[2] = x[1][:] if isinstance(x[1], list) else x[1]
    c.check_all()
    c.append([(2, 205, 7), (1, 205, 3)], rng)
    c.append([(1, 208, 100), (2, 200, 90), (0, 500, 1)], rng)        # (the copy goes back in its own block)
    c.check_all()
    attend(c, "runs16", [(1, 300, 8), (2, 289, 1), (0, 499, 2), (2, 140, 3)], 8, rng)
    assert c.ref.lost == 0
