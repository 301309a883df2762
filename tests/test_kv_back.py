"""Sequences that go back in the 8-bit cache (p0k_kv_append), again and again and to any token.

The tail holds two blocks in f16. A call that starts inside a block of which the tail holds the tokens takes them as they came;
where another block has taken the place, with the cache's `held` buffer, it takes what p0k_kv_read gave for them: f16(fp32(code *
scale)). Either way the cache's contents are known bit for bit. Attention as in test_kv_cache.py."""
import numpy as np
import pytest

import p0k
from test_kv_cache import T, Ref, _host, _host_cache, cache, quantised, refused  # noqa: F401


class TailRef(Ref):
    """Ref that knows which blocks the tail holds: the last of each parity of which tokens were kept there"""

    def __init__(self, slots, Hkv):
        super().__init__(slots, Hkv)
        self.tail, self.lost = [[None, None] for _ in range(slots)], 0

    def append(self, slot, pos, k, v):
        b, end = pos // T, pos + len(k)
        if pos % T and self.tail[slot][b % 2] != b:
            self.lost += 1
            for x in (self.k, self.v):
                x[slot] = np.concatenate([x[slot][:b * T], quantised_block(x[slot], b)[:pos % T], x[slot][pos:]])
        for q in (0, 1):
            new = [j for j in (end // T - 1, end // T) if j % 2 == q and j >= b and j * T < end]
            if new:
                self.tail[slot][q] = new[0]
            elif self.tail[slot][q] is not None and self.tail[slot][q] >= b:
                self.tail[slot][q] = None
        super().append(slot, pos, k, v)


def quantised_block(x, b):
    return quantised(x[b * T:(b + 1) * T])[1]


@pytest.mark.parametrize("call", ["append", "read", "attend"])
def test_held_refusals(call):
    assert p0k.lib().p0k_kv_held_bytes(2, 2) == 64 and p0k.lib().p0k_kv_held_bytes(1 << 20, 512) == 1 << 33
    refused(call, cache=_host_cache(held=_host(64)))
    refused(call, "held needs", cache=_host_cache(held=_host(60)))
    refused(call, "held needs", cache=_host_cache(held={"buf": _host(64), "off": 4}))
    refused(call, "multiple of 4", cache=_host_cache(held={"buf": _host(80), "off": 2}))


CHAINS = [
    [(0, 130), (126, 1), (63, 1)],                      # over two borders, the second call completes the first block again
    [(0, 130), (64, 1), (10, 1), (11, 1), (12, 60)],    # into a block that is open again, then forward
    [(0, 130), (65, 1), (60, 1), (61, 3), (64, 70)],
    [(0, 120), (120, 80), (128, 1), (100, 1), (30, 2), (32, 300)],
    [(0, 1000), (500, 3), (503, 30), (5, 1), (6, 1), (7, 640)],
    [(0, 320), (64, 1), (63, 1), (64, 64), (127, 1), (128, 1), (1, 1)],
    [(0, 400), (128, 10), (130, 10), (64, 300), (363, 1), (0, 20), (19, 200), (130, 1), (40, 3)],
]


@pytest.mark.gpu
@pytest.mark.parametrize("chain", CHAINS, ids=lambda c: "-".join(f"{p}+{n}" for p, n in c))
def test_goes_back_again(cache, chain):  # noqa: F811
    rng = np.random.default_rng(50)
    c = cache(3, 2, 20)
    c.ref = TailRef(2, 3)
    for i, (p, n) in enumerate(chain):
        c.append([(1, p, n)] + ([(0, 0, 70)] if i == 1 else []), rng, token=i % 2 == 1)
        c.check_all()
        L = len(c.ref.k[1])
        c.attend([(1, L - 1, 1), (1, max(0, L - 5), min(L, 5))], 6, rng)
    assert c.ref.lost                                    # (each chain goes back to a block that the tail no longer holds)


@pytest.mark.gpu
def test_goes_back_anywhere(cache):  # noqa: F811
    """many sequences, each back to any of its tokens or on from its end, by any number of tokens"""
    rng = np.random.default_rng(51)
    c = cache(2, 7, 9)
    c.ref = TailRef(7, 2)
    for step in range(60):
        seqs = []
        for s in rng.permutation(7)[:rng.integers(1, 8)]:
            L = len(c.ref.k[s])
            p = L if rng.random() < 0.4 else int(rng.integers(0, L + 1))
            n = int(rng.choice([1, 2, rng.integers(1, 70), rng.integers(1, 400)]))
            n = min(n, 9 * T - p)
            if n > 0:
                seqs.append((int(s), p, n))
        if seqs:
            c.append(seqs, rng, token=step % 3 == 0)
        if step % 5 == 4:
            c.check_all()
    assert c.ref.lost > 20


@pytest.mark.gpu
def test_goes_back_without_held(cache):  # noqa: F811
    """a cache without `held`: to any token of a block that the tail holds, and to any block's start"""
    rng = np.random.default_rng(52)
    c = cache(2, 1, 20)
    c.bufs.append(c.c["held"])
    c.c = {k: v for k, v in c.c.items() if k != "held"}
    c.ref = TailRef(1, 2)
    for p, n in [(0, 130), (126, 1), (127, 70), (64, 3), (66, 200), (192, 1), (128, 70), (190, 5), (64, 1), (0, 500), (448, 1), (449, 60), (449, 1)]:
        c.append([(0, p, n)], rng)
        c.check_all()
    assert c.ref.lost == 0


@pytest.mark.gpu
def test_goes_back_without_a_page(cache):  # noqa: F811
    """tokens that neither the tail nor a page holds are zeros; what the pages hold elsewhere stays"""
    rng = np.random.default_rng(53)
    c = cache(2, 1, 6, bad=[(0, 0, -1)])
    c.append([(0, 0, 200)], rng)
    c.ref.k[0][:64] = c.ref.v[0][:64] = 0
    c.append([(0, 40, 9)], rng)
    c.check_all()
