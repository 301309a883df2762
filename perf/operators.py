"""Performance cases of the key / value cache operators: what a program that serves a language model on this library asks
of them. Head size 128, f16 rows, an 8-bit cache in blocks of 64 tokens with a scale for each block, head and K / V; the
block a sequence is still filling is held in f16.

A case is a dict of plain values. Its "op" is the operator:

  rope     rotary positions on the heads of a batch of rows (a decode step's, a prompt's)
  append   rows of K / V written into the cache, and the blocks they touched read back, as a prompt's own attention does
           that must see what later steps will see
  read     cached rows back as f16 (a prefix that moves elsewhere)
  attend   attention of 1 to many queries per sequence over the cache: causal by position, optionally with a sliding
           window and sinks, optionally with capped scores

"B" sequences; "n" rows of the longest one and "L" tokens before them, both spread over the batch by _spread; "Hq" / "Hkv"
heads; "token": rows lie token-major ([row][head][128]) and not head-major. Where `own` is false the operators run as
elementary torch operations on a cache in plain layouts; where it is true, as the library's calls on the library's buffers.
"""
import math
import os
import sys

import torch

own = False
T, D = 64, 128                                   # tokens of a cache block, head size


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # sixteen sequences decoded together: the query and key heads of one token each, positions scaled for a context
        # eight times the trained one
        {"name": "rope_decode", "op": "rope", "B": 16, "n": 1, "L": 30000, "H": 40, "rd": 128, "half": True,
         "scaling": "bands", "token": False},
        # a prompt's rows far into a conversation, rotated over half of each head in the interleaved layout
        {"name": "rope_prompt", "op": "rope", "B": 1, "n": 4001, "L": 60000, "H": 40, "rd": 64, "half": False,
         "scaling": "linear", "token": True},
        # one token of each of 64 sequences into the cache
        {"name": "append_decode", "op": "append", "B": 64, "n": 1, "L": 4000, "Hkv": 8, "token": False},
        # three prompts of odd lengths into the cache, rows as a QKV projection without a head split leaves them
        {"name": "append_prompts", "op": "append", "B": 3, "n": 2777, "L": 0, "Hkv": 8, "token": True},
        # short stretches of eight sequences, few heads (one rank's share)
        {"name": "read_stretches", "op": "read", "B": 8, "n": 301, "L": 2000, "Hkv": 2, "token": False},
        # a long shared prefix back as f16
        {"name": "read_prefix", "op": "read", "B": 1, "n": 16384, "L": 100, "Hkv": 8, "token": False},
        # one token of one sequence over its cache: the smallest attention there is in earnest, latency counts
        {"name": "attend_one", "op": "attend", "B": 1, "n": 1, "L": 3776, "Hq": 32, "Hkv": 8, "window": 0, "sinks": 0,
         "cap": 0.0, "token": False},
        # a serving batch's decode step, lengths of all kinds
        {"name": "attend_batch", "op": "attend", "B": 48, "n": 1, "L": 6000, "Hq": 32, "Hkv": 8, "window": 0, "sinks": 0,
         "cap": 0.0, "token": False},
        # decode over very long streams with a window and four first tokens that stay visible
        {"name": "attend_window", "op": "attend", "B": 12, "n": 1, "L": 100000, "Hq": 32, "Hkv": 4, "window": 4096,
         "sinks": 4, "cap": 0.0, "token": False},
        # draft tokens verified: six queries per sequence
        {"name": "attend_draft", "op": "attend", "B": 8, "n": 6, "L": 9000, "Hq": 32, "Hkv": 8, "window": 0, "sinks": 0,
         "cap": 0.0, "token": True},
        # two prompts' next chunks after a long cache, capped scores
        {"name": "attend_chunk", "op": "attend", "B": 2, "n": 777, "L": 12000, "Hq": 32, "Hkv": 8, "window": 0, "sinks": 0,
         "cap": 30.0, "token": False},
        # a whole prompt over its own freshly written cache: the most matrix products
        {"name": "attend_prompt", "op": "attend", "B": 1, "n": 5003, "L": 0, "Hq": 32, "Hkv": 8, "window": 0, "sinks": 0,
         "cap": 0.0, "token": False},
    ]


def _log(rng, lo, hi):
    """a size between lo and hi, even over its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "attend", "attend", "attend", "attend"])
    token = rng.random() < 0.4
    if op == "rope":
        H, n = rng.choice([9, 20, 40, 72]), rng.choice([1, 1, _log(rng, 2, 4000)])
        B = rng.randint(1, 64) if n == 1 else rng.randint(1, max(1, min(4, 4000 // n)))
        half = rng.random() < 0.5
        return {"op": op, "B": B, "n": n, "L": _log(rng, 1, 400000), "H": H, "rd": rng.choice([32, 64, 96, 128]),
                "half": half, "scaling": rng.choice(["none", "linear", "bands"]), "token": token}
    if op in ("append", "read"):
        Hkv, n = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, _log(rng, 2, 60), _log(rng, 64, 6000)])
        if op == "read":
            n = _log(rng, 30, 12000)
        B = max(1, min(_log(rng, 1, 64), 70000 // (n * Hkv)))
        L = rng.choice([0, _log(rng, 64, 8000)])
        return {"op": op, "B": B, "n": n, "L": L, "Hkv": Hkv, "token": token}
    Hkv, rep = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    window = rng.choice([0, 0, _log(rng, 100, 5000)])
    c = {"op": op, "Hq": Hkv * rep, "Hkv": Hkv, "window": window, "sinks": rng.choice([0, 1, 4, 70]) if window else 0,
         "cap": rng.choice([0.0, 0.0, 0.0, 50.0]), "token": token}
    kind = rng.choice(["decode", "decode", "draft", "chunk", "prompt"])
    if kind in ("decode", "draft"):
        B = _log(rng, 1, 64)
        L = min(_log(rng, 50, 60000), 2500000 // (B * Hkv))
        return {**c, "B": B, "n": 1 if kind == "decode" else rng.randint(2, 16), "L": L}
    if kind == "chunk":
        B, n = rng.randint(1, 3), _log(rng, 20, 700)
        return {**c, "B": B, "n": n, "L": max(64, min(_log(rng, 100, 12000), 320000000 // (B * n * Hkv * rep)))}
    n = min(_log(rng, 100, 4000), int(math.sqrt(7e8 / (Hkv * rep))))
    return {**c, "B": max(1, min(rng.randint(1, 3), 4000 // n)), "n": n, "L": 0}


def _spread(c):
    """(pos, n) of each sequence: the first has the case's full sizes, the others less by a fixed irregular rule. Chunks of
    more than a block begin at a block's border."""
    got = []
    for b in range(c["B"]):
        f = 1.0 - 0.85 * ((b * 0.6180339887) % 1.0)
        n, p = max(1, int(c["n"] * f)), int(c["L"] * f)
        got.append((p // T * T if n > T and c["op"] == "append" else p, n))
    return got


def _seen(c, p):
    """keys that the query at position p sees"""
    w, s = c["window"], c["sinks"]
    return p + 1 if not w or p < w else w + min(s, p + 1 - w)


def work(case):
    seqs = _spread(case)
    rows = sum(n for _, n in seqs)
    if case["op"] == "rope":
        return {"bytes": 2 * rows * case["H"] * D * 2, "flops": 6 * rows * case["H"] * case["rd"] // 2}
    h = case["Hkv"]
    if case["op"] == "read":
        return {"bytes": rows * h * D * 2 * 3, "flops": 2 * rows * h * D}
    if case["op"] == "append":
        back = sum(p + n - p // T * T for p, n in seqs)                        # rows read back, in f16
        full = sum((p + n) // T * T - min((p + n) // T * T, p // T * T) for p, n in seqs)
        return {"bytes": 2 * h * D * (2 * rows + full + 2 * back), "flops": 8 * h * D * back}
    keys = sum(_seen(case, p + n - 1) if n == 1 else
               (p + n if not case["window"] else min(p + n, case["window"] + n + case["sinks"])) for p, n in seqs)
    pairs = sum(sum(_seen(case, p + i) for i in range(n)) for p, n in seqs)
    return {"bytes": keys * h * D * 2 + 2 * rows * case["Hq"] * D * 2, "flops": 4 * D * case["Hq"] * pairs}


# ------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _kv(g, rows, h):
    """rows of K and V, [row][head][128]: keys with a few large channels, values of differing size from row to row"""
    ch = 0.4 + 0.2 * torch.rand(h, D, generator=g, device="cuda") + 2.5 * (torch.rand(h, D, generator=g, device="cuda") < 0.03)
    k = (_randn(g, rows, h, D) * ch).half()
    v = (_randn(g, rows, h, D) * torch.exp(0.3 * _randn(g, rows, 1, 1))).half()
    return k, v


def _tensors(case, seed):
    """the inputs of a case, in plain layouts: all that depends on the seed"""
    g, seqs, x = _gen(seed), _spread(case), {}
    rows = sum(n for _, n in seqs)
    if case["op"] == "rope":
        x["x"] = _randn(g, rows, case["H"], D).half()
        return x
    # the tokens that the cache holds before the call (append: up to pos; otherwise all of them)
    held = [p if case["op"] == "append" else p + n for p, n in seqs]
    if case["op"] == "read":
        held = [h + 17 * b for b, h in enumerate(held)]                        # the sequence goes on behind the stretch
    x["held"] = held
    x["hk"], x["hv"] = _kv(g, sum(held), case["Hkv"])
    x["need"] = [(max(h, p + n) + T) // T for h, (p, n) in zip(held, seqs)]    # pages of each sequence
    x["order"] = torch.randperm(sum(x["need"]), generator=g, device="cuda").int()
    if case["op"] == "append":
        x["k"], x["v"] = _kv(g, rows, case["Hkv"])
    if case["op"] == "attend":
        x["q"] = (1.5 * _randn(g, rows, case["Hq"], D)).half()
    return x


# ------------------------------------------------------------------------------------------------------- buffers
_dev = None


def _device():
    global _dev
    if _dev is None:
        sys.path.insert(0, os.path.abspath(os.path.join("p0pc0rn-kernels_amd", "python")))
        import p0k
        torch.cuda.init()
        _dev = p0k.Device(0), p0k
    return _dev


class _Memory:
    """One device buffer of the library, given back when its last user is gone; torch sees it as a tensor."""

    def __init__(self, dev, shape, typestr, itemsize):
        self.dev, self.buf = dev, dev.buffer(math.prod(shape) * itemsize)
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (self.buf.ptr, False),
                                         "version": 2, "strides": None}

    def __del__(self):
        self.dev.free(self.buf)


_TYPES = {torch.float16: ("<f2", 2), torch.int32: ("<i4", 4)}


class _Buffers:
    """the library's buffers of one state, by name, and torch's views of them"""

    def __init__(self):
        self.dev, self.t, self.b, self.held = _device()[0], {}, {}, None

    def new(self, name, shape, dtype):
        m = _Memory(self.dev, shape, *_TYPES[dtype])
        self.b[name], self.t[name] = m.buf, torch.as_tensor(m, device="cuda")
        return self.t[name]

    def put(self, name, value):
        value = value.contiguous()
        self.new(name, value.shape, value.dtype)
        self.dev.done()                          # the buffer's clear is queued on the library's stream
        self.t[name].copy_(value)
        return {"buf": self.b[name]}

    def cache(self, **sizes):
        self.held = self.dev.kv_cache(**sizes)
        return self.held

    def __del__(self):
        if self.held is not None:
            self.dev.done()
            self.dev.kv_cache_free(self.held)

    def rows(self, name, x, token):
        """rows [row][head][128] in the case's order, as the library takes them"""
        n, h = x.shape[0], x.shape[1]
        o = self.put(name, x if token else x.transpose(0, 1))
        return {**o, "rs": h * D, "hs": D} if token else {**o, "rs": D, "hs": n * D}

    def out(self, name, n, h, token):
        self.new(name, (n, h, D) if token else (h, n, D), torch.float16)
        return {"buf": self.b[name], **({"rs": h * D, "hs": D} if token else {"rs": D, "hs": n * D})}


def _ints(v):
    return torch.tensor(list(v), dtype=torch.int32, device="cuda")


def _cu(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


_FREQ = {"theta": 500000.0, "factor": 8.0, "orig": 8192.0, "low": 1.0, "high": 4.0}


def prepare(case, seed):
    x, seqs = _tensors(case, seed), _spread(case)
    s = {"case": case, "own": own}
    s["pos"], s["cu"] = _ints(p for p, _ in seqs), _ints(_cu(n for _, n in seqs))
    s["rows"] = sum(n for _, n in seqs)
    if "held" in x:
        mp = max(x["need"])
        table, at = torch.zeros(case["B"], mp, dtype=torch.int32, device="cuda"), _cu(x["need"])
        for b in range(case["B"]):
            table[b, : x["need"][b]] = x["order"][at[b]: at[b + 1]]
        s["table"], s["len"] = table, _ints(x["held"])
        # the blocks that an append touches, from the start of the first one: what is read back
        s["back"] = [(p // T * T, p + n - p // T * T) for p, n in seqs]
    (_prepare_own if own else _prepare_plain)(s, x, seqs)
    torch.cuda.synchronize()
    return s


def _prepare_plain(s, x, seqs):
    c = s["case"]
    if c["op"] == "rope":
        s["x"] = x["x"] if c["token"] else x["x"].transpose(0, 1).contiguous()
        return
    h, pages = c["Hkv"], sum(x["need"])
    s["codes"] = torch.zeros(pages + 1, h, 2, T, D, dtype=torch.int8, device="cuda")      # the last page takes what has none
    s["scales"] = torch.ones(pages + 1, h, 2, device="cuda")
    s["tail"] = torch.zeros(c["B"], h, 2, T, D, dtype=torch.float16, device="cuda")
    empty = {**s, "pos": torch.zeros_like(s["pos"]), "cu": _ints(_cu(x["held"])), "blocks": max(x["need"])}
    if sum(x["held"]):
        s["tail"] = _plain_append(empty, x["hk"], x["hv"])
    lay = (lambda t: t) if c["token"] else (lambda t: t.transpose(0, 1).contiguous())
    s.update({n: lay(x[n]) for n in ("k", "v", "q") if n in x})
    s["blocks"] = max((p + n + T - 1) // T - p // T for p, n in seqs)                     # most blocks that a sequence's rows touch
    if c["op"] == "append":
        s["bpos"], s["bcu"] = _ints(p for p, _ in s["back"]), _ints(_cu(n for _, n in s["back"]))
        s["brows"], s["blen"] = sum(n for _, n in s["back"]), _ints(p + n for p, n in seqs)
    s["nmax"], s["nb"] = max(n for _, n in seqs), max(x["need"])


def _prepare_own(s, x, seqs):
    c, (dev, p0k) = s["case"], _device()
    m = s["mem"] = _Buffers()
    batch = {"pos": m.put("pos", s["pos"]), "cu": m.put("cu", s["cu"]), "B": c["B"], "rows": s["rows"]}
    if c["op"] == "rope":
        a = {"x": m.rows("x", x["x"], c["token"]), "y": m.out("y", s["rows"], c["H"], c["token"]), "H": c["H"],
             "batch": batch, "rd": c["rd"], "mode": "half" if c["half"] else "interleaved", "theta": _FREQ["theta"]}
        if c["scaling"] != "none":
            a["scaling"] = {"kind": c["scaling"], **{k: _FREQ[k] for k in ("factor", "orig", "low", "high")}}
        s["call"] = p0k.rope_args(a, dev.resolve)
        s["out"] = [m.t["y"]]
        return
    cache = m.cache(Hkv=c["Hkv"], pages=sum(x["need"]), slots=c["B"], max_pages=max(x["need"]),
                    table=m.put("table", s["table"])["buf"])
    if sum(x["held"]):
        held = {"cache": cache, "k": m.rows("hk", x["hk"], True), "v": m.rows("hv", x["hv"], True),
                "batch": {"pos": m.put("zero", torch.zeros_like(s["pos"])), "cu": m.put("hcu", _ints(_cu(x["held"]))),
                          "B": c["B"], "rows": sum(x["held"])}}
        torch.cuda.synchronize()
        dev.kv_append(held)
        dev.done()
        for n in ("hk", "hv"):                   # the rows are in the cache now
            del m.t[n], m.b[n]
    if c["op"] == "append":
        s["call"] = p0k.kv_append_args({"cache": cache, "batch": batch, "k": m.rows("k", x["k"], c["token"]),
                                        "v": m.rows("v", x["v"], c["token"])}, dev.resolve)
        batch = {"pos": m.put("bpos", _ints(p for p, _ in s["back"])), "cu": m.put("bcu", _ints(_cu(n for _, n in s["back"]))),
                 "B": c["B"], "rows": sum(n for _, n in s["back"])}
        s["len"] = _ints(p + n for p, n in seqs)
    if c["op"] in ("append", "read"):
        s["read"] = p0k.kv_read_args({"cache": cache, "batch": batch, "len": m.put("len", s["len"]),
                                      "k": m.out("ko", batch["rows"], c["Hkv"], c["token"]),
                                      "v": m.out("vo", batch["rows"], c["Hkv"], c["token"])}, dev.resolve)
        s["out"] = [m.t["ko"], m.t["vo"]]
    else:
        m.new("o", (s["rows"], c["Hq"] * D), torch.float16)
        s["call"] = p0k.kv_attention_args({"cache": cache, "batch": batch, "q": m.rows("q", x["q"], c["token"]), "Hq": c["Hq"],
                                           "o": {"buf": m.b["o"]}, "window": c["window"], "sinks": c["sinks"],
                                           "cap": c["cap"]}, dev.resolve)
        s["out"] = [m.t["o"]]


# ------------------------------------------------------------------------------------------------------- a pass
def run(s):
    """One pass through the operator. The library's calls repeat with their argument structs flattened once, as a decode
    loop makes them."""
    op = s["case"]["op"]
    if s["own"]:
        dev = _dev[0]
        if op == "rope":
            dev.rope_raw(s["call"])
        elif op == "attend":
            dev.kv_attention_raw(s["call"])
        else:
            if op == "append":
                dev.kv_append_raw(s["call"])
            dev.kv_read_raw(s["read"])
        return s["out"]
    return {"rope": _plain_rope, "append": _plain_append_read, "read": _plain_read, "attend": _plain_attend}[op](s)


def _where(pos, cu, rows):
    """sequence and position of each row"""
    r = torch.arange(rows, device="cuda")
    b = torch.searchsorted(cu[1:].long(), r, right=True)
    return b, pos[b].long() + r - cu[b]


def _plain_rope(s):
    c = s["case"]
    rd, x = c["rd"], s["x"].float()
    x = x if c["token"] else x.transpose(0, 1)                                   # [row][head][128]
    f = _FREQ["theta"] ** (-2.0 * torch.arange(rd // 2, device="cuda", dtype=torch.float64) / rd)
    if c["scaling"] == "linear":
        f = f / _FREQ["factor"]
    elif c["scaling"] == "bands":
        u = ((_FREQ["orig"] * f / (2 * math.pi) - _FREQ["low"]) / (_FREQ["high"] - _FREQ["low"])).clamp(0, 1)
        f = f * (u + (1 - u) / _FREQ["factor"])
    a = _where(s["pos"], s["cu"], s["rows"])[1].double()[:, None] * f            # positions reach 10^5: angles in 64 bits
    cos, sin = a.cos().float()[:, None], a.sin().float()[:, None]
    if c["half"]:
        x1, x2 = x[..., : rd // 2], x[..., rd // 2: rd]
        y = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin, x[..., rd:]], -1)
    else:
        x1, x2 = x[..., 0:rd:2], x[..., 1:rd:2]
        y = torch.cat([torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).flatten(-2), x[..., rd:]], -1)
    y = y.half()
    return [y if c["token"] else y.transpose(0, 1).contiguous()]


def _plain_append(s, k, v):
    """rows [row][head][128] into the cache; returns the blocks that are open afterwards"""
    B, nb = s["case"]["B"], s["blocks"]
    pos, n = s["pos"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    end = pos + n
    blk = (pos // T)[:, None] + torch.arange(nb, device="cuda")                  # [B][block]
    t = blk[..., None] * T + torch.arange(T, device="cuda")                      # [B][block][token]
    new = (t >= pos[:, None, None]) & (t < end[:, None, None])
    row = torch.where(new, s["cu"][:-1].long()[:, None, None] + t - pos[:, None, None], 0)
    old = (t < pos[:, None, None])[..., None, None, None]
    x = torch.stack([k[row], v[row]], -2)                                        # [B][block][token][head][K, V][128]
    x = torch.where(new[..., None, None, None], x, 0)
    x = torch.where(old, s["tail"].permute(0, 3, 1, 2, 4)[:, None], x)           # what the first block held already
    x = x.permute(0, 1, 3, 4, 2, 5)                                              # [B][block][head][K, V][token][128]
    amax = x.abs().amax((-1, -2)).float()
    scale = torch.where(amax > 0, amax / 127.0, 1.0)
    code = (x.double() / scale.double()[..., None, None]).round()                # next to a border 32 bits may go astray
    full = (blk + 1) * T <= end[:, None]
    page = torch.where(full, s["table"].long().gather(1, blk.clamp(max=s["table"].shape[1] - 1)), s["codes"].shape[0] - 1)
    s["codes"][page] = code.to(torch.int8)
    s["scales"][page] = scale
    last = (end // T - pos // T)                                                 # the open block among those touched
    open_ = x[torch.arange(B, device="cuda"), last.clamp(max=nb - 1)]
    return torch.where(((last < nb) & (end % T != 0))[:, None, None, None, None], open_, 0)


def _plain_append_read(s):
    k, v = (s["k"], s["v"]) if s["case"]["token"] else (s["k"].transpose(0, 1), s["v"].transpose(0, 1))
    tail = _plain_append(s, k, v)                # (what was open before the call is kept: the pass can be made again)
    return _plain_read({**s, "pos": s["bpos"], "cu": s["bcu"], "rows": s["brows"], "len": s["blen"], "tail": tail})


def _plain_read(s):
    b, t = _where(s["pos"], s["cu"], s["rows"])
    blk, off = t // T, t % T
    page = s["table"].long()[b, blk]
    x = (s["codes"][page, :, :, off].float() * s["scales"][page][..., None]).half()       # [row][head][K, V][128]
    x = torch.where((blk == s["len"][b].long() // T)[:, None, None, None], s["tail"][b, :, :, off], x)
    k, v = x[:, :, 0], x[:, :, 1]
    return [k.contiguous(), v.contiguous()] if s["case"]["token"] else [k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()]


def _plain_attend(s):
    c = s["case"]
    B, h, hq, nmax, nb = c["B"], c["Hkv"], c["Hq"], s["nmax"], s["nb"]
    rep = hq // h
    pos, n = s["pos"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    page = s["table"].long()[:, :nb]
    x = s["codes"][page].float() * s["scales"][page][..., None, None]            # [B][block][head][K, V][token][128]
    ob = ((pos + n) // T).clamp(max=nb - 1)
    x[torch.arange(B, device="cuda"), ob] = torch.where(((pos + n) // T < nb)[:, None, None, None, None], s["tail"].float(),
                                                        x[torch.arange(B, device="cuda"), ob])
    k = x[:, :, :, 0].transpose(1, 2).reshape(B, h, nb * T, D)
    v = x[:, :, :, 1].transpose(1, 2).reshape(B, h, nb * T, D)
    i = torch.arange(nmax, device="cuda")
    row = (s["cu"][:-1].long()[:, None] + i).clamp(max=s["rows"] - 1)            # [B][query], some past the sequence's end
    q = s["q"] if c["token"] else s["q"].transpose(0, 1)
    q = q[row].float().view(B, nmax, h, rep, D).permute(0, 2, 3, 1, 4).reshape(B, h, rep * nmax, D)
    a = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    if c["cap"]:
        a = c["cap"] * torch.tanh(a / c["cap"])
    p, j = (pos[:, None] + i)[..., None], torch.arange(nb * T, device="cuda")    # [B][query][1], [key]
    see = j <= p
    if c["window"]:
        see &= (j > p - c["window"]) | (j < c["sinks"])
    a = a.view(B, h, rep, nmax, nb * T).masked_fill_(~see[:, None, None], -math.inf)
    a = torch.exp(a - a.amax(-1, keepdim=True))
    o = torch.matmul(a.view(B, h, rep * nmax, nb * T), v).view(B, h, rep, nmax, D) / a.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, nmax, hq * D)
    b, t = _where(s["pos"], s["cu"], s["rows"])
    return [o[b, t - pos[b]].half()]


# ------------------------------------------------------------------------------------------------------- 64 bits
def _quantised(x, full):
    """x [token][head][128] f16 of one sequence -> the values its cache holds, in 64 bits: whole blocks through 8 bits"""
    x = x.double()
    if full == 0:
        return x
    w = x[: full * T].view(full, T, *x.shape[1:])
    a = w.abs().amax((1, 3), keepdim=True)
    sc = torch.where(a > 0, (a / 127.0).float().double(), 1.0)                   # scales are fp32 numbers
    return torch.cat([(torch.round(w / sc) * sc).view(full * T, *x.shape[1:]), x[full * T:]])


def exact(case, seed):
    x, seqs = _tensors(case, seed), _spread(case)
    cu, token, outs = _cu(n for _, n in seqs), case["token"], []
    lay = (lambda t: t) if token else (lambda t: t.transpose(0, 1))
    if case["op"] == "rope":
        rd, y = case["rd"], x["x"].double()
        t = torch.cat([p + torch.arange(n, device="cuda", dtype=torch.float64) for p, n in seqs])
        for i in range(rd // 2):
            f = math.exp(-2.0 * i / rd * math.log(_FREQ["theta"]))
            if case["scaling"] == "linear":
                f /= _FREQ["factor"]
            if case["scaling"] == "bands":
                turns = _FREQ["orig"] * f / (2 * math.pi)
                u = 0.0 if turns < _FREQ["low"] else 1.0 if turns > _FREQ["high"] else (turns - _FREQ["low"]) / (_FREQ["high"] - _FREQ["low"])
                f = u * f + (1 - u) * f / _FREQ["factor"]
            e = torch.polar(torch.ones_like(t), t * f)[:, None]
            i1, i2 = (i, i + rd // 2) if case["half"] else (2 * i, 2 * i + 1)
            z = torch.complex(y[..., i1], y[..., i2]) * e
            y[..., i1], y[..., i2] = z.real, z.imag
        return [lay(y)]
    at = _cu(x["held"])
    ko, vo = [], []
    for b, (p, n) in enumerate(seqs):
        k, v = x["hk"][at[b]: at[b + 1]], x["hv"][at[b]: at[b + 1]]
        if case["op"] == "append":
            k, v = torch.cat([k, x["k"][cu[b]: cu[b + 1]]]), torch.cat([v, x["v"][cu[b]: cu[b + 1]]])
        k, v = _quantised(k, len(k) // T), _quantised(v, len(v) // T)
        if case["op"] == "append":
            ko.append(k[p // T * T:])
            vo.append(v[p // T * T:])
        elif case["op"] == "read":
            ko.append(k[p: p + n])
            vo.append(v[p: p + n])
        else:
            q = x["q"][cu[b]: cu[b + 1]].double()
            o = torch.empty(n, case["Hq"], D, dtype=torch.float64, device="cuda")
            rep, keys = case["Hq"] // case["Hkv"], torch.arange(p + n, device="cuda")
            here = p + torch.arange(n, device="cuda")[:, None]
            hid = keys > here
            if case["window"]:
                hid = hid | ((keys <= here - case["window"]) & (keys >= case["sinks"]))
            for h in range(case["Hq"]):
                z = q[:, h] @ k[:, h // rep].T / math.sqrt(D)
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                o[:, h] = torch.softmax(z.masked_fill(hid, -math.inf), -1) @ v[:, h // rep]
            outs.append(o.view(n, case["Hq"] * D))
    if case["op"] == "attend":
        return [torch.cat(outs)]
    return [lay(torch.cat(ko)), lay(torch.cat(vo))]
