"""The 8-bit caches of uncompressed layers and attention through a window, measured: keys and values quantised as they
are written and read back, one token's attention over such a cache, and attention that sees a window of the last
tokens and a few first ones, for single tokens and for prompts.

``listed()`` holds the cases that are timed, ``draw(rng)`` gives further cases of the same ranges,
``prepare(case, seed)`` makes what a program holds before the call, ``run(state)`` is one pass through an
operator (its plain form in torch, or, where ``own`` is true, the framework's entry point), ``work(case)``
the bytes and operations the pass cannot do without and ``exact(case, seed)`` the result in float64.

The kinds of case:

- ``write``: new tokens' keys and values into the 8-bit cache (``cache8.write_kv8``), then the tokens of the blocks that
  they touched back as the values that the cache now holds (``cache8.read_kv8``), with every block's exponents;
- ``read``: whole sequences of an 8-bit cache back as rows of 16 bits (``cache8.read_kv8``);
- ``decode8``: one token's attention over an 8-bit cache, whole or through a window (``cache8.paged_decode_8``);
- ``window``: one token's attention over a 16-bit cache through a window (``window.paged_decode_window``);
- ``prefill``: causal attention of prompts through a window (``prefill.prefill_attention``).

An 8-bit cache holds codes (int8 up to 127, or e4m3 up to 448) and, for each block and head, an exponent for the keys and
one for the values: a value is code * 2^exponent. A write that holds a block's first token begins the block
anew: its exponent is the least one at which the largest new value still has a code. Any other write keeps the block's
exponent, or raises it to what its own values need and rounds the codes that are there to the new one.
Through a window of W with S first tokens, the token at place t sees place s <= t where t - s < W or s < S.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
D = 128  # head dimension
SCALE = D ** -0.5
LEAST = -126  # the least exponent, that of a block of zeros
TOP = {"int8": 127.0, "fp8": 448.0}


def listed():
    return [
        # One decode step of 64 requests: a token each, most of them behind others of its block. Latency.
        dict(name="write_step_64", kind="write", code="int8", fmt="bf16", kv=8, group=4, bs=16, n=64, lo=500, hi=4000,
             new=1, mix=1),
        # A step's prompts, as many key as query heads.
        dict(name="write_prompts_4", kind="write", code="fp8", fmt="bf16", kv=32, group=1, bs=16, n=4, lo=1001, hi=3001,
             new=0, mix=2),
        # One session's cache back in 16 bits, for a layer or a host that takes it so.
        dict(name="read_1x4096", kind="read", code="fp8", fmt="bf16", kv=32, bs=16, n=1, lo=4096, hi=4096, mix=3),
        # The sequences of a batch, of odd lengths.
        dict(name="read_16_ragged", kind="read", code="int8", fmt="fp16", kv=8, bs=32, n=16, lo=1000, hi=8191, mix=4),
        # One interactive session. Latency.
        dict(name="decode8_1x4096", kind="decode8", code="fp8", fmt="bf16", kv=32, group=1, bs=16, n=1, lo=4096, hi=4096,
             window=0, sinks=0, mix=5),
        # A serving batch at different points, four query heads a key head.
        dict(name="decode8_24_ragged", kind="decode8", code="int8", fmt="bf16", kv=8, group=4, bs=16, n=24, lo=1000,
             hi=8191, window=0, sinks=0, mix=6),
        # The largest batch: 64 requests of 8192 tokens.
        dict(name="decode8_64x8192", kind="decode8", code="fp8", fmt="bf16", kv=8, group=8, bs=64, n=64, lo=8192, hi=8192,
             window=0, sinks=0, mix=7),
        # Long sessions through a window.
        dict(name="decode8_window_32", kind="decode8", code="int8", fmt="fp16", kv=8, group=4, bs=16, n=32, lo=2000,
             hi=32767, window=4096, sinks=4, mix=8),
        # One very long session through a window of its 16-bit cache. Latency.
        dict(name="window_1x65536", kind="window", fmt="bf16", kv=8, group=4, bs=16, n=1, lo=65536, hi=65536, window=4096,
             sinks=4, mix=9),
        # A batch with one key head per query head.
        dict(name="window_32_ragged", kind="window", fmt="fp16", kv=32, group=1, bs=32, n=32, lo=600, hi=8191, window=1024,
             sinks=16, mix=10),
        # One prompt of a chat.
        dict(name="prefill_1x2047", kind="prefill", fmt="bf16", kv=8, group=4, n=1, lo=2047, hi=2047, window=512, sinks=4,
             mix=11),
        # A step's long prompts.
        dict(name="prefill_2_ragged", kind="prefill", fmt="bf16", kv=32, group=1, n=2, lo=3500, hi=6000, window=1024, sinks=16,
             mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges: sizes over their logarithm, odd ones among them."""
    kind = rng.choice(["write", "write", "read", "decode8", "decode8", "decode8", "window", "window", "prefill"])
    c = dict(kind=kind, fmt=rng.choice(["bf16", "fp16"]), kv=rng.choice([1, 2, 4, 5, 8, 8, 32]), mix=rng.randrange(1 << 30))
    if kind in ("write", "read", "decode8"):
        c["code"] = rng.choice(["int8", "fp8"])
    if kind != "read":
        c["group"] = rng.choice([1, 2, 4, 8]) if c["kv"] < 32 else 1
        if c["kv"] < 8 and rng.random() < 0.4:
            c["group"] = rng.choice([3, 5, 6, 7, 12, 16])
    if kind == "prefill":
        heads = c["kv"] * c["group"]
        c["n"] = _log(rng, 1, 8)
        c["hi"] = _log(rng, 1, min(8191, int((2 ** 31 / heads) ** 0.5)) // c["n"])
    else:
        c["bs"] = rng.choice([16, 32, 64])
        c["n"] = _log(rng, 1, 64)
        most = {"write": 2 ** 18, "read": 2 ** 20, "decode8": 2 ** 22, "window": 2 ** 21}[kind]
        c["hi"] = _log(rng, 1, min(65536, max(64, most // (c["n"] * c["kv"]))))
    c["lo"] = c["hi"] if rng.random() < 0.3 else max(1, c["hi"] // rng.choice([2, 4, 8]))
    if kind == "write":
        c["new"] = rng.choice([0, 1, 1, _log(rng, 1, c["hi"])])
    if kind in ("window", "prefill") or (kind == "decode8" and rng.random() < 0.5):
        c["window"], c["sinks"] = _log(rng, 1, max(1, min(8192, c["hi"]))), rng.choice([0, 1, 4, 16, 33])
    elif kind == "decode8":
        c["window"] = c["sinks"] = 0
    return c


# -- sizes that a case fixes, whatever the seed of its inputs --------------------------------
def _lengths(c):
    r = random.Random(c["mix"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["n"])]


def _new(c):
    """New tokens of each request of a `write` case: all of it, or at most `new` at its end."""
    return [min(L, c["new"]) if c["new"] else L for L in _lengths(c)]


def _dtype(c):
    return torch.float16 if c["fmt"] == "fp16" else torch.bfloat16


def _blocks(L, bs):
    return -(-L // bs)


# -- inputs -----------------------------------------------------------------------------------
def _gen(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 16 + salt)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=g)


def _keys(g, lead, kv):
    """Keys as a model's [*lead, kv, 128]: a spread of its own in each channel of a head about a mean of its own."""
    return _randn(g, *lead, kv, D) * _randn(g, kv, D, std=0.4).exp() + _randn(g, kv, D)


def _block_table(c, g):
    """Requests' blocks, a random permutation of the pool (block 0 is the null block)."""
    need = [_blocks(L, c["bs"]) for L in _lengths(c)]
    perm = (torch.randperm(sum(need), device="cuda", generator=g) + 1).to(torch.int32)
    bt = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    o = 0
    for b, p in enumerate(need):
        bt[b, :p] = perm[o:o + p]
        o += p
    return bt, sum(need) + 1


def _places(bt, bs, spans):
    """Slots of the places [a, e) of each request, end to end."""
    rows = torch.cat([torch.full((e - a,), b, dtype=torch.int64) for b, (a, e) in enumerate(spans)]).cuda()
    pos = torch.cat([torch.arange(a, e) for a, e in spans]).cuda()
    return bt[rows, pos // bs].long() * bs + pos % bs


def _codes(x, code):
    return x.to(torch.float8_e4m3fn).view(torch.int8) if code == "fp8" else x.round().to(torch.int8)


def _values(codes, code):
    """What codes (held as int8, whatever they are) stand for, before their exponent."""
    return (codes.view(torch.float8_e4m3fn) if code == "fp8" else codes).float()


def _need(a, code):
    """The least exponent, as a float, at which values up to `a` have codes."""
    m, k = torch.frexp(a)  # a = m 2^k, m in [1/2, 1)
    top, bits = (0.875, 9) if code == "fp8" else (127.0 / 128.0, 7)
    return torch.where(a > 0, (k - bits + (m > top)).clamp(min=LEAST), LEAST).float()


def _filled(x, code):
    """Codes and exponents [blocks, kv] of whole blocks of values x [blocks, bs, kv, 128]; the codes head by head in a
    block, as the framework lays out its 8-bit caches."""
    e = _need(x.abs().amax(dim=(1, 3)), code)
    c = torch.empty(x.shape[0], x.shape[2], x.shape[1], D, dtype=torch.int8, device="cuda").transpose(1, 2)
    c.copy_(_codes(x * torch.exp2(-e)[:, None, :, None], code))
    return c, e.to(torch.int8)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt, kv = _dtype(c), c["kv"]
    L = _lengths(c)
    if c["kind"] == "prefill":
        T, heads = sum(L), kv * c["group"]
        cu = [sum(L[:i]) for i in range(len(L) + 1)]
        q, k, v = (t.view(T, -1, D) for t in _randn(g, T, (heads + 2 * kv) * D, dtype=dt).split([heads * D, kv * D, kv * D], -1))
        of = torch.cat([torch.full((x,), i) for i, x in enumerate(L)]).cuda()
        return dict(c=c, q=q, k=k, v=v, L=L, of=of, cu=cu)
    lens = torch.tensor(L, dtype=torch.int32, device="cuda")
    bt, blocks = _block_table(c, g)
    s = dict(c=c, lens=lens, bt=bt, span=max(L))
    if c["kind"] == "window":
        s["q"] = _randn(g, c["n"], kv * c["group"], D, dtype=dt)
        s["kc"], s["vc"] = _keys(g, (blocks, c["bs"]), kv).to(dt), _randn(g, blocks, c["bs"], kv, D, dtype=dt)
        return s
    kc, ke = _filled(_keys(g, (blocks, c["bs"]), kv).to(dt).float(), c["code"])
    vc, ve = _filled(_randn(g, blocks, c["bs"], kv, D, dtype=dt).float(), c["code"])
    s.update(kc=kc, vc=vc, exponents=torch.stack([ke, ve], dim=-1).contiguous())
    if c["kind"] == "decode8":
        s["q"] = _randn(g, c["n"], kv * c["group"], D, dtype=dt)
    elif c["kind"] == "read":
        s["back"] = _places(bt, c["bs"], [(0, x) for x in L])
    else:
        new, heads = _new(c), kv * c["group"]
        s["slots"] = _places(bt, c["bs"], [(x - m, x) for x, m in zip(L, new)])
        s["back"] = _places(bt, c["bs"], [((x - m) // c["bs"] * c["bs"], x) for x, m in zip(L, new)])
        T = sum(new)
        # Rows of a step's projection, whose first part is its queries; the keys a little larger than what the cache has
        # seen, so that some blocks' exponents grow.
        rows = _randn(g, T, (heads + 2 * kv) * D, dtype=dt)
        k, s["v"] = (t.view(T, kv, D) for t in rows.split([heads * D, kv * D, kv * D], dim=-1)[1:])
        s["k"] = k.copy_(_keys(g, (T,), kv) * 1.2)
    return s


# -- one pass ---------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"write": _plain_write, "read": _plain_read, "decode8": _plain_decode8, "window": _plain_window,
            "prefill": _plain_prefill}[s["c"]["kind"]](s)


_modules = None


def _own(s):
    global _modules
    if _modules is None:
        sys.path.insert(0, os.path.join(ROOT, "star-kv-serve_amd"))
        from starkv_serve.kernels import cache8, prefill, window
        _modules = cache8, prefill, window
    cache8, prefill, window = _modules
    c = s["c"]
    seen = window.Window(c["window"], c["sinks"]) if c.get("window") else None
    if c["kind"] == "prefill":
        return prefill.prefill_attention(s["q"], s["k"], s["v"], s["L"], SCALE, window=seen)
    if c["kind"] == "window":
        return window.paged_decode_window(s["q"], s["kc"], s["vc"], s["bt"], s["lens"], s["span"], SCALE, seen)
    kc, vc = (t.view(torch.float8_e4m3fn) if c["code"] == "fp8" else t for t in (s["kc"], s["vc"]))
    cache = cache8.Cache8(kc, vc, s["exponents"])
    if c["kind"] == "decode8":
        return cache8.paged_decode_8(s["q"], cache, s["bt"], s["lens"], s["span"], SCALE, window=seen)
    if c["kind"] == "read":
        k, v = cache8.read_kv8(cache, s["back"], _dtype(c))
        return dict(k=k, v=v)
    cache8.write_kv8(s["k"], s["v"], cache, s["slots"])
    k, v = cache8.read_kv8(cache, s["back"], _dtype(c))
    return dict(k=k, v=v, exponents=s["exponents"])


# -- the plain forms --------------------------------------------------------------------------
def _plain_write(s):
    c = s["c"]
    bs, code = c["bs"], c["code"]
    off = s["slots"] % bs
    blocks, at = torch.unique(s["slots"] // bs, return_inverse=True)  # the touched ones, each token's place among them
    fresh = torch.zeros_like(blocks).index_reduce_(0, at, (off == 0).long(), "amax")[:, None] > 0
    for i, (x, codes) in enumerate(((s["k"], s["kc"]), (s["v"], s["vc"]))):
        x, old, held = x.float(), s["exponents"][blocks, :, i].float(), codes[blocks]
        e = _need(torch.zeros_like(old).index_reduce_(0, at, x.abs().amax(-1), "amax"), code)
        e = torch.where(fresh, e, torch.maximum(e, old))
        less = torch.exp2(torch.where(fresh, 0.0, old - e))[:, None, :, None]
        held = _codes(_values(held, code) * less, code)
        held[at, off] = _codes(x * torch.exp2(-e[at])[..., None], code)
        codes[blocks] = held
        s["exponents"][blocks, :, i] = e.to(torch.int8)
    return dict(_plain_read(s), exponents=s["exponents"])


def _plain_read(s):
    c = s["c"]
    blk, off = s["back"] // c["bs"], s["back"] % c["bs"]
    scale = torch.exp2(s["exponents"].float())[blk]
    k, v = (_values(t[blk, off], c["code"]) * scale[..., i, None] for i, t in enumerate((s["kc"], s["vc"])))
    return dict(k=k.to(_dtype(c)), v=v.to(_dtype(c)))


def _seen(s):
    """The places [n, most] that a request's newest token sees, each once, and which of them there are."""
    c, lens = s["c"], s["lens"].long()[:, None]
    if not c["window"]:
        at = torch.arange(s["span"], device="cuda")[None, :]
        return at.expand(c["n"], -1), at < lens
    first = (lens - c["window"]).clamp(min=0)
    w = min(c["window"], s["span"])
    at = torch.arange(c["sinks"] + w, device="cuda")[None, :]
    sink = at < c["sinks"]
    place = torch.where(sink, at, first + at - c["sinks"])
    there = torch.where(sink, at < torch.minimum(first, lens), place < lens)
    return torch.where(there, place, 0), there


def _attend(q, k, v, there):
    """Attention of q [n, kv, group, 128] over k, v [n, kv, t, 128] where `there` [n, t], in 32 bits."""
    score = torch.matmul(q.float(), k.transpose(-1, -2).contiguous()) * SCALE
    score = score.masked_fill(~there[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    return torch.matmul(p / p.sum(-1, keepdim=True).clamp(min=1e-30), v)


def _plain_decode8(s):
    c = s["c"]
    n, kv, bs = c["n"], c["kv"], c["bs"]
    at, there = _seen(s)
    blk = s["bt"].long().gather(1, at // bs)
    scale = torch.exp2(s["exponents"].float())[blk]
    k, v = ((_values(t[blk, at % bs], c["code"]) * scale[..., i, None]).transpose(1, 2).contiguous()
            for i, t in enumerate((s["kc"], s["vc"])))
    return _attend(s["q"].view(n, kv, c["group"], D), k, v, there).reshape(n, -1, D).to(s["q"].dtype)


def _plain_window(s):
    c = s["c"]
    n, kv, bs = c["n"], c["kv"], c["bs"]
    at, there = _seen(s)
    blk = s["bt"].long().gather(1, at // bs)
    k, v = (t[blk, at % bs].float().transpose(1, 2).contiguous() for t in (s["kc"], s["vc"]))
    return _attend(s["q"].view(n, kv, c["group"], D), k, v, there).reshape(n, -1, D).to(s["q"].dtype)


def _plain_prefill(s):
    c, T = s["c"], s["q"].shape[0]
    kv = c["kv"]
    q = s["q"].view(T, kv, -1, D).permute(1, 2, 0, 3).reshape(kv, -1, D).float()
    k, v = (t.transpose(0, 1).contiguous().float() for t in (s["k"], s["v"]))
    t = torch.arange(T, device="cuda")
    start = torch.tensor(s["cu"], device="cuda")[s["of"]]
    back = t[:, None] - t[None, :]
    hidden = (s["of"][:, None] != s["of"][None, :]) | (back < 0) | ((back >= c["window"]) & ((t - start)[None, :] >= c["sinks"]))
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(kv, -1, T, T).mul_(SCALE).masked_fill_(hidden, -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p.view(kv, -1, T), v).view(kv, -1, T, D) / p.sum(-1, keepdim=True)
    return o.permute(2, 0, 1, 3).reshape(T, -1, D).to(s["q"].dtype)


# -- what a pass cannot do without ------------------------------------------------------------
def _seen_of(c, L):
    """Places that the token behind L - 1 others sees."""
    return min(L, c["window"] + min(c["sinks"], max(L - c["window"], 0))) if c["window"] else L


def work(case):
    c, L = case, _lengths(case)
    kv, heads = c["kv"], c["kv"] * c.get("group", 1)
    if c["kind"] == "write":
        new, bs = _new(c), c["bs"]
        first = [(x - m) // bs * bs for x, m in zip(L, new)]
        T, back = sum(new), sum(L) - sum(first)
        blocks = sum(_blocks(x - f, bs) for x, f in zip(L, first))
        # The new rows in 16 bits read and in 8 written, the others of their blocks in 8 read, all of them in 16 written.
        return {"bytes": kv * D * 2 * (3 * T + back - T + 2 * back) + blocks * kv * 4 + 8 * (T + back),
                "flops": 4 * kv * D * (T + back)}
    if c["kind"] == "read":
        return {"bytes": sum(L) * (kv * D * 2 * 3 + 8) + sum(_blocks(x, c["bs"]) for x in L) * kv * 2, "flops": 2 * kv * D * sum(L)}
    if c["kind"] == "prefill":
        pairs = sum(_seen_of(c, t + 1) for x in L for t in range(x))
        return {"bytes": sum(L) * (heads + kv) * 4 * D, "flops": pairs * heads * 4 * D}
    tokens = sum(_seen_of(c, x) for x in L)
    size = 1 if c["kind"] == "decode8" else 2
    return {"bytes": tokens * kv * D * 2 * size + sum(_blocks(_seen_of(c, x), c["bs"]) for x in L) * (4 + 2 * kv * (2 - size))
            + c["n"] * heads * 4 * D, "flops": tokens * heads * 4 * D}


# -- the definition in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    return {"write": _exact_write, "read": _exact_read, "decode8": _exact_decode, "window": _exact_decode,
            "prefill": _exact_prefill}[c["kind"]](s, c)


def _grid(code):
    """Every value of a code, ascending, in float64."""
    if code == "int8":
        return torch.arange(-127, 128, dtype=torch.float64, device="cuda")
    up = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (x - 10) for x in range(1, 16) for m in range(8)]
    up = torch.tensor(up[:-1], dtype=torch.float64, device="cuda")  # the last pattern is no number
    return torch.cat([-up[1:].flip(0), up])


def _nearest(x, grid):
    """The grid's value nearest to x, of two equally near ones the one whose place from 0 is even."""
    j = torch.searchsorted(grid, x.contiguous()).clamp(1, grid.numel() - 1)
    lo, hi = grid[j - 1], grid[j]
    even = (j - grid.numel() // 2) % 2 == 0
    return torch.where((hi - x < x - lo) | ((hi - x == x - lo) & even), hi, lo)


def _held(s, c, i):
    """The codes' values [blocks, bs, kv, 128] of keys (0) or values (1) and their exponents, in 64 bits."""
    return _values((s["kc"], s["vc"])[i], c["code"]).double(), s["exponents"][..., i].double()


def _exact_write(s, c):
    grid, bs, out = _grid(c["code"]), c["bs"], {}
    exponents = s["exponents"].clone()
    table, start = s["bt"].tolist(), 0
    runs = []  # (block, first offset, first row, rows)
    for b, (L, m) in enumerate(zip(_lengths(c), _new(c))):
        p = L - m
        while p < L:
            upto = min(L, (p // bs + 1) * bs)
            runs.append((table[b][p // bs], p % bs, start + p - (L - m), upto - p))
            p = upto
        start += m
    for i, name in enumerate("kv"):
        held, e = _held(s, c, i)
        x = s[name].double()
        # Runs of one kind together: those with the same first offset and number of rows.
        for off, rows in sorted({(r[1], r[3]) for r in runs}):
            these = [r for r in runs if (r[1], r[3]) == (off, rows)]
            blk = torch.tensor([r[0] for r in these], device="cuda")
            at = torch.tensor([r[2] for r in these], device="cuda")[:, None] + torch.arange(rows, device="cuda")
            y = x[at]                                                          # [runs, rows, kv, D]
            need = torch.log2((y.abs().amax(dim=(1, 3)) / TOP[c["code"]]).clamp(min=2.0 ** LEAST)).ceil()
            e_new = need if off == 0 else torch.maximum(need, e[blk])
            if off:
                old = _nearest(held[blk] * torch.exp2(e[blk] - e_new)[:, None, :, None], grid)
                held[blk] = old
            held[blk, off:off + rows] = _nearest(y * torch.exp2(-e_new)[:, None, :, None], grid)
            e[blk] = e_new
        exponents[..., i] = e.to(torch.int8)
        out[name] = (held * torch.exp2(e)[:, None, :, None]).flatten(0, 1)[s["back"]]
    return dict(out, exponents=exponents)


def _exact_read(s, c):
    rows = [(held * torch.pow(2.0, e)[:, None, :, None]).flatten(0, 1)[s["back"]] for held, e in (_held(s, c, 0), _held(s, c, 1))]
    return dict(k=rows[0], v=rows[1])


def _exact_decode(s, c):
    n, kv, group, bs = c["n"], c["kv"], c["group"], c["bs"]
    out = torch.zeros(n, kv * group, D, dtype=torch.float64, device="cuda")
    for b, L in enumerate(_lengths(c)):
        rows = torch.arange(L, device="cuda")
        if c["window"]:
            rows = rows[(rows < c["sinks"]) | (L - 1 - rows < c["window"])]
        blk, off = s["bt"][b].long()[rows // bs], rows % bs
        if c["kind"] == "decode8":
            k, v = (_values(t[blk, off], c["code"]).double() * 2.0 ** s["exponents"][blk][..., i, None].double()
                    for i, t in enumerate((s["kc"], s["vc"])))
        else:
            k, v = s["kc"][blk, off].double(), s["vc"][blk, off].double()
        for h in range(kv):
            q = s["q"][b, h * group:(h + 1) * group].double()
            p = torch.softmax((q @ k[:, h].t().contiguous()) * SCALE, dim=-1)
            out[b, h * group:(h + 1) * group] = p @ v[:, h]
    return out


def _exact_prefill(s, c):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for a, e in zip(s["cu"], s["cu"][1:]):
        t = torch.arange(e - a, device="cuda")
        sees = (t[None, :] <= t[:, None]) & ((t[None, :] > t[:, None] - c["window"]) | (t[None, :] < c["sinks"]))
        for h in range(out.shape[1]):
            k, v = (x[a:e, h // c["group"]].double() for x in (s["k"], s["v"]))
            score = (s["q"][a:e, h].double() @ k.t().contiguous()) * SCALE
            out[a:e, h] = torch.softmax(torch.where(sees, score, -math.inf), dim=-1) @ v
    return out
