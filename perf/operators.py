"""The cache operators of uncompressed layers, measured: normed queries and keys with their rotation and cache
write, block selection with the decode over the selected blocks, and the decode that sums attention weights
with the eviction that goes by them.

``listed()`` holds the cases that are timed, ``draw(rng)`` gives further cases of the same ranges,
``prepare(case, seed)`` makes what a program holds before the call, ``run(state)`` is one pass through an
operator (its plain form in torch, or, where ``own`` is true, the framework's entry point), ``work(case)``
the bytes and operations the pass cannot do without and ``exact(case, seed)`` the result in float64.

The kinds of case:

- ``norm_rope``: per-head RMS norm of q and k, their rotation, k and v into the paged cache
  (``model_ops.norm_rope_write``);
- ``bounds``: the elementwise least and largest key of the cache blocks that new tokens touched
  (``sparse_decode.update_key_bounds``);
- ``select``: the blocks whose bounds promise the largest scores (``sparse_decode.select_blocks``);
- ``sparse``: one token's attention over selected blocks (``sparse_decode.paged_decode_sparse``);
- ``weighted``: one token's attention over its whole cache, the tokens' weights summed up
  (``evict.paged_decode_weighted``);
- ``evict``: a cache cut to the tokens of the largest summed weights (``evict.evict``).
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
EPS = 1e-6


def listed():
    return [
        # One step of a small batch: 16 tokens' q, k and v, in front of each layer's attention. Latency.
        dict(name="norm_rope_step_16", kind="norm_rope", fmt="bf16", kv=8, group=4, tokens=16, half=False, bs=16, mix=1),
        # A step's prompts, 8191 tokens in all, as many key as query heads; the prefill's fp16 rows too.
        dict(name="norm_rope_prompts_8191", kind="norm_rope", fmt="bf16", kv=32, group=1, tokens=8191, half=True, bs=16,
             mix=2),
        # After one decode step of 64 requests: the bounds of each one's last block. Latency.
        dict(name="bounds_step_64", kind="bounds", fmt="bf16", kv=8, group=4, n=64, lo=512, hi=4096, new=1, bs=16, mix=3),
        # After two long prompts: the bounds of every block of theirs, 32 tokens a block.
        dict(name="bounds_prompts_2x16384", kind="bounds", fmt="fp16", kv=32, group=1, n=2, lo=16384, hi=16384,
             new=16384, bs=32, mix=4),
        # One long session chooses 128 of its 4096 blocks. Latency.
        dict(name="select_1x65536", kind="select", fmt="bf16", kv=8, group=4, n=1, lo=65536, hi=65536, bs=16, keep=128,
             sink=1, recent=2, mix=5),
        # A batch of long sessions of odd lengths.
        dict(name="select_32_ragged", kind="select", fmt="bf16", kv=8, group=4, n=32, lo=4001, hi=32767, bs=16, keep=128,
             sink=1, recent=2, mix=6),
        # The long session's attention over 2048 of its 65536 tokens. Latency.
        dict(name="sparse_1x65536", kind="sparse", fmt="bf16", kv=8, group=4, n=1, lo=65536, hi=65536, bs=16, keep=128,
             sink=1, recent=2, mix=7),
        # The largest: a batch with one key head per query head, 64 blocks of 32 tokens each.
        dict(name="sparse_32_ragged", kind="sparse", fmt="fp16", kv=32, group=1, n=32, lo=1500, hi=16000, bs=32, keep=64,
             sink=1, recent=2, mix=8),
        # One interactive session whose weights are summed up.
        dict(name="weighted_1x4096", kind="weighted", fmt="bf16", kv=32, group=1, n=1, lo=4096, hi=4096, bs=16, mix=9),
        # A serving batch at different points, four query heads a key head.
        dict(name="weighted_24_ragged", kind="weighted", fmt="bf16", kv=8, group=4, n=24, lo=1000, hi=8191, bs=16,
             mix=10),
        # One session over its budget by a few steps: 2176 tokens cut to 2048.
        dict(name="evict_1x2176", kind="evict", fmt="bf16", kv=32, group=1, n=1, lo=2176, hi=2176, bs=16, keep=2048,
             sink=4, recent=256, mix=11),
        # A batch's prompts cut to their budget before decoding.
        dict(name="evict_16_ragged", kind="evict", fmt="fp16", kv=8, group=4, n=16, lo=4097, hi=8192, bs=16, keep=2048,
             sink=4, recent=256, mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges: sizes over their logarithm, odd ones among them."""
    kind = rng.choice(["norm_rope", "norm_rope", "bounds", "select", "select", "sparse", "sparse", "weighted", "weighted",
                       "evict", "evict"])
    c = dict(kind=kind, fmt=rng.choice(["bf16", "fp16"]), kv=rng.choice([1, 2, 4, 5, 8, 8, 32]), bs=rng.choice([16, 32, 64]),
             mix=rng.randrange(1 << 30))
    c["group"] = rng.choice([1, 2, 4, 8]) if c["kv"] < 32 else 1
    if c["kv"] < 8 and rng.random() < 0.4:
        c["group"] = rng.choice([3, 5, 6, 7])
    if kind == "norm_rope":
        c["tokens"] = _log(rng, 1, 8191)
        c["half"] = rng.random() < 0.5 and c["tokens"] > 64
        return c
    c["n"] = _log(rng, 1, 64)
    most = {"bounds": 2 ** 21, "select": 2 ** 24, "sparse": 2 ** 23, "weighted": 2 ** 20, "evict": 2 ** 19}[kind]
    top = min(65536, max(64, most // (c["n"] * c["kv"])))
    c["hi"] = _log(rng, 16, top)
    c["lo"] = c["hi"] if rng.random() < 0.3 else max(1, c["hi"] // rng.choice([2, 4, 8]))
    if kind == "bounds":
        c["new"] = rng.choice([1, _log(rng, 1, c["hi"]), c["hi"]])
    if kind in ("select", "sparse"):
        c["sink"], c["recent"] = rng.choice([0, 1, 2]), rng.choice([1, 2, 4])
        blocks = -(-c["hi"] // c["bs"])
        c["keep"] = c["sink"] + c["recent"] + _log(rng, 1, min(512, max(1, blocks // 2)))
        if kind == "sparse":
            c["keep"] = max(c["sink"] + c["recent"], min(c["keep"], 2 ** 20 // (c["n"] * c["kv"] * c["bs"])))
    if kind == "evict":
        c["sink"], c["recent"] = rng.choice([0, 1, 4]), rng.choice([1, 8, 33])
        c["keep"] = c["sink"] + c["recent"] + _log(rng, 1, max(1, c["hi"] * 7 // 8))
    return c


# -- sizes that a case fixes, whatever the seed of its inputs --------------------------------
def _lengths(c):
    r = random.Random(c["mix"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["n"])]


def _dtype(c):
    return torch.float16 if c["fmt"] == "fp16" else torch.bfloat16


def _blocks(L, bs):
    return -(-L // bs)


# -- inputs -----------------------------------------------------------------------------------
def _gen(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 16 + salt)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=g)


def _keys(g, blocks, c):
    """Keys as a model's: a spread of their own in each channel of a head about a mean of its own."""
    k = _randn(g, blocks, c["bs"], c["kv"], D, dtype=_dtype(c))
    k.mul_(_randn(g, c["kv"], D, std=0.4).exp().to(k.dtype)).add_(_randn(g, c["kv"], D).to(k.dtype))
    return k


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


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt, kv, heads = _dtype(c), c["kv"], c["kv"] * c["group"]
    if c["kind"] == "norm_rope":
        T, bs = c["tokens"], c["bs"]
        qkv = _randn(g, T, (heads + 2 * kv) * D, dtype=dt)
        q, k, v = (t.view(T, -1, D) for t in qkv.split([heads * D, kv * D, kv * D], dim=-1))
        table = 16384
        inv = 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
        ang = torch.arange(table, device="cuda", dtype=torch.float64)[:, None] * inv
        blocks = _blocks(T, bs) + 1
        return dict(c=c, q=q, k=k, v=v, cos_sin=torch.cat([ang.cos(), ang.sin()], dim=-1).to(dt),
                    qw=(1 + _randn(g, D, std=0.3)).to(dt), kw=(1 + _randn(g, D, std=0.3)).to(dt),
                    pos=torch.randint(0, table, (T,), device="cuda", generator=g),
                    slots=torch.randperm(blocks * bs, device="cuda", generator=g)[:T].contiguous(),
                    kc=_randn(g, blocks, bs, kv, D, dtype=dt), vc=_randn(g, blocks, bs, kv, D, dtype=dt))
    L = _lengths(c)
    lens = torch.tensor(L, dtype=torch.int32, device="cuda")
    bt, blocks = _block_table(c, g)
    s = dict(c=c, lens=lens, bt=bt, span=max(L))
    if c["kind"] != "bounds" and c["kind"] != "evict":
        s["q"] = _randn(g, c["n"], heads, D, dtype=dt)
    if c["kind"] == "select":
        x = torch.stack([_keys(g, blocks, dict(c, bs=1)), _keys(g, blocks, dict(c, bs=1))], dim=3)
        s["bounds"] = torch.stack([x.amin(3), x.amax(3)], dim=3).squeeze(1).contiguous()
        return s
    s["kc"] = _keys(g, blocks, c)
    if c["kind"] == "bounds":
        s["bounds"] = torch.zeros(blocks, kv, 2, D, dtype=dt, device="cuda")
        return s
    s["vc"] = _randn(g, blocks, c["bs"], kv, D, dtype=dt)
    if c["kind"] == "sparse":
        s["selected"] = _some_blocks(c, L, g)
    else:
        # Summed weights: a few tokens hold most of it, some have none.
        w = (2.0 * _randn(g, c["n"], kv, max(L))).exp_() * 0.01
        s["weights"] = w * (_randn(g, c["n"], kv, max(L)) > -1.6)
    return s


def _some_blocks(c, L, g):
    """A choice of blocks for each request and head: the first and last ones and random others, ascending."""
    nb = torch.tensor([_blocks(x, c["bs"]) for x in L], device="cuda")[:, None, None]
    j = torch.arange(max(int(nb.max()), c["keep"]), device="cuda")
    r = torch.rand(c["n"], c["kv"], j.numel(), device="cuda", generator=g)
    r = torch.where((j < c["sink"]) | (j >= nb - c["recent"]), r + 1, r).masked_fill(j >= nb, -1)
    at = r.topk(c["keep"], dim=-1).indices
    at = torch.where(at < nb, at, j.numel()).sort(-1).values
    return torch.where(at < j.numel(), at, -1).to(torch.int32).contiguous()


# -- one pass ---------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    return {"norm_rope": _plain_norm_rope, "bounds": _plain_bounds, "select": _plain_select, "sparse": _plain_sparse,
            "weighted": _plain_weighted, "evict": _plain_evict}[s["c"]["kind"]](s)


_modules = None


def _own(s):
    global _modules
    if _modules is None:
        sys.path.insert(0, os.path.join(ROOT, "star-kv-serve_amd"))
        from starkv_serve.kernels import evict, model_ops, sparse_decode
        _modules = model_ops, sparse_decode, evict
    model_ops, sparse_decode, evict = _modules
    c = s["c"]
    if c["kind"] == "norm_rope":
        q, k, k16, v16 = model_ops.norm_rope_write(s["pos"], s["q"], s["k"], s["v"], s["cos_sin"], s["qw"], s["kw"], EPS,
                                                   s["kc"], s["vc"], s["slots"], keep_k=False, half=c["half"])
        return dict(q=q, kc=s["kc"], vc=s["vc"], **(dict(k16=k16, v16=v16) if c["half"] else {}))
    if c["kind"] == "bounds":
        sparse_decode.update_key_bounds(s["kc"], s["bounds"], s["bt"], s["lens"], c["new"])
        return s["bounds"]
    if c["kind"] == "select":
        return sparse_decode.select_blocks(s["q"], s["bounds"], s["bt"], s["lens"], s["span"], c["bs"], c["keep"],
                                           c["sink"], c["recent"])
    if c["kind"] == "sparse":
        return sparse_decode.paged_decode_sparse(s["q"], s["kc"], s["vc"], s["bt"], s["lens"], s["selected"], SCALE)
    if c["kind"] == "weighted":
        out = evict.paged_decode_weighted(s["q"], s["kc"], s["vc"], s["bt"], s["lens"], s["span"], SCALE, s["weights"])
        return dict(out=out, weights=s["weights"])
    lens, weights = evict.evict(s["kc"], s["vc"], s["bt"], s["lens"], s["weights"], c["keep"], c["sink"], c["recent"])
    return dict(kc=s["kc"], vc=s["vc"], lens=lens, weights=weights)


# -- the plain forms --------------------------------------------------------------------------
def _plain_norm_rope(s):
    def rotated(x, w):
        x = x.float()
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
        cos, sin = s["cos_sin"][s["pos"]].float()[:, None, :].chunk(2, dim=-1)
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)

    q, k = rotated(s["q"], s["qw"]).to(s["q"].dtype), rotated(s["k"], s["kw"]).to(s["k"].dtype)
    bs = s["c"]["bs"]
    at = s["slots"] // bs, s["slots"] % bs
    s["kc"][at] = k
    s["vc"][at] = s["v"]
    out = dict(q=q, kc=s["kc"], vc=s["vc"])
    if s["c"]["half"]:
        out.update(k16=k.to(torch.float16), v16=s["v"].to(torch.float16))
    return out


def _plain_bounds(s):
    c = s["c"]
    bs, lens = c["bs"], s["lens"].long()[:, None]
    j = torch.arange(s["bt"].shape[1], device="cuda")
    b, j = ((j >= (lens - c["new"]).clamp(min=0) // bs) & (j * bs < lens)).nonzero(as_tuple=True)
    blocks = s["bt"][b, j].long()
    there = (j[:, None] * bs + torch.arange(bs, device="cuda") < lens[b])[:, :, None, None]
    k = s["kc"][blocks]
    low = k.masked_fill(~there, math.inf).amin(1)
    s["bounds"][blocks] = torch.stack([low, k.masked_fill(~there, -math.inf).amax(1)], dim=2)
    return s["bounds"]


def _plain_select(s):
    c = s["c"]
    n, kv, keep = c["n"], c["kv"], c["keep"]
    # 64 bits: which of two nearly equal blocks is chosen must not depend on the order of a sum.
    q = s["q"].view(n, kv, c["group"], D).double()
    up, down = q.clamp(min=0).sum(2)[:, None], q.clamp(max=0).sum(2)[:, None]
    low, high = s["bounds"][s["bt"].long()].unbind(3)
    score = ((up * high + down * low).sum(-1)).float().transpose(1, 2)
    nb = ((s["lens"].long() + c["bs"] - 1) // c["bs"])[:, None, None]
    j = torch.arange(score.shape[2], device="cuda")
    score = score.masked_fill((j < c["sink"]) | (j >= nb - c["recent"]), math.inf).masked_fill(j >= nb, -math.inf)
    at = score.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    at = torch.where(at < nb, at, 1 << 30).sort(-1).values
    at = torch.where(at < nb, at, -1).to(torch.int32)
    return torch.cat([at, at.new_full((n, kv, keep - at.shape[2]), -1)], dim=-1) if at.shape[2] < keep else at


def _attend(q, k, v, there):
    """(attention of q [n, kv, group, 128] over k, v [n, kv, t, 128] where `there`, its weights), in 32 bits."""
    score = (torch.matmul(q.float(), k.float().transpose(-1, -2).contiguous()) * SCALE)
    score = score.masked_fill(~there[:, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(p, v.float()), p


def _plain_sparse(s):
    c = s["c"]
    n, kv, bs = c["n"], c["kv"], c["bs"]
    sel = s["selected"].long()
    blocks = s["bt"].long()[:, None, :].expand(n, kv, -1).gather(2, sel.clamp(min=0))
    head = torch.arange(kv, device="cuda")[None, :, None]
    k, v = (t.transpose(1, 2)[blocks, head].reshape(n, kv, -1, D) for t in (s["kc"], s["vc"]))
    pos = sel[..., None] * bs + torch.arange(bs, device="cuda")
    there = ((sel[..., None] >= 0) & (pos < s["lens"].long()[:, None, None, None])).reshape(n, kv, -1)
    out, _ = _attend(s["q"].view(n, kv, c["group"], D), k, v, there)
    return out.reshape(n, -1, D).to(s["q"].dtype)


def _plain_weighted(s):
    c = s["c"]
    n, kv, span = c["n"], c["kv"], s["span"]
    k, v = (t[s["bt"].long()].reshape(n, -1, kv, D)[:, :span].transpose(1, 2) for t in (s["kc"], s["vc"]))
    lens = s["lens"].long()[:, None, None]
    j = torch.arange(span, device="cuda")
    out, p = _attend(s["q"].view(n, kv, c["group"], D), k, v, (j < lens).expand(n, kv, span))
    s["weights"].mul_(j != lens - 1).add_(p.sum(2))
    return dict(out=out.reshape(n, -1, D).to(s["q"].dtype), weights=s["weights"])


def _plain_evict(s):
    c = s["c"]
    n, kv, bs, keep, w = c["n"], c["kv"], c["bs"], min(c["keep"], s["span"]), s["weights"]
    lens = s["lens"].long()[:, None, None]
    j = torch.arange(w.shape[2], device="cuda")
    rank = w.masked_fill((j < c["sink"]) | (j >= lens - c["recent"]), math.inf).masked_fill(j >= lens, -math.inf)
    at = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    to = torch.arange(keep, device="cuda").expand(n, kv, keep)
    left = lens.clamp(max=c["keep"])
    b, h, i = (to < left).nonzero(as_tuple=True)
    at = at[b, h, i]
    bt, new = s["bt"].long(), torch.zeros_like(w)
    new[b, h, i] = w[b, h, at]
    src, dst = (bt[b, at // bs], at % bs, h), (bt[b, i // bs], i % bs, h)
    s["kc"][dst] = s["kc"][src]
    s["vc"][dst] = s["vc"][src]
    return dict(kc=s["kc"], vc=s["vc"], lens=left.flatten().to(torch.int32), weights=new)


# -- what a pass cannot do without ------------------------------------------------------------
def work(case):
    c = case
    kv, heads = c["kv"], c["kv"] * c["group"]
    if c["kind"] == "norm_rope":
        rows = c["tokens"] * (heads + 2 * kv)
        moved = 2 * rows + (2 * c["tokens"] * kv if c["half"] else 0)
        return {"bytes": moved * 2 * D + c["tokens"] * (2 * D + 16), "flops": 10 * D * rows}
    L, bs = _lengths(c), c["bs"]
    if c["kind"] == "bounds":
        first = [max(0, x - c["new"]) // bs for x in L]
        tokens, blocks = sum(x - f * bs for x, f in zip(L, first)), sum(_blocks(x, bs) - f for x, f in zip(L, first))
        return {"bytes": kv * 2 * D * (tokens + 2 * blocks), "flops": 2 * kv * D * tokens}
    if c["kind"] == "select":
        blocks = sum(_blocks(x, bs) for x in L)
        return {"bytes": blocks * (kv * 4 * D + 4) + c["n"] * (heads * 2 * D + kv * c["keep"] * 4),
                "flops": blocks * kv * 4 * D}
    if c["kind"] in ("sparse", "weighted"):
        tokens = sum(min(x, c["keep"] * bs) if c["kind"] == "sparse" else x for x in L)
        extra = c["n"] * c["keep"] * 4 if c["kind"] == "sparse" else tokens * 8
        return {"bytes": tokens * kv * 4 * D + extra * kv + c["n"] * heads * 4 * D, "flops": tokens * heads * 4 * D}
    moved = sum(c["keep"] - c["sink"] if x > c["keep"] else 0 for x in L)
    return {"bytes": kv * (sum(L) * 4 + sum(min(x, c["keep"]) for x in L) * 4 + moved * 8 * D), "flops": kv * sum(L)}


# -- the definition in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    return {"norm_rope": _exact_norm_rope, "bounds": _exact_bounds, "select": _exact_select, "sparse": _exact_attention,
            "weighted": _exact_attention, "evict": _exact_evict}[c["kind"]](s, c)


def _exact_norm_rope(s, c):
    bs, T = c["bs"], c["tokens"]
    angle = s["cos_sin"].double()[s["pos"]]

    def unit(x, w):
        x = x.double()
        norm = torch.sqrt((x * x).sum(-1) / D + EPS)
        x = torch.view_as_complex(torch.stack(torch.split(x * w.double() / norm[..., None], D // 2, dim=-1), dim=-1).contiguous())
        turn = torch.complex(angle[:, :D // 2].contiguous(), angle[:, D // 2:].contiguous())
        x = x * turn[:, None, :]
        return torch.cat([x.real, x.imag], dim=-1)

    q, k = unit(s["q"], s["qw"]), unit(s["k"], s["kw"])
    kc, vc = s["kc"].double().flatten(0, 1), s["vc"].double().flatten(0, 1)
    kc[s["slots"]], vc[s["slots"]] = k, s["v"].double()
    out = dict(q=q, kc=kc.view(s["kc"].shape), vc=vc.view(s["vc"].shape))
    if c["half"]:
        out.update(k16=k, v16=s["v"].double())
    return out


def _exact_bounds(s, c):
    bounds, bs, table = s["bounds"].double(), c["bs"], s["bt"].tolist()
    for b, L in enumerate(_lengths(c)):
        first = max(0, L - c["new"]) // bs
        whole = torch.tensor(table[b][first:L // bs], dtype=torch.long, device="cuda")
        if whole.numel():
            k = s["kc"][whole].double()
            bounds[whole, :, 0], bounds[whole, :, 1] = k.min(1).values, k.max(1).values
        if L % bs:
            k = s["kc"][table[b][L // bs], :L % bs].double()
            bounds[table[b][L // bs], :, 0], bounds[table[b][L // bs], :, 1] = k.min(0).values, k.max(0).values
    return bounds


def _exact_select(s, c):
    n, kv, keep = c["n"], c["kv"], c["keep"]
    out = torch.full((n, kv, keep), -1, dtype=torch.int32)
    q = s["q"].view(n, kv, c["group"], D).double()
    for b, L in enumerate(_lengths(c)):
        nb = _blocks(L, c["bs"])
        near = s["bounds"][s["bt"][b, :nb].long()].double()                    # [nb, kv, 2, D]
        score = torch.zeros(nb, kv, dtype=torch.float64, device="cuda")
        for g in range(c["group"]):
            score += (q[b, None, :, g, None, :] * near).amax(2).sum(-1)
        score = score.float().cpu()
        for h in range(kv):
            must = [j for j in range(nb) if j < c["sink"] or j >= nb - c["recent"]]
            rest = sorted((j for j in range(c["sink"], nb - c["recent"])), key=lambda j: (-score[j, h].item(), j))
            chosen = sorted((must + rest)[:keep])
            out[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out.cuda()


def _exact_attention(s, c):
    n, kv, group, bs = c["n"], c["kv"], c["group"], c["bs"]
    out = torch.zeros(n, kv * group, D, dtype=torch.float64, device="cuda")
    weights = s["weights"].double() if c["kind"] == "weighted" else None
    for b, L in enumerate(_lengths(c)):
        rows = torch.arange(L, device="cuda")
        for h in range(kv):
            if c["kind"] == "sparse":
                chosen = s["selected"][b, h].long()
                mark = torch.zeros(_blocks(L, bs), dtype=torch.bool, device="cuda")
                mark[chosen[chosen >= 0]] = True
                rows = mark.repeat_interleave(bs)[:L].nonzero().flatten()
            at = s["bt"][b].long()[rows // bs], rows % bs
            k, v = s["kc"][at[0], at[1], h].double(), s["vc"][at[0], at[1], h].double()
            q = s["q"][b, h * group:(h + 1) * group].double()
            p = torch.softmax((q @ k.t().contiguous()) * SCALE, dim=-1)
            out[b, h * group:(h + 1) * group] = p @ v
            if weights is not None:
                weights[b, h, L - 1] = 0
                weights[b, h, :L] += p.sum(0)
    return out if weights is None else dict(out=out, weights=weights)


def _exact_evict(s, c):
    kc, vc, new = s["kc"].double(), s["vc"].double(), torch.zeros_like(s["weights"], dtype=torch.float64)
    lens = []
    for b, L in enumerate(_lengths(c)):
        left = min(L, c["keep"])
        lens.append(left)
        table = s["bt"][b].long()
        for h in range(c["kv"]):
            w = s["weights"][b, h, :L].double()
            kept = torch.arange(L, device="cuda")
            if L > c["keep"]:
                middle = kept[c["sink"]:L - c["recent"]]
                by = torch.argsort(w[middle], descending=True, stable=True)[:c["keep"] - c["sink"] - c["recent"]]
                kept = torch.cat([kept[:c["sink"]], middle[by].sort().values, kept[L - c["recent"]:]])
            to = torch.arange(left, device="cuda")
            new[b, h, :left] = w[kept]
            for t in (kc, vc):
                t[table[to // c["bs"]], to % c["bs"], h] = t[table[kept // c["bs"]], kept % c["bs"], h]
    return dict(kc=kc, vc=vc, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), weights=new)
