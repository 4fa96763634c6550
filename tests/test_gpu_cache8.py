"""8-bit caches on the GPU: the quantising write against its definition, value for value, rows read back, and one token's
attention over them against float64.

Writes and reads are exact: scales are powers of two, so a code is one rounding of an exact quotient.

The attention's tolerance, u = finfo(type).eps / 2 of the result's type, e = 2^-24 that of fp32, K and V the cache's
values, s the scores (natural units), c the exponents of the values' blocks, t the tokens:
- a score: 128 exact products summed in fp32 in any order, the scales exact but for scale log2(e) and the argument:
  ds <= 132 e scale sum |q K|. A bf16 query in fp16 is exact above 2^-28 of its row's largest, below off by 2^-39 of
  that: 2^-39 scale max|q| sum |K|.
- a weight: 2 ds (its own score's and the sum's), the exponentials' arguments, differences of scores and references
  that are rounded: 8 e (max |s| / ln 2 + max |c| + 24), and the two fp16 values that hold it, 2^-22.
- fp16 ends at 2^-24: a weight of a value, relative to the reference of s + c, is off by 2^-25 where the largest is at
  least 2^7: t 2^-32 max_t (p 2^c) max |code|.
- the sums of t terms in fp32: (t + 16) e sum p |V|. The result's rounding u |out|, fp16 below its range 2^-25.
"""
import math

import pytest
import torch

from cache8_plain import D, E, SCALE, Plain8, attention, visible
from starkv_serve.kernels.cache8 import Cache8, paged_decode_8, read_kv8, write_kv8
from starkv_serve.kernels.window import Window

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
I8, F8 = torch.int8, torch.float8_e4m3fn


def some_cache(nb, bs, H, dtype, cuda, g, layout="heads"):
    """A cache with codes and exponents everywhere."""
    if layout == "heads":
        c = Cache8.zeros(nb, bs, H, dtype, cuda)
    elif layout == "tokens":
        k, v = (torch.zeros(nb, bs, H, D, dtype=I8, device=cuda).view(dtype) for _ in range(2))
        c = Cache8(k, v, torch.zeros(nb, H, 2, dtype=I8, device=cuda))
    else:  # one tensor of a block's keys and values, exponents inside wider rows
        kv = torch.zeros(nb, 2, bs, H, D, dtype=I8, device=cuda).view(dtype)
        c = Cache8(kv[:, 0], kv[:, 1], torch.zeros(nb, H + 3, 6, dtype=I8, device=cuda)[:, 1:H + 1, 2:4])
    for t in (c.k, c.v):
        x = (torch.randn(t.shape, generator=g) * 40).clamp(-127, 127)
        t.copy_((x.round() if dtype == I8 else x).to(dtype))
    c.exponents.copy_(torch.randint(-9, -3, c.exponents.shape, generator=g))
    return c


def rows(n, H, dt, cuda, g, strided=True):
    x = torch.randn(n, 2, H + 1, D, generator=g).to(dt).to(cuda)
    if not strided:
        return x[:, 0, :H].contiguous(), x[:, 1, :H].contiguous()
    return x[:, 0, :H], x[:, 1, 1:]


# -- writes -----------------------------------------------------------------------------------
@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dt,bs,H,n,layout,bits", [(BF16, 16, 2, 1, "heads", 64), (F16, 32, 5, 9, "tokens", 32),
                                                   (BF16, 16, 8, 64, "pairs", 64), (F16, 1024, 1, 256, "heads", 32)])
def test_write_few(cuda, code, dt, bs, H, n, layout, bits):
    """Decode steps' writes: scattered slots, several tokens of a block, padding."""
    g = torch.Generator().manual_seed(n)
    nb = max(4, 2 * n // bs)
    c = some_cache(nb, bs, H, code, cuda, g, layout)
    want = Plain8(c)
    k, v = rows(n, H, dt, cuda, g)
    k.mul_(torch.exp2(torch.randint(-6, 7, (n, 1, 1), generator=g).float()).to(dt).to(cuda))  # some raise their block's exponent
    slots = torch.randperm(nb * bs, generator=g)[:n]
    slots[torch.rand(n, generator=g) < 0.1] = -1
    if n > 2:
        slots[1] = nb * bs + 3
    slots = slots.to(torch.int64 if bits == 64 else torch.int32).to(cuda)
    write_kv8(k, v, c, slots)
    want.write(k, v, slots)
    assert want.same(c)
    write_kv8(k, v, c, slots)  # again: nothing changes
    assert want.same(c)


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dt,bs,H,lens,order,layout", [(BF16, 16, 4, [257], "runs", "heads"), (F16, 32, 3, [300, 1, 45, 16], "runs", "tokens"),
                                                       (BF16, 64, 2, [200, 333], "shuffled", "pairs"),
                                                       (F16, 16, 1, [17, 400], "reversed", "heads"), (BF16, 1024, 1, [1500], "runs", "heads"),
                                                       (BF16, 16, 40, [261], "shuffled", "heads"),
                                                       (BF16, 16, 4, [1025], "runs", "heads"), (F16, 32, 3, [1100, 1, 45, 16], "runs", "tokens"),
                                                       (BF16, 64, 2, [600, 777], "shuffled", "pairs"), (F16, 16, 1, [17, 1400], "reversed", "heads"),
                                                       (BF16, 1024, 1, [2500], "shuffled", "heads"), (BF16, 16, 40, [1061], "shuffled", "heads"),
                                                       (F16, 128, 5, [1024], "runs", "heads"), (BF16, 16, 17, [1003, 20], "runs", "heads"),
                                                       (BF16, 32, 9, [40, 18, 33], "runs", "heads"), (F16, 64, 3, [50, 29, 77], "runs", "heads"),
                                                       (BF16, 32, 7, [1040, 30], "shuffled", "pairs"), (F16, 64, 5, [65, 1100], "reversed", "tokens"),
                                                       (BF16, 256, 3, [100, 500], "runs", "heads"), (F16, 512, 2, [1200, 90], "shuffled", "heads"),
                                                       (BF16, 64, 40, [2100, 30], "runs", "heads"), (F16, 64, 17, [300, 1800, 90], "shuffled", "heads"),
                                                       (BF16, 32, 33, [2070], "reversed", "pairs"), (F16, 256, 20, [1000, 45, 1100], "runs", "tokens")])
def test_write_prompts(cuda, code, dt, bs, H, lens, order, layout):
    """Whole prompts and continued ones, in any order of tokens."""
    g = torch.Generator().manual_seed(sum(lens))
    need = [-(-L // bs) + 1 for L in lens]
    nb = sum(need) + 2
    c = some_cache(nb, bs, H, code, cuda, g, layout)
    want = Plain8(c)
    perm = torch.randperm(nb, generator=g).tolist()
    slots, o = [], 0
    for i, L in enumerate(lens):
        first = 0 if i % 2 == 0 else 5  # every second one goes on behind 5 tokens of its first block
        slots += [perm[o + p // bs] * bs + p % bs for p in range(first, first + L)]
        o += need[i]
    slots = torch.tensor(slots)
    n = slots.numel()
    if order == "shuffled":
        slots = slots[torch.randperm(n, generator=g)]
        slots[::50] = -1
    elif order == "reversed":
        slots = slots.flip(0)
    k, v = rows(n, H, dt, cuda, g)
    v[n // 2].mul_(30)
    write_kv8(k, v, c, slots.to(cuda))
    want.write(k, v, slots)
    assert want.same(c)


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dt,bs,H,n,layout", [(BF16, 16, 8, 700, "heads"), (F16, 64, 3, 1024, "pairs"), (BF16, 16, 19, 1030, "tokens"), (F16, 32, 1, 2050, "heads")])
def test_write_many_steps(cuda, code, dt, bs, H, n, layout):
    """A token each for many requests, twice: some blocks begin, some exponents grow."""
    g = torch.Generator().manual_seed(n)
    nb = n + 7
    c = some_cache(nb, bs, H, code, cuda, g, layout)
    want = Plain8(c)
    blocks = torch.randperm(nb, generator=g)[:n]
    for _ in range(2):
        k, v = rows(n, H, dt, cuda, g)
        k.mul_(torch.exp2(torch.randint(-6, 7, (n, 1, 1), generator=g).float()).to(dt).to(cuda))
        slots = blocks * bs + torch.randint(0, bs, (n,), generator=g)
        slots[torch.rand(n, generator=g) < 0.05] = -1
        write_kv8(k, v, c, slots.to(cuda))
        want.write(k, v, slots)
        assert want.same(c)


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("bs,n", [(32, 20), (64, 40), (128, 90), (1024, 700), (64, 1060), (512, 1400)])
def test_write_into_half_full_blocks(cuda, code, bs, n):
    """Chunks of a prompt behind others of the same blocks, larger and smaller ones, so that codes that are there are rounded
    again by several waves; an infinite value in the last."""
    g = torch.Generator().manual_seed(n)
    H, nb = 6, -(-4 * n // bs) + 2
    c = some_cache(nb, bs, H, code, cuda, g)
    want = Plain8(c)
    for i, scale in enumerate((1.0, 2.0 ** 5, 2.0 ** -9, 2.0 ** 7)):
        k, v = rows(n, H, BF16, cuda, g)
        k.mul_(scale)
        v.mul_(2.0 ** i)
        if i == 3:
            v[n // 2, 4, 3] = math.inf
        slots = bs + i * n + torch.arange(n)
        write_kv8(k, v, c, slots.to(cuda))
        want.write(k, v, slots)
        assert want.same(c), i


@pytest.mark.parametrize("n", [3, 300, 1100])
@pytest.mark.parametrize("code,top", [(I8, 127), (F8, 448)])
def test_write_exponents(cuda, code, top, n):
    """Values at the borders of an exponent, zeros, the types' smallest and largest values, and halves between codes."""
    g = torch.Generator().manual_seed(7)
    bs = 16
    for dt in (BF16, F16):
        big = torch.finfo(dt).max
        tiny = 2.0 ** -133 if dt == BF16 else 2.0 ** -24
        edge = [0.0, -0.0, tiny, -tiny, float(top), top * 2.0 ** -9, top * 1.0078125, -top * 4.0, 2.0 ** -3, 255.0, 1.75, big, -big, 0.5, 1.5,
                2.5, 2.0 ** -100 if dt == BF16 else 2.0 ** -14]
        H = len(edge)
        nb = max(24, n // bs + 9)
        c = some_cache(nb, bs, H, code, cuda, g)
        c.exponents[5:9] = -126
        want = Plain8(c)
        k = (torch.randint(-4, 5, (n, H, D), generator=g).double() / 4 * torch.tensor(edge, dtype=torch.float64)[None, :, None]).to(dt)
        k[0, :, 0] = torch.tensor(edge).to(dt)
        v = k.flip(1).contiguous()
        slots = torch.randperm(nb * bs, generator=g)[:n]
        write_kv8(k.to(cuda), v.to(cuda), c, slots.to(cuda))
        want.write(k, v, slots)
        assert want.same(c)


@pytest.mark.parametrize("n", [6, 290, 1111])
@pytest.mark.parametrize("code", [I8, F8])
def test_write_not_finite(cuda, code, n):
    """Infinities and NaN make the head's block NaN, other heads and blocks not; a new first token ends that."""
    g = torch.Generator().manual_seed(n)
    bs, H, nb = 16, 3, max(24, n // 16 + 6)
    c = some_cache(nb, bs, H, code, cuda, g)
    want = Plain8(c)
    k, v = rows(n, H, BF16, cuda, g)
    k[0, 1, 5], v[1, 0, 127], v[2, 2, 0] = math.inf, math.nan, -math.inf
    slots = torch.tensor([16 + 3, 32, 48 + 15] + list(range(64, 64 + n - 3)))
    write_kv8(k, v, c, slots.to(cuda))
    want.write(k, v, slots)
    assert want.same(c) and int((c.exponents == -128).sum()) == 3
    got = read_kv8(c, slots.to(cuda), F32)
    assert got[0][0, 1].isnan().all() and got[1][1, 0].isnan().all() and got[0][1].isfinite().all()
    more, _ = rows(n, H, BF16, cuda, g)
    slots2 = torch.tensor([16 + 4, 32, 48] + list(range(64, 64 + n - 3)))
    write_kv8(more, more, c, slots2.to(cuda))
    want.write(more, more, slots2)
    assert want.same(c) and int((c.exponents == -128).sum()) == 1


@pytest.mark.parametrize("n", [5, 400, 1200])
def test_write_same_slot_twice(cuda, n):
    """Two tokens with one slot: one of them is there, and the block's other rows are right."""
    g = torch.Generator().manual_seed(n)
    nb = max(32, n // 16 + 8)
    c = some_cache(nb, 16, 2, I8, cuda, g)
    one, other = Plain8(c), Plain8(c)
    k, v = rows(n, 2, BF16, cuda, g)
    slots = torch.randperm(nb * 16, generator=g)[:n]
    slots[3] = slots[0]
    write_kv8(k, v, c, slots.to(cuda))
    keep = torch.ones(n, dtype=torch.bool)
    keep[0] = False
    one.write(k[keep.to(cuda)], v[keep.to(cuda)], slots[keep])
    keep[0], keep[3] = True, False
    other.write(k[keep.to(cuda)], v[keep.to(cuda)], slots[keep])
    assert one.same(c) or other.same(c)


def test_steps_equal_any_grouping(cuda):
    """Requests' steps one by one and together give the same cache."""
    g = torch.Generator().manual_seed(3)
    n, H, bs, nb = 12, 4, 16, 14
    a = some_cache(nb, bs, H, F8, cuda, g)
    b = Cache8(a.k.clone(), a.v.clone(), a.exponents.clone())
    base = (torch.randperm(nb, generator=g)[:n] * bs).to(cuda)
    for step in range(20):
        k, v = rows(n, H, BF16, cuda, g)
        at = base + step % bs
        write_kv8(k, v, a, at)
        for i in range(0, n, 5):
            write_kv8(k[i:i + 5], v[i:i + 5], b, at[i:i + 5])
    assert all(torch.equal(x.view(I8), y.view(I8)) for x, y in zip(a.tensors, b.tensors))


# -- rows back --------------------------------------------------------------------------------
@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dt,H,layout", [(BF16, 3, "heads"), (F16, 8, "tokens"), (F32, 1, "pairs")])
def test_read(cuda, code, dt, H, layout):
    g = torch.Generator().manual_seed(H)
    c = some_cache(9, 32, H, code, cuda, g, layout)
    c.exponents[2, 0] = torch.tensor([-126, 20], dtype=I8)
    c.exponents[3, H - 1, 1] = -128
    want = Plain8(c)
    for n in (0, 1, 77, 9 * 32):
        slots = torch.randperm(9 * 32, generator=g)[:n]
        if n > 1:
            slots[0], slots[n // 2] = -1, 9 * 32
        got = read_kv8(c, slots.to(cuda).to(torch.int32 if n == 77 else torch.int64), dt)
        for z in range(2):
            assert got[z].shape == (n, H, D) and got[z].dtype == dt
            assert torch.equal(got[z].cpu().double().nan_to_num(7.0), want.rows(z, slots).to(dt).double().nan_to_num(7.0))


def test_read_returns_what_was_written(cuda):
    """Values that codes hold come back as they were."""
    g = torch.Generator().manual_seed(1)
    for code, top in ((I8, 127), (F8, 448)):
        c = Cache8.zeros(4, 16, 2, code, cuda)
        x = torch.randint(-top, top + 1, (64, 2, D), generator=g).double()
        x = (x if code == I8 else x.to(F8).double()) * 2.0 ** -5
        x[:, :, 0] = top * 2.0 ** -5
        slots = torch.arange(64, device=cuda)
        write_kv8(x.to(F16).to(cuda), x.flip(0).to(F16).to(cuda), c, slots)
        k, v = read_kv8(c, slots, F16)
        assert torch.equal(k.cpu().double(), x) and torch.equal(v.cpu().double(), x.flip(0))


# -- the decode -------------------------------------------------------------------------------
def session(lens, H, bs, code, cuda, g, layout="heads", spare=2, window=None):
    """(cache, block table, lengths): every row that no request has is NaN (e4m3) or the least code, every block that none sees
    has exponents of NaN and is -1 in the table."""
    need = [-(-L // bs) for L in lens]
    nb = max(1, sum(need)) + spare
    c = some_cache(nb, bs, H, code, cuda, g, layout)
    k, v = c.k.cpu(), c.v.cpu()
    perm = torch.randperm(nb, generator=g).tolist()
    bt = torch.full((len(lens), max(max(need), 1) + 1), -1, dtype=torch.int32)
    ex = torch.full(c.exponents.shape, -128, dtype=I8)
    bad = -128 if code == I8 else 127
    kb, vb = k.view(I8).clone().fill_(bad), v.view(I8).clone().fill_(bad)
    o = 0
    for b, L in enumerate(lens):
        seen = {s // bs for s in visible(L, window)}
        for j in range(need[b]):
            blk = perm[o + j]
            rows_ = min(bs, L - j * bs)
            kb[blk, :rows_], vb[blk, :rows_] = k.view(I8)[blk, :rows_], v.view(I8)[blk, :rows_]
            if j in seen:
                bt[b, j] = blk
                ex[blk] = c.exponents[blk].cpu()
        o += need[b]
    c.k.view(I8).copy_(kb)
    c.v.view(I8).copy_(vb)
    c.exponents.copy_(ex)
    return c, bt.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)


def close(got, q, c, bt, lens, window, scale=SCALE, what=""):
    plain, u = Plain8(c), torch.finfo(q.dtype).eps / 2
    table, H = bt.cpu().long(), c.k.shape[2]
    G = q.shape[1] // H
    qc = q.cpu().double()
    for b, L in enumerate(lens):
        places = visible(L, window)
        if not places:
            assert (got[b] == 0).all(), what
            continue
        at = torch.tensor(places)
        slots = table[b, at // plain.bs] * plain.bs + at % plain.bs
        K, V = plain.rows(0, slots), plain.rows(1, slots)
        ev = plain.exponents[slots // plain.bs, :, 1].double()
        codes = plain.held[1][slots // plain.bs, slots % plain.bs]
        for h in range(H):
            x = qc[b, h * G:(h + 1) * G]
            out, mass, ds, most = attention(x, K[:, h], V[:, h], scale)
            if q.dtype == BF16:
                ds += 2.0 ** -39 * abs(scale) * x.abs().max().item() * K[:, h].abs().sum(-1).max().item()
            t = len(places)
            p = torch.softmax(x @ K[:, h].t() * scale, dim=-1)
            tol = (mass * (2 * ds + 8 * E * (most / math.log(2) + ev[:, h].abs().max() + 24) + 2.0 ** -22 + (t + 16) * E)
                   + t * 2.0 ** -32 * (p * torch.exp2(ev[:, h])).max() * codes[:, h].abs().max() + u * out.abs() * 1.01)
            if q.dtype == F16:
                tol = tol + 2.0 ** -25
            y = got[b, h * G:(h + 1) * G].double().cpu()
            assert y.isfinite().all(), (what, b, h)
            off = ((y - out).abs() - tol).max().item()
            assert off <= 0, (what, b, h, off)


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("dt,H,G,bs,lens,layout", [
    (BF16, 2, 4, 16, [1, 16, 17, 300, 0], "heads"), (F16, 1, 1, 32, [513], "tokens"), (BF16, 3, 8, 64, [65, 1000], "pairs"),
    (F16, 2, 16, 16, [40, 5, 333], "heads"), (BF16, 1, 9, 16, [129], "heads"), (F16, 5, 3, 16, [2000, 31], "heads"),
    (BF16, 1, 2, 1024, [1023, 2050], "heads"), (BF16, 40, 1, 16, [100] * 30, "heads"), (BF16, 1, 1, 16, [9000], "heads")])
def test_decode(cuda, code, dt, H, G, bs, lens, layout):
    g = torch.Generator().manual_seed(sum(lens) + G)
    c, bt, sl = session(lens, H, bs, code, cuda, g, layout)
    q = torch.randn(len(lens), 2, H * G, D, generator=g).to(dt).to(cuda)[:, 1]
    close(paged_decode_8(q, c, bt, sl, max(lens), SCALE), q, c, bt, lens, None)
    # a longer span, as in a captured step, and lengths in 64 bits
    close(paged_decode_8(q, c, bt, sl.long(), 1 << 20, SCALE), q, c, bt, lens, None)


@pytest.mark.parametrize("size,sinks", [(1, 0), (1, 1), (15, 0), (16, 4), (17, 16), (33, 17), (100, 40), (64, 0), (1000, 300), (5000, 4)])
def test_decode_through_a_window(cuda, size, sinks):
    g = torch.Generator().manual_seed(size + sinks)
    w = Window(size, sinks)
    for code, dt, H, G, bs in ((I8, BF16, 2, 4, 16), (F8, F16, 1, 12, 32)):
        lens = [0, 1, 15, 16, 17, 64, 100, 129, 400, 1111]
        c, bt, sl = session(lens, H, bs, code, cuda, g, window=w)
        q = torch.randn(len(lens), H * G, D, generator=g).to(dt).to(cuda)
        close(paged_decode_8(q, c, bt, sl, max(lens), SCALE, window=w), q, c, bt, lens, w, what=(code, dt))


@pytest.mark.parametrize("n,H,G,most", [(65, 1, 2, 40), (200, 2, 1, 300), (131, 40, 1, 33), (300, 1, 16, 17), (24, 5, 1, 3), (200, 8, 2, 60),
                                        (64, 32, 1, 100), (300, 2, 4, 170), (4200, 1, 1, 20)])
def test_decode_of_many_requests(cuda, n, H, G, most):
    """More requests than a wave looks at, none among them with tokens or all; ranges that hold many and that cut some."""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, most + 1, (n,), generator=g)
    lens[torch.rand(n, generator=g) < 0.3] = 0
    lens[:3], lens[-2:] = 0, 0
    lens[n // 2] = 40 * most
    lens = lens.tolist()
    c, bt, sl = session(lens, H, 16, I8, cuda, g)
    q = torch.randn(n, H * G, D, generator=g).to(BF16).to(cuda)
    got = paged_decode_8(q, c, bt, sl, max(lens), SCALE)
    close(got, q, c, bt, lens, None)
    assert torch.equal(got, paged_decode_8(q, c, bt, sl, 1 << 20, SCALE))
    # any order of requests: each one's result is its own (ranges cut others, so sums may be joined elsewhere)
    back = torch.randperm(n, generator=g)
    close(paged_decode_8(q[back.to(cuda)], c, bt[back.to(cuda)], sl[back.to(cuda)], max(lens), SCALE), q[back.to(cuda)], c, bt[back.to(cuda)],
          [lens[i] for i in back], None)
    assert (paged_decode_8(q, c, bt, sl * 0, 1 << 20, SCALE) == 0).all()


@pytest.mark.parametrize("G", [2, 9])
@pytest.mark.parametrize("L", [1, 100, 257, 700, 2500, 20000])
def test_decode_of_one_request(cuda, L, G):
    """Few and many parts of one request, joined by as many waves as its longest length asks for."""
    g = torch.Generator().manual_seed(L)
    c, bt, sl = session([L], 1, 16, F8, cuda, g)
    q = torch.randn(1, G, D, generator=g).to(F16).to(cuda)
    for span in (L, 1 << 20):
        close(paged_decode_8(q, c, bt, sl, span, SCALE), q, c, bt, [L], None)
    two = paged_decode_8(q.repeat(2, 1, 1), c, bt.repeat(2, 1), torch.cat([sl * 0, sl]), 1 << 20, SCALE)
    assert (two[0] == 0).all()
    close(two[1:], q, c, bt, [L], None)


def test_decode_of_more_heads_than_workgroups(cuda):
    """One range for all pages: no partials, and rows without tokens written with the others."""
    g = torch.Generator().manual_seed(20)
    lens, H = [30, 0, 5], 600
    c, bt, sl = session(lens, H, 16, F8, cuda, g)
    q = torch.randn(3, H, D, generator=g).to(F16).to(cuda)
    close(paged_decode_8(q, c, bt, sl, 64, SCALE), q, c, bt, lens, None)


@pytest.mark.parametrize("n", [400, 1100])
def test_calls_on_two_streams(cuda, n):
    """Writes, reads and decodes of two caches at once, each on a stream of its own."""
    g = torch.Generator().manual_seed(21)
    H, nb, steps = 4, max(64, n // 16 + 5), 20
    jobs = []
    for code in (I8, F8):
        c = some_cache(nb, 16, H, code, cuda, g)
        jobs.append(dict(c=c, plain=Plain8(c), k=rows(n, H, BF16, cuda, g), slots=torch.randperm(nb * 16, generator=g)[:n].to(cuda),
                         q=torch.randn(3, 8, D, generator=g).to(BF16).to(cuda), bt=torch.randperm(64, generator=g)[:60].view(3, 20).int().to(cuda),
                         sl=torch.tensor([320, 17, 200], device=cuda).int(), stream=torch.cuda.Stream(), got=[]))
    torch.cuda.synchronize()
    for _ in range(steps):
        for j in jobs:
            with torch.cuda.stream(j["stream"]):
                write_kv8(*j["k"], j["c"], j["slots"])
                j["got"].append((paged_decode_8(j["q"], j["c"], j["bt"], j["sl"], 320, SCALE), read_kv8(j["c"], j["slots"])[0]))
    torch.cuda.synchronize()
    for j in jobs:
        j["plain"].write(*j["k"], j["slots"].cpu())
        assert j["plain"].same(j["c"])
        first, back = j["got"][0]
        close(first, j["q"], j["c"], j["bt"], [320, 17, 200], None)
        assert all(torch.equal(first, x) and torch.equal(back, y) for x, y in j["got"])


def test_decode_cuts_lengths_and_leaves_bad_blocks_out(cuda):
    g = torch.Generator().manual_seed(5)
    c, bt, sl = session([200, 300], 2, 16, I8, cuda, g)
    q = torch.randn(2, 4, D, generator=g).to(BF16).to(cuda)
    close(paged_decode_8(q, c, bt, sl, 130, SCALE), q, c, bt, [130, 130], None)
    assert torch.equal(paged_decode_8(q, c, bt, torch.tensor([-3, 1 << 30], device=cuda), 10 ** 6, SCALE)[0], torch.zeros_like(q[0]))
    # a block outside the cache holds no tokens: the same as the other request's without them
    bad = bt.clone()
    bad[0, 3], bad[0, 7] = 10 ** 6, -5
    got = paged_decode_8(q, c, bad, sl, 300, SCALE)
    left = torch.cat([bt[0, :3], bt[0, 4:7], bt[0, 8:13]])[None]
    close(got[:1], q[:1], c, left, [200 - 32], None)


def test_decode_of_unlike_exponents(cuda):
    """First tokens of large weight and tiny values among others of large ones, and the other way round; values near the types'
    ends: what a token contributes keeps its bits."""
    g = torch.Generator().manual_seed(11)
    for code in (I8, F8):
        for e_first, e_rest, boost in ((-60, -5, 60.0), (-5, -60, 60.0), (-100, -100, 0.0), (112, 112, 0.0), (-126, 100, 30.0), (-40, 0, -40.0)):
            lens, H, G = [70, 300], 1, 4
            c, bt, sl = session(lens, H, 16, code, cuda, g)
            q = torch.randn(2, G, D, generator=g).to(BF16).to(cuda)
            c.exponents[..., 1] = e_rest
            for b in range(2):
                c.exponents[int(bt[b, 0]), :, 1] = e_first
                # the first block's keys along the queries' mean: their weights grow or vanish together
                along = q[b].float().mean(0)
                k0 = (along / along.abs().max() * 100).cpu()
                c.k[int(bt[b, 0]), :, 0] = (k0.round() if code == I8 else k0).to(code).to(cuda)
                c.exponents[int(bt[b, 0]), :, 0] = -3
            close(paged_decode_8(q, c, bt, sl, 300, SCALE), q, c, bt, lens, None, what=(code, e_first, e_rest))


def test_decode_where_next_to_no_weight_counts(cuda):
    """A block whose weights are 2^-100 to 2^-400 of the others' and whose values are as much larger, and one whose are not; keys
    and queries at opposite ends of their type."""
    g = torch.Generator().manual_seed(22)
    for code in (I8, F8):
        for e_first, e_rest, key in ((-100, 100, 0), (-126, 110, -1), (-60, 60, -1), (110, -126, 0), (0, 100, 0)):
            lens = [40, 300]
            c, bt, sl = session(lens, 1, 16, code, cuda, g)
            q = torch.randn(2, 1, D, generator=g).to(BF16).to(cuda)
            c.exponents[..., 1] = torch.where(c.exponents[..., 1] == -128, -128, e_rest)
            for b in range(2):
                first = int(bt[b, 0])
                c.exponents[first, :, 1] = e_first
                along = q[b, 0].float() / q[b, 0].float().abs().max() * 100
                c.k[first, :, 0] = (along.round() if code == I8 else along).to(code)
                c.exponents[first, :, 0] = key
            close(paged_decode_8(q, c, bt, sl, 300, SCALE), q, c, bt, lens, None, what=(code, e_first, e_rest, key))
        c, bt, sl = session([200, 50], 2, 16, code, cuda, g)
        for power in (-112, -120, 112, 120):  # scores of an ordinary size all the same
            q = (torch.randn(2, 4, D, generator=g) * 2.0 ** power).to(BF16).to(cuda)
            c.exponents[..., 0] = torch.where(c.exponents[..., 0] == -128, -128, max(-7 - power, -126) if power > 0 else -7 - power)
            close(paged_decode_8(q, c, bt, sl, 200, SCALE), q, c, bt, [200, 50], None, what=(code, power))


def test_decode_of_partials_of_unlike_weights(cuda):
    """Parts of one request, joined from many workgroups, whose weights and whose values differ by 2^150 the other way round: each
    part gives about half of the result."""
    g = torch.Generator().manual_seed(23)
    for code in (I8, F8):
        L = 4096
        c, bt, sl = session([L], 1, 16, code, cuda, g)
        q = torch.zeros(1, 2, D)
        q[..., 0], q[0, 1, 1] = 1.0, 0.5
        q = q.to(F16).to(cuda)
        half = bt[0, :L // 16].long().view(2, -1)
        c.k.view(I8)[half.flatten()] = 0
        score = 104 / SCALE  # natural units: 2^150 between the halves
        e = torch.tensor(100.0, dtype=torch.float64).to(code)
        for b in half[0].tolist():
            c.k[b, :, 0, 0] = e.to(cuda)
        c.exponents[half.flatten(), :, 0] = 0
        c.exponents[half[0], :, 1], c.exponents[half[1], :, 1] = -80, 70
        scale = score * SCALE / 100.0
        got = paged_decode_8(q, c, bt, sl, L, scale)
        close(got, q, c, bt, [L], None, scale, what=code)
        both = [Plain8(c).rows(1, (h.cpu()[:, None] * 16 + torch.arange(16)).flatten())[:, 0].sum(0) for h in half]
        assert both[0].abs().max() * math.exp(104) > 0.01 * both[1].abs().max() and both[1].abs().max() > 0.01 * both[0].abs().max() * math.exp(104)


def test_decode_of_large_and_small_queries(cuda):
    g = torch.Generator().manual_seed(12)
    c, bt, sl = session([100, 100, 100, 100], 1, 16, I8, cuda, g)
    c.exponents[..., 0] = torch.where(c.exponents[..., 0] == -128, -128, -7)
    q = torch.randn(4, 2, D, generator=g)
    q[0] *= 2.0 ** -120
    q[1] *= 2.0 ** 40
    q[2] = 0.0
    q[3, :, ::2] *= 2.0 ** -20
    q = q.to(BF16).to(cuda)
    for b, scale in ((0, 2.0 ** 110), (1, 2.0 ** -45), (2, SCALE), (3, SCALE), (3, -SCALE)):
        got = paged_decode_8(q[b:b + 1], c, bt[b:b + 1], sl[b:b + 1], 100, scale)
        close(got, q[b:b + 1], c, bt[b:b + 1], [100], None, scale, what=(b, scale))


def test_decode_of_blocks_that_are_nan(cuda):
    """An exponent of -128 makes NaN of the rows that see the block, and of them alone."""
    g = torch.Generator().manual_seed(13)
    lens, H, G = [200, 200, 200], 2, 4
    for code in (I8, F8):
        c, bt, sl = session(lens, H, 16, code, cuda, g)
        q = torch.randn(3, H * G, D, generator=g).to(F16).to(cuda)
        before = paged_decode_8(q, c, bt, sl, 200, SCALE)
        c.exponents[bt[0, 5].long(), 0, 0] = -128
        c.exponents[bt[1, 2].long(), 1, 1] = -128
        got = paged_decode_8(q, c, bt, sl, 200, SCALE)
        nan = torch.zeros(3, H * G, D, dtype=torch.bool)
        nan[0, :G], nan[1, G:] = True, True
        assert torch.equal(got.isnan().cpu(), nan)
        assert torch.equal(got[~nan.to(cuda)], before[~nan.to(cuda)])
        w = paged_decode_8(q, c, bt, sl, 200, SCALE, window=Window(40, 16))
        assert w.isfinite().all()


def test_decode_scores_of_minus_infinity(cuda):
    """A query that overflows: tokens whose scores are -inf weigh 0, a row of them alone is NaN."""
    g = torch.Generator().manual_seed(14)
    c, bt, sl = session([400], 1, 16, I8, cuda, g)
    c.k[bt[0].clamp(min=0).long()] = 0
    k = c.k.view(I8)
    for j in range(20):
        k[bt[0, j].long(), :, 0] = -100
    c.exponents[..., 0] = torch.where(c.exponents[..., 0] == -128, -128, 60)
    q = torch.full((1, 2, D), 2.0 ** 60, dtype=BF16, device=cuda)
    q[0, 1] = 1.0
    got = paged_decode_8(q, c, bt, sl, 400, 2.0 ** 10)
    # head 0: scores -100 * 2^60 * 2^60 * 128 * 2^10 = -inf in the first 20 blocks, 0 in the others
    plain = Plain8(c)
    rest = torch.arange(320, 400)
    slots = bt.cpu().long()[0, rest // 16] * 16 + rest % 16
    want = plain.rows(1, slots)[:, 0].mean(0)
    assert (got[0, 0].cpu().double() - want).abs().max() <= 2 * 2.0 ** -8 * want.abs().max()
    k[bt[0, 20:25].long()] = -100
    got = paged_decode_8(q, c, bt, sl, 400, 2.0 ** 10)
    assert got[0, 0].isnan().all()


def test_offsets_past_31_bits(cuda):
    """Blocks at the far end of a cache of more than 2^31 bytes a tensor."""
    nb, bs, H = 70000, 64, 4
    g = torch.Generator().manual_seed(15)
    k = torch.zeros(nb, H, bs, D, dtype=I8, device=cuda).transpose(1, 2)
    v = torch.zeros_like(k, memory_format=torch.preserve_format)
    assert k.stride() == v.stride() and k.numel() > 2 ** 31
    c = Cache8(k, v, torch.full((nb, H, 2), -126, dtype=I8, device=cuda))
    table = torch.tensor([[nb - 1, 3, nb - 2, 40000, nb // 2]], dtype=torch.int32, device=cuda)
    L = 5 * bs - 7
    place = torch.arange(L, device=cuda)
    slots = table[0, place // bs].long() * bs + place % bs
    kk, vv = rows(L, H, BF16, cuda, g, strided=False)
    write_kv8(kk, vv, c, slots)       # through the map
    write_kv8(kk[-9:], vv[-9:], c, slots[-9:])
    small = Cache8(k[table[0].long()], v[table[0].long()], c.exponents[table[0].long()])
    plain = Plain8(small)
    want = Plain8(Cache8.zeros(5, bs, H, I8, "cpu"))
    want.write(kk, vv, torch.arange(L))
    assert want.same(small)
    got = read_kv8(c, slots, BF16)
    assert torch.equal(got[0].cpu().double(), plain.rows(0, torch.arange(L)))
    q = torch.randn(1, 2 * H, D, generator=g).to(BF16).to(cuda)
    sl = torch.tensor([L], device=cuda)
    local = torch.arange(5, dtype=torch.int32, device=cuda)[None]
    out = paged_decode_8(q, c, table, sl, L, SCALE)
    assert torch.equal(out, paged_decode_8(q, small, local, sl, L, SCALE))
    close(out, q, small, local, [L], None)


def test_captured_steps(cuda):
    """A write and its decode captured once, replayed over new inputs with eager work between."""
    g = torch.Generator().manual_seed(16)
    lens, H, G, bs = [30, 100, 64], 2, 4, 16
    c, bt, sl = session([L + 20 for L in lens], H, bs, F8, cuda, g)
    pos = torch.tensor(lens, device=cuda)
    k, v = rows(3, H, BF16, cuda, g, strided=False)
    q = torch.randn(3, H * G, D, generator=g).to(BF16).to(cuda)

    def step():
        slots = bt[torch.arange(3, device=cuda), pos // bs].long() * bs + pos % bs
        write_kv8(k, v, c, slots)
        return paged_decode_8(q, c, bt, (pos + 1).to(torch.int32), 256, SCALE, window=Window(50, 4)), slots

    start = [t.clone() for t in c.tensors]
    step()
    for a, b in zip(c.tensors, start):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, slots = step()
    plain = Plain8(c)
    for i in range(5):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        plain.write(k, v, slots)
        assert plain.same(c)
        eager = paged_decode_8(q, c, bt, (pos + 1).to(torch.int32), 256, SCALE, window=Window(50, 4))
        assert torch.equal(out, eager)
        close(out, q, c, bt, [L + i + 1 for L in lens], Window(50, 4))
        torch.cuda.synchronize()
        pos.add_(1)


@pytest.mark.parametrize("n", [500, 1500])
def test_captured_prompt_writes(cuda, n):
    """A captured write of a prompt's size replays over other slots."""
    g = torch.Generator().manual_seed(17)
    nb = max(64, n // 16 + 9)
    c = some_cache(nb, 16, 2, I8, cuda, g)
    k, v = rows(n, 2, F16, cuda, g, strided=False)
    slots = torch.arange(n, device=cuda)
    plain = Plain8(c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_kv8(k, v, c, slots)
    for i in range(4):
        slots.copy_(torch.randperm(nb * 16, generator=g)[:n])
        k.copy_(torch.randn(k.shape, generator=g) * 2.0 ** i)
        graph.replay()
        plain.write(k, v, slots)
        assert plain.same(c)
        torch.randn(1000, 1000, device=cuda).sum().item()


def test_inputs_written_on_the_callers_stream(cuda):
    """Launches go on the stream that the caller has made current, behind its work."""
    g = torch.Generator().manual_seed(18)
    H, n = 2, 300
    src = some_cache(32, 16, H, F8, cuda, g)
    k0, v0 = rows(n, H, BF16, cuda, g, strided=False)
    q0 = torch.randn(1, 4, D, generator=g).to(BF16).to(cuda)
    slots0 = torch.randperm(32 * 16, generator=g)[:n].to(cuda)
    table, sl = torch.arange(32, dtype=torch.int32, device=cuda)[None], torch.tensor([500], device=cuda)

    def run(c, k, v, q, slots):
        write_kv8(k, v, c, slots)
        write_kv8(k[:3], v[:3], c, slots[:3])
        return [paged_decode_8(q, c, table, sl, 512, SCALE), *read_kv8(c, slots, BF16), *c.tensors]

    def copy(c):
        return Cache8(*(t.clone() for t in c.tensors))

    want = [t.clone() for t in run(copy(src), k0, v0, q0, slots0)]
    c = some_cache(32, 16, H, F8, cuda, g)
    k, v, q, slots = torch.zeros_like(k0), torch.zeros_like(v0), torch.zeros_like(q0), torch.arange(n, device=cuda)
    busy = torch.randn(4096, 4096, device=cuda)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(30):
            busy = busy @ busy * 1e-3
        for a, b in zip((*c.tensors, k, v, q, slots), (*src.tensors, k0, v0, q0, slots0)):
            a.copy_(b)
        got = [t.clone() for t in run(c, k, v, q, slots)]
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a.view(I8) if a.dtype == F8 else a, b.view(I8) if b.dtype == F8 else b)


def test_refusals(cuda):
    """What the operators refuse before a launch."""
    c = Cache8.zeros(4, 16, 2, I8, cuda)
    k = torch.zeros(3, 2, D, dtype=BF16, device=cuda)
    slots = torch.arange(3, device=cuda)
    q, bt, sl = torch.zeros(1, 4, D, dtype=BF16, device=cuda), torch.zeros(1, 4, dtype=torch.int32, device=cuda), torch.ones(1, device=cuda).int()
    with pytest.raises(ValueError, match="slots"):
        write_kv8(k, k, c, slots[:2])
    with pytest.raises(ValueError, match="slots"):
        write_kv8(k, k, c, slots.float())
    with pytest.raises(RuntimeError, match="one dtype"):
        write_kv8(k, k.half(), c, slots)
    with pytest.raises(RuntimeError, match="bf16 or fp16"):
        write_kv8(k.float(), k.float(), c, slots)
    with pytest.raises(RuntimeError, match="heads"):
        write_kv8(k[:, :1], k[:, :1], c, slots)
    with pytest.raises(RuntimeError, match="layout"):
        write_kv8(k, k, Cache8(c.k, c.v.contiguous(), c.exponents), slots)
    with pytest.raises(RuntimeError, match="exponents"):
        write_kv8(k, k, Cache8(c.k, c.v, c.exponents.int()), slots)
    with pytest.raises(RuntimeError, match="single memory location"):
        write_kv8(k, k, Cache8(c.k, c.k, c.exponents), slots)
    with pytest.raises(RuntimeError, match="codes of"):
        read_kv8(Cache8(c.k.view(torch.uint8), c.v.view(torch.uint8), c.exponents), slots)
    with pytest.raises(RuntimeError, match="block_size"):
        read_kv8(Cache8(*(torch.zeros(1, 2048, 1, D, dtype=I8, device=cuda) for _ in range(2)), torch.zeros(1, 1, 2, dtype=I8, device=cuda)), slots)
    with pytest.raises(RuntimeError, match="dtype"):
        read_kv8(c, slots, torch.float64)
    with pytest.raises(RuntimeError, match="query heads"):
        paged_decode_8(q.repeat(1, 9, 1), c, bt, sl, 16, SCALE)
    with pytest.raises(RuntimeError, match="bf16 or fp16"):
        paged_decode_8(q.float(), c, bt, sl, 16, SCALE)
    with pytest.raises(RuntimeError, match="max_seq_len"):
        paged_decode_8(q, c, bt, sl, 0, SCALE)
    with pytest.raises(RuntimeError, match="block_table"):
        paged_decode_8(q, c, bt.repeat(2, 1), sl, 16, SCALE)
    with pytest.raises(NotImplementedError, match="no gradient"):
        paged_decode_8(q.requires_grad_(), c, bt, sl, 16, SCALE)
    assert paged_decode_8(q[:0].detach(), c, bt[:0], sl[:0], 16, SCALE).shape == (0, 4, D)
    write_kv8(k[:0], k[:0], c, slots[:0])
