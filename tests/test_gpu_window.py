"""Attention through a window on the GPU against float64: one token's over 16-bit caches, and prompts'.

Tolerances, u = finfo(type).eps / 2 of the result's type, e = 2^-24 that of fp32, s the scores (natural units), t the
tokens, p the softmax weights:
- a score: 128 products summed in fp32 in any order, the scale and the exponential's argument: ds <= 132 e scale sum |q k|.
  The arguments of the exponentials are differences of rounded scores and references: 8 e (max |s| / ln 2 + 24).
- the decode: weights of at least 22 bits of the cache's type, 2^-22; 2 ds; sums of t terms (t + 16) e; all times sum p |v|.
  fp16 weights below its normal range are off by 2^-25 where the largest is at least 2^7: t 2^-32 max |v|.
- prompts: q, k and v are fp16 values here (of bf16 or fp16 inputs that it holds exactly), the weights of the values are rounded to
  fp16 once, 2^-11, and below its normal range off by 2^-25 where the largest is at least 2^-8 of the reference (the
  reference moves when a score passes it by 2^8, and is a score): t 2^-25 max |v|.
- the result's rounding u |out|, fp16 below its range 2^-25.
"""
import math

import pytest
import torch

from cache8_plain import D, E, SCALE, attention, visible
from starkv_serve.kernels.prefill import prefill_attention
from starkv_serve.kernels.stock_decode import paged_decode_full
from starkv_serve.kernels.window import Window, paged_decode_window

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
SEEN = [(1, 0), (1, 1), (15, 0), (16, 4), (17, 16), (33, 17), (100, 40), (64, 0), (63, 129), (1000, 300), (2 ** 31 - 1, 2 ** 31 - 1)]


# -- one token --------------------------------------------------------------------------------
def session(lens, H, bs, dt, cuda, g, window, layout="plain"):
    """(k, v, block table, lengths): places that no request sees are NaN, blocks of which none is seen -1 in the table."""
    need = [-(-L // bs) for L in lens]
    nb = max(1, sum(need)) + 2
    perm = torch.randperm(nb, generator=g).tolist()
    bt = torch.full((len(lens), max(max(need), 1) + 1), -1, dtype=torch.int32)
    k, v = (torch.full((nb, bs, H, D), math.nan) for _ in range(2))
    o = 0
    for b, L in enumerate(lens):
        for s in visible(L, window):
            blk = perm[o + s // bs]
            bt[b, s // bs] = blk
            k[blk, s % bs], v[blk, s % bs] = torch.randn(H, D, generator=g), torch.randn(H, D, generator=g)
        o += need[b]
    if layout == "plain":
        k, v = k.to(dt).to(cuda), v.to(dt).to(cuda)
    elif layout == "pairs":
        kv = torch.stack([k, v], dim=1).to(dt).to(cuda)
        k, v = kv[:, 0], kv[:, 1]
    else:
        k, v = (t.transpose(1, 2).contiguous().to(dt).to(cuda).transpose(1, 2) for t in (k, v))
    return k, v, bt.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)


def close(got, q, k, v, bt, lens, window, what=""):
    table, bs, H, u = bt.cpu().long(), k.shape[1], k.shape[2], torch.finfo(q.dtype).eps / 2
    G = q.shape[1] // H
    for b, L in enumerate(lens):
        at = torch.tensor(visible(L, window), dtype=torch.long)
        if not len(at):
            assert (got[b] == 0).all(), what
            continue
        K, V = (t.cpu()[table[b, at // bs], at % bs].double() for t in (k, v))
        for h in range(H):
            out, mass, ds, most = attention(q[b, h * G:(h + 1) * G].cpu().double(), K[:, h], V[:, h])
            t = len(at)
            tol = mass * (2 * ds + 8 * E * (most / math.log(2) + 24) + 2.0 ** -22 + (t + 16) * E) + u * out.abs() * 1.01
            if q.dtype == F16:
                tol = tol + t * 2.0 ** -32 * V.abs().max() + 2.0 ** -25
            y = got[b, h * G:(h + 1) * G].double().cpu()
            assert y.isfinite().all(), (what, b, h)
            off = ((y - out).abs() - tol).max().item()
            assert off <= 0, (what, b, h, off)


@pytest.mark.parametrize("size,sinks", SEEN)
@pytest.mark.parametrize("dt,H,G,bs,layout", [(BF16, 2, 4, 16, "plain"), (F16, 1, 12, 32, "pairs"), (BF16, 3, 1, 64, "heads")])
def test_decode(cuda, size, sinks, dt, H, G, bs, layout):
    g = torch.Generator().manual_seed(size % 1000 + sinks % 1000)
    w = Window(size, sinks)
    lens = [0, 1, 15, 16, 17, 64, 100, 129, 400, 1111]
    k, v, bt, sl = session(lens, H, bs, dt, cuda, g, w, layout)
    q = torch.randn(len(lens), 2, H * G, D, generator=g).to(dt).to(cuda)[:, 1]
    close(paged_decode_window(q, k, v, bt, sl, max(lens), SCALE, w), q, k, v, bt, lens, w, (size, sinks))
    close(paged_decode_window(q, k, v, bt, sl.long(), 1 << 24, SCALE, w), q, k, v, bt, lens, w, (size, sinks))


def test_decode_of_long_requests(cuda):
    """Many splits, several looks at the table, and a whole window beside the decode that has none."""
    g = torch.Generator().manual_seed(2)
    for w in (Window(9000, 4), Window(20000, 0), Window(8300, 600)):
        lens = [20000, 9003]
        k, v, bt, sl = session(lens, 1, 16, BF16, cuda, g, w)
        q = torch.randn(2, 4, D, generator=g).to(BF16).to(cuda)
        got = paged_decode_window(q, k, v, bt, sl, 20000, SCALE, w)
        close(got, q, k, v, bt, lens, w)
        if w.size >= 20000:
            full = paged_decode_full(q, k, v, bt, sl, 20000, SCALE)
            assert (got.float() - full.float()).abs().max() <= 2 * 2.0 ** -8 * full.abs().max()


def test_decode_of_infinite_values(cuda):
    """An infinite value that is seen gives infinities, one out of sight nothing; scores of -inf weigh 0."""
    g = torch.Generator().manual_seed(3)
    for dt in (BF16, F16):
        w = Window(50, 4)
        k, v, bt, sl = session([200], 1, 16, dt, cuda, g, None)
        q = torch.randn(1, 2, D, generator=g).to(dt).to(cuda)
        before = paged_decode_window(q, k, v, bt, sl, 200, SCALE, w)
        row = lambda s: (int(bt[0, s // 16]), s % 16, 0)  # noqa: E731
        k[row(100)], v[row(100)] = math.nan, math.inf
        v[row(149)] = -math.inf
        assert torch.equal(paged_decode_window(q, k, v, bt, sl, 200, SCALE, w), before)
        v[row(2)][5], v[row(199)][7] = math.inf, -math.inf
        got = paged_decode_window(q, k, v, bt, sl, 200, SCALE, w)
        assert (got[..., 5] == math.inf).all() and (got[..., 7] == -math.inf).all()
        rest = [d for d in range(D) if d not in (5, 7)]
        assert torch.equal(got[..., rest], before[..., rest])
        k[row(3)] = 0
        k[row(3)][0] = math.inf
        q[..., 0] = -1.0
        v[row(2)][5] = v[row(199)][7] = 0
        v[row(3)] = 100.0
        got = paged_decode_window(q, k, v, bt, sl, 200, SCALE, w)
        k[row(3)] = 0
        k[row(3)][0] = 60000.0 if dt == F16 else 1e30
        assert torch.equal(got, paged_decode_window(q, k, v, bt, sl, 200, SCALE, w))


def test_decode_of_bad_blocks_and_lengths(cuda):
    g = torch.Generator().manual_seed(4)
    w = Window(70, 20)
    k, v, bt, sl = session([200, 300], 2, 16, F16, cuda, g, None)
    q = torch.randn(2, 4, D, generator=g).to(F16).to(cuda)
    close(paged_decode_window(q, k, v, bt, sl, 130, SCALE, w), q, k, v, bt, [130, 130], w)
    bad = bt.clone()
    bad[0, 9], bad[0, 10] = 10 ** 6, -7
    got = paged_decode_window(q, k, v, bad, sl, 300, SCALE, w)
    at = [s for s in visible(200, w) if s // 16 not in (9, 10)]
    K, V = (torch.stack([t.cpu()[int(bt[0, s // 16]), s % 16, 0] for s in at]).double() for t in (k, v))
    want = attention(q[0, :2].cpu().double(), K, V)[0]
    assert (got[0, :2].cpu().double() - want).abs().max() <= 2.0 ** -10 * V.abs().max()
    zero = paged_decode_window(q, k, v, bt, torch.tensor([-1, 0], device=cuda), 300, SCALE, w)
    assert (zero == 0).all()


def test_decode_past_31_bits(cuda):
    """Blocks at the far end of a cache whose offsets pass 2^31."""
    g = torch.Generator().manual_seed(5)
    nb, bs, H = 140000, 64, 2
    cache = torch.zeros(2, nb, bs, H, D, dtype=BF16, device=cuda)
    table = torch.tensor([[nb - 1, 5, nb - 2, nb // 2]], dtype=torch.int32, device=cuda)
    k, v = cache[0], cache[1]
    for t in (k, v):
        t[table[0].long()] = torch.randn(4, bs, H, D, generator=g).to(BF16).to(cuda)
    q = torch.randn(1, 8, D, generator=g).to(BF16).to(cuda)
    sl, w = torch.tensor([230], device=cuda), Window(100, 30)
    got = paged_decode_window(q, k, v, table, sl, 256, SCALE, w)
    close(got, q, k[table[0].long()], v[table[0].long()], torch.arange(4, dtype=torch.int32)[None], [230], w)


def test_captured_steps(cuda):
    g = torch.Generator().manual_seed(6)
    w = Window(64, 4)
    lens = [100, 300]
    k, v, bt, sl = session([L + 8 for L in lens], 2, 16, BF16, cuda, g, None)
    sl = torch.tensor(lens, dtype=torch.int32, device=cuda)
    q = torch.randn(2, 8, D, generator=g).to(BF16).to(cuda)
    paged_decode_window(q, k, v, bt, sl, 4096, SCALE, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_decode_window(q, k, v, bt, sl, 4096, SCALE, w)
    for i in range(5):
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        assert torch.equal(out, paged_decode_window(q, k, v, bt, sl, 4096, SCALE, w))
        close(out, q, k, v, bt, [L + i for L in lens], w)
        torch.cuda.synchronize()
        sl.add_(1)


# -- prompts ----------------------------------------------------------------------------------
def prompts_close(got, q, k, v, lens, w, what="", scale=SCALE, fine=None):
    G, u, o = q.shape[1] // k.shape[1], torch.finfo(got.dtype).eps / 2, 0
    for L in filter(None, lens):
        t = torch.arange(L)
        sees = (t[None, :] <= t[:, None]) & ((t[:, None] - t[None, :] < w.size) | (t[None, :] < w.sinks))
        for h in range(q.shape[1]):
            x, K, V = q[o:o + L, h].cpu().double(), k[o:o + L, h // G].cpu().double(), v[o:o + L, h // G].cpu().double()
            s = (x @ K.t() * scale).masked_fill(~sees, -math.inf)
            p = torch.softmax(s, dim=-1)
            ds = 2 * 132 * E * abs(scale) * (x.abs() @ K.abs().t()).masked_fill(~sees, 0).amax(-1, keepdim=True)
            most = s.masked_fill(~sees, 0).abs().amax(-1, keepdim=True)
            n = sees.sum(-1, keepdim=True)
            out, mass = p @ V, p @ V.abs()
            tol = (mass * (ds + 8 * E * (most / math.log(2) + 24) + 2.0 ** -11 + (n + 16) * E) + n * 2.0 ** -25 * V.abs().max()
                   + u * out.abs() * 1.01 + (2.0 ** -25 if got.dtype == F16 else 0))
            y = got[o:o + L, h].cpu().double()
            assert y.isfinite().all(), (what, h)
            off = (y - out).abs() - tol
            off = (off if fine is None else off[fine[o:o + L, h]]).max().item()
            assert off <= 0, (what, L, h, off)
        o += L


@pytest.mark.parametrize("size,sinks", SEEN + [(127, 64), (128, 65), (129, 0), (200, 200)])
@pytest.mark.parametrize("dt,H,G", [(BF16, 1, 8), (F16, 2, 1)])
def test_prompts(cuda, size, sinks, dt, H, G):
    g = torch.Generator().manual_seed(size % 1000 + sinks % 1000)
    lens = [1, 63, 64, 0, 65, 130, 700, 257]
    T = sum(lens)
    q, k, v = (t.view(T, -1, D) for t in torch.randn(T, (G + 2) * H * D, generator=g).to(dt).to(cuda).split([G * H * D, H * D, H * D], -1))
    w = Window(size, sinks)
    prompts_close(prefill_attention(q, k, v, lens, SCALE, window=w), q, k, v, lens, w, (size, sinks))


def test_prompts_of_other_types_and_scales(cuda):
    """fp32 queries, a given output, heads that do not divide by 8, scales of either sign and of none."""
    g = torch.Generator().manual_seed(8)
    lens, w = [300, 90], Window(100, 10)
    q = (torch.randint(-64, 65, (390, 3, D), generator=g) / 32.0).to(cuda)  # fp32 values that fp16 holds
    k, v = (torch.randn(390, 1, D, generator=g).to(F16).to(cuda) for _ in range(2))
    for scale in (SCALE, -SCALE, 0.0, 4 * SCALE):
        out = torch.full((390, 3, D), math.nan, device=cuda, dtype=BF16)
        got = prefill_attention(q, k, v, lens, scale, out=out, window=w)
        assert got is out
        prompts_close(out, q, k, v, lens, w, scale, scale)


def test_prompts_of_any_strides(cuda):
    """bf16 keys where they lie: broadcast over heads or tokens, rows in the middle of wider ones, unaligned ones; values past
    fp16's range are the one thing that is not taken."""
    g = torch.Generator().manual_seed(12)
    L, w = 300, Window(70, 5)
    wide = torch.randn(L, 5, 3 * D, generator=g).to(BF16).to(cuda)
    q = torch.randn(L, 4, D, generator=g).to(BF16).to(cuda)
    v = torch.randn(L, 2, D, generator=g).to(BF16).to(cuda)
    for k in (wide[:, 1:3, D:2 * D], wide[:, :1, :D].expand(L, 2, D), wide[:1, :2, :D].expand(L, 2, D), wide[:, ::2, 8:8 + D][:, :2],
              wide[:, 2:4, 4:4 + D], wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :2, :D]):
        prompts_close(prefill_attention(q, k, v, [L], SCALE, window=w), q, k, v, [L], w, k.stride())
    one = wide[7:8, :2, :D]
    prompts_close(prefill_attention(q[:1], one.as_strided(one.shape, (0, 3 * D, 1)), v[:1], [1], SCALE, window=w), q, one, v, [1], w)
    k = wide[:, :2, :D] * 1e20  # keys of any size that bf16 has
    prompts_close(prefill_attention(q, k, v, [L], SCALE * 1e-20, window=w), q, k, v, [L], w, "large", SCALE * 1e-20)


def test_prompts_of_any_fp16_strides(cuda):
    """fp16 keys and values where they lie, with strides of one kind or two, broadcast, unaligned, of one token."""
    g = torch.Generator().manual_seed(14)
    L, w = 300, Window(70, 5)
    wide = torch.randn(L, 6, 3 * D, generator=g).to(F16).to(cuda)
    q = torch.randn(L, 4, D, generator=g).to(F16).to(cuda)
    by_head = wide.transpose(0, 1).contiguous().transpose(0, 1)
    for k, v in ((wide[:, 1:3, D:2 * D], wide[:, 3:5, :D]), (wide[:, :1, :D].expand(L, 2, D), wide[:, 5:, D:2 * D].expand(L, 2, D)),
                 (wide[:1, :2, :D].expand(L, 2, D), wide[4:5, :2, :D].expand(L, 2, D)), (wide[:, ::3, 8:8 + D], wide[:, 1::3, 16:16 + D]),
                 (wide[:, 2:4, 4:4 + D], wide[:, :2, 4:4 + D]), (wide[:, :2, :D], wide[:, 2:4, 2:2 + D]), (by_head[:, :2, :D], by_head[:, 4:, D:2 * D]),
                 (by_head[:, :2, :D], wide[:, :2, :D])):
        prompts_close(prefill_attention(q, k, v, [L - 20, 20], SCALE, window=w), q, k, v, [L - 20, 20], w, (k.stride(), v.stride()))
    k1, v1 = (t.as_strided((1, 2, D), (8, 3 * D, 1)) for t in (wide[7:8, :2, :D], wide[9:10, :2, :D]))
    prompts_close(prefill_attention(q[:1], k1, v1, [1], SCALE, window=w), q[:1], k1, v1, [1], w)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_prompts_of_infinite_values(cuda, dt):
    """Infinite values and NaN reach the rows that see them, and no others; keys that are not finite the same."""
    g = torch.Generator().manual_seed(13)
    lens, w, H, G = [400, 70, 200], Window(100, 20), 2, 2
    T = sum(lens)
    q, k, v = (torch.randn(T, h, D, generator=g).to(dt) for h in (H * G, H, H))
    clean = v.clone()
    odd = [(3, 0, 7, math.inf), (40, 0, 8, math.nan), (41, 0, 9, -math.inf), (150, 0, 7, -math.inf), (399, 0, 1, math.inf), (250, 1, 100, math.inf),
           (251, 1, 100, math.inf), (400 + 69, 0, 3, math.nan), (470 + 64, 1, 2, -math.inf), (470 + 199, 1, 127, math.nan)]
    for t, h, d, x in odd:
        v[t, h, d], clean[t, h, d] = x, 0.0
    got = prefill_attention(q.to(cuda), k.to(cuda), v.to(cuda), lens, SCALE, window=w).cpu()
    expect = torch.zeros(T, H * G, D)  # what the infinite values that a row sees sum up to
    start = 0
    for L in lens:
        t = torch.arange(L)
        sees = (t[None, :] <= t[:, None]) & ((t[:, None] - t[None, :] < w.size) | (t[None, :] < w.sinks))
        for at, h, d, x in odd:
            if start <= at < start + L:
                expect[start:start + L, h * G:(h + 1) * G, d] += torch.where(sees[:, at - start], x, 0.0)[:, None]
        start += L
    fine = expect == 0
    assert torch.equal(got.isnan(), expect.isnan()) and torch.equal(got[expect.isinf()].float(), expect[expect.isinf()])
    assert 0 < int(expect.isnan().sum()) < T and got[fine].isfinite().all()
    prompts_close(torch.where(fine, got, 0.0).to(dt), q, k, clean, lens, w, "zero", fine=fine)
    # a NaN key: its row's sight is NaN, the others' rows are as without it
    k[100, 0, 5] = math.nan
    got = prefill_attention(q.to(cuda), k.to(cuda), clean.to(cuda), lens, SCALE, window=w).cpu()
    bad = torch.zeros(T, H * G, dtype=torch.bool)
    bad[100:200, :G] = True
    assert torch.equal(got.isnan().all(-1), bad) and torch.equal(got.isnan().any(-1), bad)


def test_prompts_large_keys_out_of_sight(cuda):
    """Keys that a row does not see do not change it: not by a bit from row 288 on, and by roundings in rows 264 to 287, for
    which 32 rows of a wave move their references together and the rows in front of them see some of the keys."""
    g = torch.Generator().manual_seed(9)
    L, w = 500, Window(64, 3)
    q, k, v = (torch.randn(L, 1, D, generator=g).to(F16).to(cuda) for _ in range(3))
    k[3:200] *= 500  # rows from 264 on see none of these
    got = prefill_attention(q, k, v, [L], SCALE, window=w)
    k2 = k.clone()
    k2[3:200] /= 500
    other = prefill_attention(q, k2, v, [L], SCALE, window=w)
    assert torch.equal(got[288:], other[288:])
    prompts_close(other, q, k2, v, [L], w)
    other[264:] = got[264:]
    prompts_close(other, q, k2, v, [L], w)


def test_a_window_of_the_whole_prompt_is_the_causal_attention(cuda):
    g = torch.Generator().manual_seed(10)
    lens = [333, 77]
    q, k, v = (torch.randn(410, h, D, generator=g).to(BF16).to(cuda) for h in (4, 2, 2))
    a, b = prefill_attention(q, k, v, lens, SCALE), prefill_attention(q, k, v, lens, SCALE, window=Window(333))
    assert (a.float() - b.float()).abs().max() <= 3 * 2.0 ** -8 * a.abs().max()


def test_on_the_callers_stream(cuda):
    g = torch.Generator().manual_seed(11)
    w = Window(40, 4)
    k0, v0, bt, sl = session([200], 2, 16, BF16, cuda, g, None)
    q0 = torch.randn(1, 4, D, generator=g).to(BF16).to(cuda)
    p0 = [torch.randn(200, h, D, generator=g).to(BF16).to(cuda) for h in (4, 2, 2)]

    def run(q, k, v, p):
        return [paged_decode_window(q, k, v, bt, sl, 200, SCALE, w), prefill_attention(*p, [200], SCALE, window=w)]

    want = run(q0, k0, v0, p0)
    xs = [torch.zeros_like(t) for t in (q0, k0, v0, *p0)]
    busy = torch.randn(4096, 4096, device=cuda)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(30):
            busy = busy @ busy * 1e-3
        for a, b in zip(xs, (q0, k0, v0, *p0)):
            a.copy_(b)
        got = [t.clone() for t in run(*xs[:3], xs[3:])]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(cuda):
    q, k = torch.zeros(1, 4, D, dtype=BF16, device=cuda), torch.zeros(4, 16, 2, D, dtype=BF16, device=cuda)
    bt, sl, w = torch.zeros(1, 4, dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda), Window(8, 1)
    with pytest.raises(RuntimeError, match="dtype"):
        paged_decode_window(q.half(), k, k, bt, sl, 16, SCALE, w)
    with pytest.raises(RuntimeError, match="max_seq_len"):
        paged_decode_window(q, k, k, bt, sl, 0, SCALE, w)
    with pytest.raises(RuntimeError, match="query heads"):
        paged_decode_window(q.repeat(1, 9, 1), k, k, bt, sl, 16, SCALE, w)
    with pytest.raises(RuntimeError, match="block_table"):
        paged_decode_window(q, k, k, bt, sl.repeat(2), 16, SCALE, w)
    with pytest.raises(RuntimeError, match="window"):
        paged_decode_window(q, k, k, bt, sl, 16, SCALE, None)
    with pytest.raises(NotImplementedError, match="no gradient"):
        paged_decode_window(q.requires_grad_(), k, k, bt, sl, 16, SCALE, w)
    with pytest.raises(NotImplementedError, match="no gradient"):
        prefill_attention(q, k[0, :1], k[0, :1], [1], SCALE, window=w)
    assert paged_decode_window(q.detach()[:0], k, k, bt[:0], sl[:0], 16, SCALE, w).shape == (0, 4, D)
