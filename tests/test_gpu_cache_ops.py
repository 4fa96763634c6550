"""The operators over uncompressed caches against plain float64 forms: normed q and k with their rotation and
cache write, key bounds, block selection, the decode over selected blocks, the weighing decode and eviction.

Tolerances, u = finfo(type).eps / 2 the rounding of a stored value, e = 2^-24 that of fp32:
- attention: a score is a sum of 128 products in fp32 in any order, off by ds <= (128 + 4) e scale sum |q k| (natural
  units: the products are exact, the scale and the exponential's argument take 4 more roundings). A softmax weight
  is then off by 2 ds + 8 e relative (its own score's error and the sum's; 8 e: exp2, the sums' scale factors), and
  rounded to the cache's type, as is the sum that divides: 2 u (1 + u) relative. out = sum p v: times sum p |v|, plus
  fp32 sums over t tokens, t e sum p |v|, plus the result's own rounding u |out|. fp16 weights below its normal range
  are off by 2^-25 where the largest weight is at least 2^7: t 2^-32 max |v|.
- summed weights: (2 ds + (t + 16) e) times each new weight (the sum l of t terms), plus e of the total.
- normed rows: 20 e relative on each rotated term (16 products and 3 lane sums of squares, their root halving that,
  mean, eps, division, two products, the rotation's two), then u of the result, or fp16's 2^-25 below its range.
"""
import math

import pytest
import torch

from starkv_serve.kernels import model_ops as mo
from starkv_serve.kernels.evict import evict, paged_decode_weighted
from starkv_serve.kernels.sparse_decode import key_bounds_like, paged_decode_sparse, select_blocks, update_key_bounds
from starkv_serve.kernels.stock_decode import paged_decode_full

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
D = 128
SCALE = D ** -0.5
E = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


# -- caches -----------------------------------------------------------------------------------
def make_caches(cuda, lens, Hkv, bs, dt, seed, layout="plain", spare=3):
    """(k_cache, v_cache, block_table, seq_lens): every slot NaN but the requests' tokens."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-L // bs) for L in lens]
    nb = sum(need) + spare
    perm = torch.randperm(nb, generator=g)
    width = max(max(need), 1) + 1
    bt = torch.full((len(lens), width), -1, dtype=torch.int32)
    k, v = (torch.full((nb, bs, Hkv, D), math.nan) for _ in range(2))
    o = 0
    for b, L in enumerate(lens):
        blocks = perm[o:o + need[b]]
        o += need[b]
        bt[b, :need[b]] = blocks.int()
        for t in (k, v):
            rows = torch.full((need[b] * bs, Hkv, D), math.nan)
            rows[:L] = torch.randn(L, Hkv, D, generator=g)
            t[blocks] = rows.view(need[b], bs, Hkv, D)
    if layout == "plain":
        k, v = k.to(dt).to(cuda), v.to(dt).to(cuda)
    elif layout == "pairs":  # keys and values of a block side by side
        kv = torch.stack([k, v], dim=1).to(dt).to(cuda)
        k, v = kv[:, 0], kv[:, 1]
    else:  # heads outside tokens
        k, v = (t.transpose(1, 2).contiguous().to(dt).to(cuda).transpose(1, 2) for t in (k, v))
    return k, v, bt.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)


def rows_of(cache, bt, b, h, tokens):
    """[t, 128] float64 of a request's tokens (CPU)."""
    bs = cache.shape[1]
    c, t = cache.cpu(), bt.cpu()[b].long()
    return torch.stack([c[t[i // bs], i % bs, h] for i in tokens]).double() if len(tokens) else torch.zeros(0, D).double()


def attention64(q, k, v, dt):
    """(out, its tolerance, weights, their tolerance) of q [G, 128] over k, v [t, 128], float64."""
    q, t = q.double(), k.shape[0]
    s = q @ k.t() * SCALE
    ds = ((128 + 4) * E * SCALE * (q.abs() @ k.abs().t())).max().item()
    p = torch.softmax(s, dim=-1)
    u = half_step(dt)
    out, mass = p @ v, p @ v.abs()
    tol = mass * (2 * u * (1 + u) + 2 * ds + (t + 8) * E) + u * out.abs() * 1.01
    if dt == F16:
        tol = tol + t * 2.0 ** -32 * v.abs().max() + 2.0 ** -25
    return out, tol, p, p * (2 * ds + (t + 16) * E)


def check(got, want, tol, what):
    off = ((got.double().cpu() - want).abs() - tol).max().item()
    assert torch.isfinite(got).all(), what
    assert off <= 0, (what, off)


# -- normed rows ------------------------------------------------------------------------------
def norm_rope64(x, w, pos, table, eps):
    x, w = x.double().cpu(), w.double().cpu()
    cos, sin = table.double().cpu()[pos.cpu()].chunk(2, dim=-1)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    a, b = y.chunk(2, dim=-1)
    cos, sin = cos[:, None], sin[:, None]
    z = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    size = torch.cat([(a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()], dim=-1)
    return z, size


@pytest.mark.parametrize("T,H,Hkv,dt,wdt,tdt,pdt", [(1, 32, 32, BF16, BF16, BF16, torch.int64),
                                                    (37, 6, 2, F16, F32, F32, torch.int32),
                                                    (300, 8, 1, BF16, F32, F16, torch.int64),
                                                    (5, 3, 3, F16, F16, BF16, torch.int64)])
def test_norm_rope_write(cuda, T, H, Hkv, dt, wdt, tdt, pdt):
    g = torch.Generator().manual_seed(T)
    qkv = (torch.randn(T, (H + 2 * Hkv) * D, generator=g) * torch.randn(T, 1, generator=g).exp()).to(dt).to(cuda)
    q, k, v = (t.view(T, -1, D) for t in qkv.split([H * D, Hkv * D, Hkv * D], dim=-1))
    if T > 4:
        q[1, 0] = 0  # a row of zeros stays one
    table = torch.randn(50, D, generator=g).clamp(-1, 1).to(tdt).to(cuda)
    pos = torch.randint(-3, 50, (T,), generator=g).to(pdt).to(cuda)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdt).to(cuda) for _ in range(2))
    nb, eps = (T + 15) // 16 + 1, 1e-6
    slots = torch.randperm(nb * 16, generator=g)[:T].to(cuda)
    if T > 4:
        slots[2], slots[3] = -1, nb * 16 + 5  # neither is written
    kc, vc = (torch.randn(nb, 16, Hkv, D, generator=g).to(dt).to(cuda) for _ in range(2))
    kw0, vw0 = kc.clone(), vc.clone()
    qo, ko, k16, v16 = mo.norm_rope_write(pos, q, k, v, table, qw, kw, eps, kc, vc, slots, True, True)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        want, size = norm_rope64(x, w, pos.long(), table, eps)
        check(got, want, 20 * E * size + half_step(dt) * (want.abs() + 20 * E * size) + (2.0 ** -25 if dt == F16 else 1e-38),
              "rows")
    assert torch.equal(k16, ko.to(F16)) and torch.equal(v16, v.to(F16))
    there = (slots >= 0) & (slots < nb * 16)
    kw0.view(-1, Hkv, D)[slots[there]], vw0.view(-1, Hkv, D)[slots[there]] = ko[there], v[there]
    assert torch.equal(kc, kw0) and torch.equal(vc, vw0)
    q2, k2 = mo.norm_rope(pos, q, k, table, qw, kw, eps)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)
    assert torch.equal(mo.norm_rope(pos, q, None, table, qw, None, eps)[0], qo)


def test_norm_rope_fp32_and_no_tokens(cuda):
    g = torch.Generator().manual_seed(3)
    q = torch.randn(9, 2, D, generator=g).to(cuda)
    table = torch.randn(20, D, generator=g).clamp(-1, 1).to(cuda)
    pos, w = torch.arange(9, device=cuda), torch.randn(D, generator=g).to(cuda)
    got, none = mo.norm_rope(pos, q, None, table, w, None, 1e-5)
    want, size = norm_rope64(q, w, pos, table, 1e-5)
    assert none is None
    check(got, want, 21 * E * size, "fp32 rows")
    got, k = mo.norm_rope(pos[:0], q[:0], q[:0], table, w, w, 1e-5)
    assert got.shape == k.shape == (0, 2, D)


# -- bounds -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("layout", ["plain", "pairs", "heads"])
@pytest.mark.parametrize("Hkv,bs,lens,new", [(1, 16, [1, 0, 15, 16, 17, 100], 1), (5, 32, [200, 33, 64, 7], 40),
                                             (8, 64, [129, 1, 500], 1000), (3, 16, [40, 64], 17)])
def test_key_bounds(cuda, dt, layout, Hkv, bs, lens, new):
    kc, _, bt, sl = make_caches(cuda, lens, Hkv, bs, dt, 11, layout)
    got = key_bounds_like(kc).fill_(7.0)
    want = got.cpu()
    for b, L in enumerate(lens):
        for j in range(max(0, L - new) // bs, -(-L // bs)):
            for h in range(Hkv):
                rows = rows_of(kc, bt, b, h, range(j * bs, min(L, (j + 1) * bs)))
                blk = int(bt[b, j])
                want[blk, h, 0], want[blk, h, 1] = rows.amin(0).to(dt), rows.amax(0).to(dt)
    update_key_bounds(kc, got, bt, sl, new)
    assert torch.equal(got.cpu(), want)


def test_key_bounds_keep_nan_and_infinities(cuda):
    kc, _, bt, sl = make_caches(cuda, [20], 1, 16, BF16, 5)
    kc[bt[0, 0].long(), 3, 0, :3] = torch.tensor([math.nan, math.inf, -math.inf], dtype=BF16, device=cuda)
    bounds = key_bounds_like(kc)
    update_key_bounds(kc, bounds, bt, sl, 20)
    b = bounds[bt[0, 0].long(), 0].float()
    assert b[:, 0].isnan().all() and b[1, 1] == math.inf and b[0, 2] == -math.inf
    assert torch.isfinite(b[:, 3:]).all()


# -- selection --------------------------------------------------------------------------------
def select_plain(q, bounds, bt, lens, span, bs, keep, sink, recent):
    q, bounds, bt = q.double().cpu(), bounds.double().cpu(), bt.cpu().long()
    n, H, _ = q.shape
    Hkv = bounds.shape[1]
    G = H // Hkv
    out = torch.full((n, Hkv, keep), -1, dtype=torch.int32)
    for b, L in enumerate(lens):
        nb = -(-min(L, span, bt.shape[1] * bs) // bs)
        for h in range(Hkv):
            x = bounds[bt[b, :nb], h]
            s = torch.zeros(nb, dtype=torch.float64)
            for g in range(G):
                s += torch.maximum(q[b, h * G + g] * x[:, 0], q[b, h * G + g] * x[:, 1]).sum(-1)
            s = s.float()
            if nb <= keep:
                chosen = list(range(nb))
            else:
                rest = range(sink, nb - recent)
                rest = sorted(rest, key=lambda j: (-math.inf if s[j].isnan() else -s[j].item(), j))
                chosen = sorted([*range(sink), *rest[:keep - sink - recent], *range(nb - recent, nb)])
            out[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out


def make_bounds(cuda, lens, Hkv, bs, dt, seed, small=False):
    """Bounds of every block, `small`: of few whole numbers, so that many scores are equal."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-L // bs) for L in lens]
    nb = sum(need) + 2
    x = torch.randint(-2, 3, (nb, Hkv, 2, D), generator=g) // 2 if small else torch.randn(nb, Hkv, 2, D, generator=g)
    x = x.float().sort(dim=2).values.to(dt)
    perm = torch.randperm(nb, generator=g).int()
    bt = torch.full((len(lens), max(need) + 2), -5, dtype=torch.int32)
    o = 0
    for b, m in enumerate(need):
        bt[b, :m] = perm[o:o + m]
        o += m
    return x.to(cuda), bt.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("small", [False, True])
@pytest.mark.parametrize("Hkv,G,bs,lens,keep,sink,recent", [
    (1, 1, 16, [1, 0, 16, 17, 4000], 3, 1, 2), (2, 4, 32, [5000, 3000, 64, 33], 17, 1, 2), (3, 7, 16, [2000, 1999], 50, 0, 0),
    (8, 1, 64, [9000, 128, 65], 5, 2, 3), (1, 16, 16, [1600], 99, 0, 1), (2, 2, 16, [640, 500], 1, 0, 1),
    (4, 8, 16, [20000, 333], 700, 4, 9), (20, 2, 16, [3000, 500], 40, 1, 2), (32, 1, 32, [5000], 12, 0, 1),
    (5, 3, 16, [1200, 1100, 90], 9, 2, 1), (2, 9, 16, [900], 20, 1, 1)])
def test_select_blocks(cuda, dt, small, Hkv, G, bs, lens, keep, sink, recent):
    bounds, bt, sl = make_bounds(cuda, lens, Hkv, bs, dt, 21, small)
    g = torch.Generator().manual_seed(22)
    q = torch.randint(-2, 3, (len(lens), Hkv * G, D), generator=g) if small else torch.randn(len(lens), Hkv * G, D, generator=g)
    q = q.to(dt).to(cuda)
    for span in (max(max(lens), 1), max(1, max(lens) * 2 // 3)):
        got = select_blocks(q, bounds, bt, sl, span, bs, keep, sink, recent)
        assert torch.equal(got.cpu(), select_plain(q, bounds, bt, lens, span, bs, keep, sink, recent))


@pytest.mark.parametrize("blocks", [12800, 16384, 16387, 32768, 33000])
def test_select_blocks_long(cuda, blocks):
    """Rows of as many values as the choice keeps in registers, and of more; a table of more columns than needed."""
    lens = [16 * blocks - 11, 16 * 12288, 16 * 9000 - 3]
    bounds, bt, sl = make_bounds(cuda, lens, 1, 16, BF16, 31)
    q = torch.randn(3, 2, D, generator=torch.Generator().manual_seed(32)).to(BF16).to(cuda)
    got = select_blocks(q, bounds, bt.long(), sl.long(), max(lens), 16, 513, 1, 2)
    assert torch.equal(got.cpu(), select_plain(q, bounds, bt, lens, max(lens), 16, 513, 1, 2))


def test_select_blocks_extremes(cuda):
    """Scores of NaN, both infinities, the type's largest values and zeros of both signs."""
    bounds, bt, sl = make_bounds(cuda, [16 * 40], 1, 16, BF16, 41)
    bounds.zero_()
    row = bt[0].long()
    big = torch.finfo(BF16).max
    for j, (lo, hi) in {5: (math.nan, math.nan), 9: (1.0, math.inf), 12: (-big, big), 13: (-big, big), 20: (-0.0, 0.0),
                        25: (-1.0, -1.0), 30: (math.nan, 1.0)}.items():
        bounds[row[j], 0, 0, 0], bounds[row[j], 0, 1, 0] = lo, hi
    q = torch.zeros(1, 1, D, dtype=BF16, device=cuda)
    q[0, 0, 0] = 1.5
    for keep in (1, 2, 3, 4, 5, 6, 30, 38, 39):
        got = select_blocks(q, bounds, bt, sl, 640, 16, keep, 0, 0)[0, 0].tolist()
        order = [5, 30, 9, 12, 13] + [j for j in range(40) if j not in (5, 9, 12, 13, 25, 30)] + [25]
        assert got == sorted(order[:keep]), keep


# -- the decode over selected blocks ----------------------------------------------------------
SPARSE = [(1, 1, 16, [1, 0, 15, 17, 200], 4, "plain"), (2, 4, 16, [700, 333, 16], 9, "pairs"),
          (3, 7, 32, [1000, 31], 5, "heads"), (8, 2, 64, [900, 64, 129], 6, "plain"), (1, 16, 16, [2500], 120, "plain"),
          (4, 1, 16, [5000, 4999], 301, "pairs"), (2, 9, 16, [300, 77], 11, "heads"), (1, 12, 1024, [3000], 3, "plain"),
          (5, 3, 16, [400], 25, "plain")]


def pick(lens, Hkv, bs, keep, seed):
    """Ascending random blocks a request and head, -1 behind; one row in four has none at all."""
    g = torch.Generator().manual_seed(seed)
    out = torch.full((len(lens), Hkv, keep), -1, dtype=torch.int32)
    for b, L in enumerate(lens):
        nb = -(-L // bs)
        for h in range(Hkv):
            m = min(keep, nb, int(torch.randint(0, nb + 1, (1,), generator=g)) if (b + h) % 4 else nb)
            out[b, h, :m] = torch.randperm(nb, generator=g)[:m].sort().values.int()
            if m and h % 2:
                out[b, h, m - 1] = nb - 1 if m == 1 or out[b, h, m - 2] < nb - 1 else out[b, h, m - 1]
    return out


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("Hkv,G,bs,lens,keep,layout", SPARSE)
def test_sparse_decode(cuda, dt, Hkv, G, bs, lens, keep, layout):
    kc, vc, bt, sl = make_caches(cuda, lens, Hkv, bs, dt, 51, layout)
    g = torch.Generator().manual_seed(52)
    q = torch.randn(len(lens), Hkv * G + 2, D, generator=g).to(dt).to(cuda)[:, 1:-1]
    sel = pick(lens, Hkv, bs, keep, 53)
    got = paged_decode_sparse(q, kc, vc, bt, sl, sel.to(cuda), SCALE)
    for b, L in enumerate(lens):
        for h in range(Hkv):
            tokens = [t for j in sel[b, h].tolist() if j >= 0 for t in range(j * bs, min(L, (j + 1) * bs))]
            mine = got[b, h * G:(h + 1) * G]
            if not tokens:
                assert (mine == 0).all()
                continue
            k, v = rows_of(kc, bt, b, h, tokens), rows_of(vc, bt, b, h, tokens)
            out, tol, _, _ = attention64(q[b, h * G:(h + 1) * G].cpu(), k, v, dt)
            check(mine, out, tol, (b, h))


def test_sparse_decode_places_outside(cuda):
    """Places behind a request's blocks, negative ones and block ids outside the cache hold no tokens; order does not
    matter beyond rounding."""
    kc, vc, bt, sl = make_caches(cuda, [100, 40], 1, 16, BF16, 61)
    q = torch.randn(2, 3, D, generator=torch.Generator().manual_seed(62)).to(BF16).to(cuda)
    good = torch.tensor([[[0, 4, 6]], [[1, 2, -1]]], dtype=torch.int32, device=cuda)
    odd = torch.tensor([[[-7, 6, 99, 0, 4, 7]], [[2, 3, -1, 1, 1 << 30, -1 << 31]]], dtype=torch.int32, device=cuda)
    want = paged_decode_sparse(q, kc, vc, bt, sl, good, SCALE)
    got = paged_decode_sparse(q, kc, vc, bt, sl, odd, SCALE)
    for b, tokens in ((0, [*range(16), *range(64, 80), *range(96, 100)]), (1, [*range(16, 40)])):
        out, tol, _, _ = attention64(q[b].cpu(), rows_of(kc, bt, b, 0, tokens), rows_of(vc, bt, b, 0, tokens), BF16)
        check(want[b], out, tol, b)
        check(got[b], out, tol, b)
    bt2 = bt.clone()
    bt2[0, 4], bt2[1, 1] = kc.shape[0], -1
    got = paged_decode_sparse(q, kc, vc, bt2, sl, good, SCALE)
    for b, tokens in ((0, [*range(16), *range(96, 100)]), (1, [*range(32, 40)])):
        out, tol, _, _ = attention64(q[b].cpu(), rows_of(kc, bt, b, 0, tokens), rows_of(vc, bt, b, 0, tokens), BF16)
        check(got[b], out, tol, b)


def test_sparse_decode_of_everything_is_the_decode(cuda):
    lens = [1000, 77, 512]
    kc, vc, bt, sl = make_caches(cuda, lens, 8, 16, BF16, 71)
    q = torch.randn(3, 32, D, generator=torch.Generator().manual_seed(72)).to(BF16).to(cuda)
    sel = select_blocks(q, key_bounds_like(kc), bt, sl, 1000, 16, 70, 1, 2)
    got, want = paged_decode_sparse(q, kc, vc, bt, sl, sel, SCALE), paged_decode_full(q, kc, vc, bt, sl, 1000, SCALE)
    for b, L in enumerate(lens):
        for h in range(8):
            k, v = rows_of(kc, bt, b, h, range(L)), rows_of(vc, bt, b, h, range(L))
            _, tol, _, _ = attention64(q[b, 4 * h:4 * h + 4].cpu(), k, v, BF16)
            check(got[b, 4 * h:4 * h + 4], want[b, 4 * h:4 * h + 4].double().cpu(), 2 * tol, (b, h))


def test_large_scores(cuda):
    """Scores that rise and fall by thousands from page to page, and a single token's weight of one."""
    kc, vc, bt, sl = make_caches(cuda, [400, 1], 1, 16, F16, 81)
    g = torch.Generator().manual_seed(82)
    ramp = torch.cat([torch.linspace(-60, 60, 200), torch.linspace(60, -60, 200)])
    for t in range(400):
        kc[bt[0, t // 16].long(), t % 16] *= ramp[t].item()
    q = (4 * torch.randn(2, 4, D, generator=g)).to(F16).to(cuda)
    sel = torch.arange(25, dtype=torch.int32, device=cuda).expand(2, 1, 25).contiguous()
    w = torch.zeros(2, 1, 400, device=cuda)
    for got in (paged_decode_sparse(q, kc, vc, bt, sl, sel, SCALE), paged_decode_weighted(q, kc, vc, bt, sl, 400, SCALE, w)):
        out, tol, p, wtol = attention64(q[0].cpu(), rows_of(kc, bt, 0, 0, range(400)), rows_of(vc, bt, 0, 0, range(400)), F16)
        check(got[0], out, tol, "ramp")
        assert torch.equal(got[1], vc[bt[1, 0].long(), 0].expand(4, D))
    check(w[0, 0], p.sum(0), wtol.sum(0) + 8 * E * p.sum(0) + 1e-37, "weights")
    assert abs(w[1, 0, 0].item() - 4) <= 64 * E


def test_infinite_and_nan_values_stay_in_their_rows(cuda):
    """A NaN or infinite value behind a request's end changes nothing; one within it shows in its request alone."""
    kc, vc, bt, sl = make_caches(cuda, [37, 37], 2, 16, BF16, 91)
    q = torch.randn(2, 2, D, generator=torch.Generator().manual_seed(92)).to(BF16).to(cuda)
    sel = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda).expand(2, 2, 3).contiguous()
    vc[bt[0, 2].long(), 5:] = math.inf
    clean = paged_decode_sparse(q, kc, vc, bt, sl, sel, SCALE)
    assert torch.isfinite(clean).all()
    vc[bt[0, 1].long(), 3, 0, 7] = math.inf
    kc[bt[1, 1].long(), 3, 1, 0] = math.nan
    w = torch.zeros(2, 2, 64, device=cuda)
    for got in (paged_decode_sparse(q, kc, vc, bt, sl, sel, SCALE), paged_decode_weighted(q, kc, vc, bt, sl, 37, SCALE, w)):
        assert got[0, 0, 7] == math.inf and torch.isfinite(got[0, 0, :7]).all() and torch.isfinite(got[0, 0, 8:]).all()
        assert torch.isfinite(got[0, 1]).all() and torch.isfinite(got[1, 0]).all() and got[1, 1].isnan().all()
    assert torch.isfinite(w[0]).all() and torch.isfinite(w[1, 0]).all() and w[1, 1, :37].isnan().all() and (w[1, 1, 37:] == 0).all()


# -- the weighing decode ----------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("Hkv,G,bs,lens,span,layout", [
    (1, 1, 16, [1, 0, 15, 17, 200], 200, "plain"), (2, 4, 16, [700, 333, 16], 700, "pairs"),
    (3, 7, 32, [1000, 31], 900, "heads"), (8, 2, 64, [900, 64, 129], 2000, "plain"), (1, 16, 16, [5000], 5000, "plain"),
    (32, 1, 16, [1300, 1025], 1300, "plain"), (1, 5, 16, [9000], 9001, "heads"), (2, 11, 16, [300, 77], 300, "pairs"),
    (1, 3, 256, [700], 700, "plain"), (1, 1, 16, [70000], 70000, "plain")])
def test_weighted_decode(cuda, dt, Hkv, G, bs, lens, span, layout):
    kc, vc, bt, sl = make_caches(cuda, lens, Hkv, bs, dt, 101, layout)
    g = torch.Generator().manual_seed(102)
    q = torch.randn(len(lens), Hkv * G, D, generator=g).to(dt).to(cuda)
    wide = torch.rand(len(lens), Hkv, max(span, max(lens)) + 7, generator=g).to(cuda)
    w = wide[:, :, 1:-2]
    before = wide.cpu()
    got = paged_decode_weighted(q, kc, vc, bt, sl, span, SCALE, w)
    after = wide.cpu()
    for b in range(len(lens)):
        L = min(lens[b], span)
        for h in range(Hkv):
            mine = got[b, h * G:(h + 1) * G]
            old = before[b, h].double()
            new = old.clone()
            if L:
                k, v = rows_of(kc, bt, b, h, range(L)), rows_of(vc, bt, b, h, range(L))
                out, tol, p, wtol = attention64(q[b, h * G:(h + 1) * G].cpu(), k, v, dt)
                check(mine, out, tol, (b, h))
                new[L] = 0  # the newest token's entry is set
                new[1:L + 1] += p.sum(0)
                check(after[b, h, 1:L + 1], new[1:L + 1], wtol.sum(0) + (G + 2) * E * new[1:L + 1] + 1e-37, (b, h, "w"))
            else:
                assert (mine == 0).all()
            assert torch.equal(after[b, h, L + 1:], before[b, h, L + 1:]) and after[b, h, 0] == before[b, h, 0]
    again = before.to(cuda)
    assert torch.equal(paged_decode_weighted(q, kc, vc, bt.long(), sl.long(), span, SCALE, again[:, :, 1:-2]), got)
    assert torch.equal(again, wide)  # the same bits every time


def test_long_ranges_of_a_workgroup(cuda):
    """So many requests that each one's head is one workgroup's, over more pages than are looked up at a time. The
    requests read the same blocks, each with a query of its own."""
    bs, Hkv, L, blocks = 256, 8, 8900, 36
    g = torch.Generator(device=cuda).manual_seed(191)
    kc, vc = (torch.empty(blocks, bs, Hkv, D, device=cuda).normal_(generator=g).to(BF16) for _ in range(2))
    one = torch.randperm(blocks, generator=torch.Generator().manual_seed(192))[:35].int().to(cuda)
    k, v = (t[one.long()].reshape(-1, Hkv, D)[:L].permute(1, 0, 2).cpu() for t in (kc, vc))
    for n, weighted in ((70, False), (520, True)):
        q = torch.empty(n, Hkv, D, device=cuda).normal_(generator=g).to(BF16)
        bt, sl = one.expand(n, -1), torch.full((n,), L, dtype=torch.int32, device=cuda)
        sl[1] = 8193
        if weighted:
            w = torch.zeros(n, Hkv, L, device=cuda)
            got = paged_decode_weighted(q, kc, vc, bt, sl, L, SCALE, w)
        else:
            sel = torch.arange(35, dtype=torch.int32, device=cuda).expand(n, Hkv, -1)
            got = paged_decode_sparse(q, kc, vc, bt, sl, sel, SCALE)
        for b in (0, 1, n // 2, n - 1):
            for h in (0, 3, 7):
                t = int(sl[b])
                out, tol, p, ptol = attention64(q[b, h:h + 1].cpu(), k[h, :t].double(), v[h, :t].double(), BF16)
                check(got[b, h:h + 1], out, tol, (n, b, h))
                if weighted:
                    check(w[b, h, :t], p[0], ptol[0] + 4 * E * p[0] + 1e-37, (n, b, h, "w"))
                    assert (w[b, h, t:] == 0).all()


# -- eviction ---------------------------------------------------------------------------------
def evict_plain(kc, vc, bt, lens, w, keep, sink, recent):
    kc, vc, bt, w = kc.cpu().clone(), vc.cpu().clone(), bt.cpu().long(), w.cpu()
    bs, new, left = kc.shape[1], torch.zeros_like(w.cpu()), []
    for b, L in enumerate(lens):
        left.append(min(L, keep))
        for h in range(kc.shape[2]):
            kept = list(range(L))
            if L > keep:
                mid = sorted(range(sink, L - recent), key=lambda i: (-math.inf if w[b, h, i].isnan() else -w[b, h, i].item(), i))
                kept = sorted([*range(sink), *mid[:keep - sink - recent], *range(L - recent, L)])
            new[b, h, :len(kept)] = w[b, h, kept]
            for c in (kc, vc):
                rows = torch.stack([c[bt[b, i // bs], i % bs, h] for i in kept]) if kept else None
                for j in range(len(kept)):
                    c[bt[b, j // bs], j % bs, h] = rows[j]
    return kc, vc, torch.tensor(left, dtype=torch.int32), new


def same(a, b):
    return torch.equal(a.cpu().nan_to_num(nan=12345.0), b.cpu().nan_to_num(nan=12345.0))


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("Hkv,bs,lens,keep,sink,recent,layout,ties", [
    (1, 16, [1, 0, 15, 17, 200], 16, 1, 2, "plain", False), (2, 16, [700, 333, 16], 300, 4, 32, "pairs", True),
    (3, 32, [1000, 31], 1, 0, 1, "heads", False), (8, 64, [900, 64, 129], 128, 0, 128, "plain", True),
    (1, 16, [2500, 2049], 2048, 0, 0, "plain", False), (2, 16, [1500], 1499, 4, 32, "plain", True),
    (4, 16, [700], 20, 10, 10, "heads", False), (1, 16, [90, 40], 1 << 30, 0, 0, "plain", False),
    (33, 16, [300, 170, 290, 100], 128, 2, 9, "plain", True), (1, 512, [1200], 700, 1, 1, "plain", False),
    (8, 16, [1300, 900, 1250, 40], 600, 3, 20, "pairs", True), (17, 16, [1200], 1100, 3, 20, "heads", False)])
def test_evict(cuda, dt, Hkv, bs, lens, keep, sink, recent, layout, ties):
    kc, vc, bt, sl = make_caches(cuda, lens, Hkv, bs, dt, 111, layout)
    g = torch.Generator().manual_seed(112)
    w = torch.randn(len(lens), Hkv, max(lens) + 9, generator=g).exp()
    if ties:
        w = (w * 2).floor() / 2 * (torch.rand(w.shape, generator=g) > 0.3)
    wide = w.to(cuda)
    want = evict_plain(kc, vc, bt, lens, w, keep, sink, recent)
    got_lens, got_w = evict(kc, vc, bt, sl, wide, keep, sink, recent)
    assert torch.equal(got_lens.cpu(), want[2]) and torch.equal(got_w.cpu(), want[3]) and torch.equal(wide.cpu(), w)
    assert same(kc, want[0]) and same(vc, want[1])


@pytest.mark.parametrize("lens,keep", [([13000, 12400], 12000), ([17000, 16385], 16000), ([33000, 32769], 30000)])
def test_evict_long_and_extreme_weights(cuda, lens, keep):
    """Rows that the choice keeps in registers and longer ones; weights of NaN, infinity and zeros of both signs; int64
    tables."""
    kc, vc, bt, sl = make_caches(cuda, lens, 1, 16, BF16, 121)
    w = torch.rand(2, 1, lens[0], generator=torch.Generator().manual_seed(122))
    w[0, 0, 500], w[0, 0, 700], w[0, 0, 900:1000], w[0, 0, 1000:1100] = math.nan, math.inf, -0.0, 0.0
    want = evict_plain(kc, vc, bt, lens, w, keep, 2, 50)
    got_lens, got_w = evict(kc, vc, bt.long(), sl.long(), w.to(cuda), keep, 2, 50)
    assert torch.equal(got_lens.cpu(), want[2]) and same(got_w, want[3]) and same(kc, want[0]) and same(vc, want[1])


@pytest.mark.parametrize("gone", [[3], [2, 3], [0, 1, 2, 3, 4, 5, 6], [6], [5, 6]])
def test_blocks_outside_the_cache_hold_no_tokens(cuda, gone):
    """Block ids outside the cache (a table's padding that a length runs into): no bounds, the lowest score, no attention,
    a weight of 0, no move."""
    L, Hkv, bs = 100, 2, 16
    kc, vc, bt, sl = make_caches(cuda, [L, 40], Hkv, bs, BF16, 201)
    g = torch.Generator().manual_seed(202)
    q = torch.randn(2, 4, D, generator=g).to(BF16).to(cuda)
    bt2 = bt.clone()
    bt2[0, gone] = torch.tensor([-1, kc.shape[0], 1 << 30, -1 << 31, -7, kc.shape[0] + 1, -1], dtype=torch.int32, device=cuda)[:len(gone)]
    there = [t for t in range(L) if t // bs not in gone]
    bounds = key_bounds_like(kc).fill_(3.0)
    update_key_bounds(kc, bounds, bt2, sl, L)
    want = key_bounds_like(kc).fill_(3.0)
    update_key_bounds(kc, want, bt, sl, L)
    want[bt[0, gone].long()] = 3.0
    assert torch.equal(bounds, want)
    keep = max(1, 7 - len(gone))
    sel = select_blocks(q, bounds, bt2, sl, L, bs, keep, 0, 0)
    if len(gone) < 7:
        assert sel[0].tolist() == [[j for j in range(7) if j not in gone]] * Hkv
    w = torch.rand(2, Hkv, 128, generator=g).to(cuda)
    old = w.clone()
    out = paged_decode_weighted(q, kc, vc, bt2, sl, 128, SCALE, w)
    for h in range(Hkv):
        if there:
            want_out, tol, p, ptol = attention64(q[0, 2 * h:2 * h + 2].cpu(), rows_of(kc, bt, 0, h, there), rows_of(vc, bt, 0, h, there), BF16)
            check(out[0, 2 * h:2 * h + 2], want_out, tol, h)
        else:
            assert (out[0] == 0).all()
        new = old[0, h].double().cpu()
        new[L - 1] = 0
        slack = 4 * E * new
        if there:
            new[there] += p.sum(0)
            slack[there] += ptol.sum(0) + 4 * E * p.sum(0)
        check(w[0, h], new, slack + 1e-37, h)
    before = kc.clone(), vc.clone()
    lens, kept = evict(kc, vc, bt2, sl, w, 50, 2, 10)
    assert lens.tolist() == [50, 40]
    for h in range(Hkv):
        mid = sorted(range(2, 90), key=lambda i: (-w[0, h, i].item(), i))[:38]
        order = [0, 1, *sorted(mid), *range(90, 100)]
        assert torch.equal(kept[0, h, :50], w[0, h, order])
        for now, then in zip((kc, vc), before):
            for j, t in enumerate(order):
                if j // bs in gone:
                    continue
                row = now[bt[0, j // bs].long(), j % bs, h]
                source = t if t // bs not in gone else j  # a row without a source stays
                assert torch.equal(row, then[bt[0, source // bs].long(), source % bs, h])


# -- uses -------------------------------------------------------------------------------------
def test_offsets_past_32_bits(cuda):
    """Blocks behind 2^31 elements of the caches."""
    bs, Hkv = 16, 8
    blocks = 2 ** 31 // (bs * Hkv * D) + 40
    kc, vc = (torch.empty(blocks, bs, Hkv, D, dtype=BF16, device=cuda) for _ in range(2))
    ids = torch.tensor([blocks - 1, 3, blocks - 7, blocks - 20], device=cuda)
    g = torch.Generator(device=cuda).manual_seed(131)
    sk, sv = (torch.empty(4, bs, Hkv, D, device=cuda).normal_(generator=g).to(BF16) for _ in range(2))
    kc[ids], vc[ids] = sk, sv
    bt, sl = ids.int()[None], torch.tensor([60], dtype=torch.int32, device=cuda)
    small = torch.arange(4, dtype=torch.int32, device=cuda)[None]
    q = torch.empty(1, 16, D, device=cuda).normal_(generator=g).to(BF16)
    bounds, sb = key_bounds_like(kc), key_bounds_like(sk)
    update_key_bounds(kc, bounds, bt, sl, 60)
    update_key_bounds(sk, sb, small, sl, 60)
    assert torch.equal(bounds[ids], sb)
    sel, ssel = (select_blocks(q, x, t, sl, 60, bs, 2, 0, 1) for x, t in ((bounds, bt), (sb, small)))
    assert torch.equal(sel, ssel)
    assert torch.equal(paged_decode_sparse(q, kc, vc, bt, sl, sel, SCALE), paged_decode_sparse(q, sk, sv, small, sl, sel, SCALE))
    w, sw = torch.zeros(1, Hkv, 64, device=cuda), torch.zeros(1, Hkv, 64, device=cuda)
    assert torch.equal(paged_decode_weighted(q, kc, vc, bt, sl, 60, SCALE, w),
                       paged_decode_weighted(q, sk, sv, small, sl, 60, SCALE, sw)) and torch.equal(w, sw)
    evict(kc, vc, bt, sl, w, 30, 1, 5)
    evict(sk, sv, small, sl, sw, 30, 1, 5)
    assert torch.equal(kc[ids], sk) and torch.equal(vc[ids], sv)


def run_all(x):
    """A step over selected blocks, a weighing one and a cut, as tensors."""
    q, k = mo.norm_rope(x["pos"], x["q"], None, x["table"], x["w"], None, 1e-6)
    update_key_bounds(x["kc"], x["bounds"], x["bt"], x["sl"], 1)
    sel = select_blocks(q, x["bounds"], x["bt"], x["sl"], 1000, 16, 20, 1, 2)
    out = paged_decode_sparse(q, x["kc"], x["vc"], x["bt"], x["sl"], sel, SCALE)
    full = paged_decode_weighted(q, x["kc"], x["vc"], x["bt"], x["sl"], 1000, SCALE, x["weights"])
    lens, kept = evict(x["kc"], x["vc"], x["bt"], x["sl"], x["weights"], 500, 4, 32)
    return [q, sel, out, full, lens, kept, x["kc"], x["vc"], x["bounds"], x["weights"]]


def make_all(cuda, seed):
    kc, vc, bt, sl = make_caches(cuda, [1000, 500, 731], 4, 16, BF16, seed)
    g = torch.Generator().manual_seed(seed)
    x = dict(kc=kc, vc=vc, bt=bt, sl=sl, bounds=key_bounds_like(kc), weights=torch.rand(3, 4, 1000, generator=g).to(cuda),
             q=torch.randn(3, 12, D, generator=g).to(BF16).to(cuda), table=torch.randn(1024, D, generator=g).clamp(-1, 1).to(cuda),
             w=torch.rand(D, generator=g).to(cuda), pos=(sl - 1).long())
    update_key_bounds(kc, x["bounds"], bt, sl, 1000)
    return x


def test_captured_and_replayed(cuda):
    """Two captured graphs over states of their own, replayed in turn with eager work between: each replay equals the
    eager run of the same step, from the state the last replay left."""
    states, twins = [make_all(cuda, s) for s in (141, 142)], [make_all(cuda, s) for s in (141, 142)]
    run_all(make_all(cuda, 143))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run_all(x))
        graphs.append(graph)
    for step in range(4):
        for i in (0, 1):
            for x in (states[i], twins[i]):
                x["q"].mul_(1.0 if step == 0 else 1.25)
            graphs[i].replay()
            want = run_all(twins[i])
            torch.cuda.synchronize()
            for got, ref in zip(outs[i], want):
                assert same(got, ref)


def test_on_another_stream(cuda):
    """Work on a stream of the caller's, its inputs ready only there, while the default stream is busy."""
    x, want = make_all(cuda, 151), run_all(make_all(cuda, 151))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device=cuda)
    for _ in range(20):
        busy = busy @ busy * 1e-3
    with torch.cuda.stream(stream):
        x["q"].copy_(x["q"].clone())
        got = run_all(x)
    stream.synchronize()
    for a, b in zip(got, want):
        assert same(a, b)
    torch.cuda.synchronize()


def test_no_requests(cuda):
    x = make_all(cuda, 161)
    q, bt, sl = x["q"][:0], x["bt"][:0], x["sl"][:0]
    update_key_bounds(x["kc"], x["bounds"], bt, sl, 1)
    sel = select_blocks(q, x["bounds"], bt, sl, 1000, 16, 20)
    assert sel.shape == (0, 4, 20)
    assert paged_decode_sparse(q, x["kc"], x["vc"], bt, sl, sel, SCALE).shape == q.shape
    assert paged_decode_weighted(q, x["kc"], x["vc"], bt, sl, 1000, SCALE, x["weights"][:0]).shape == q.shape
    lens, kept = evict(x["kc"], x["vc"], bt, sl, x["weights"][:0], 500)
    assert lens.shape == (0,) and kept.shape == (0, 4, 1000)


# -- refusals ---------------------------------------------------------------------------------
def calls(x):
    """Each operator as a function of one tensor to put in another's place."""
    slots = torch.arange(3, device=x["q"].device)
    k = x["q"][:, :4]
    return dict(
        norm=lambda **r: mo.norm_rope(r.get("pos", x["pos"]), r.get("q", x["q"]), r.get("k"), r.get("table", x["table"]),
                                      r.get("w", x["w"]), r.get("kw"), 1e-6),
        write=lambda **r: mo.norm_rope_write(x["pos"], r.get("q", x["q"]), r.get("k", k), r.get("v", k), x["table"], x["w"],
                                             r.get("kw", x["w"]), 1e-6, r.get("kc", x["kc"]), r.get("vc", x["vc"]),
                                             r.get("slots", slots), False, False),
        bounds=lambda **r: update_key_bounds(r.get("kc", x["kc"]), r.get("bounds", x["bounds"]), r.get("bt", x["bt"]),
                                             r.get("sl", x["sl"]), 1),
        select=lambda **r: select_blocks(r.get("q", x["q"]), r.get("bounds", x["bounds"]), r.get("bt", x["bt"]),
                                         r.get("sl", x["sl"]), 1000, r.get("bs", 16), r.get("keep", 5), 1, 2),
        sparse=lambda **r: paged_decode_sparse(r.get("q", x["q"]), r.get("kc", x["kc"]), r.get("vc", x["vc"]), r.get("bt", x["bt"]),
                                               r.get("sl", x["sl"]), r.get("sel", x["sel"]), SCALE),
        weighted=lambda **r: paged_decode_weighted(r.get("q", x["q"]), r.get("kc", x["kc"]), r.get("vc", x["vc"]),
                                                   r.get("bt", x["bt"]), r.get("sl", x["sl"]), r.get("span", 1000), SCALE,
                                                   r.get("weights", x["weights"])),
        evict=lambda **r: evict(r.get("kc", x["kc"]), r.get("vc", x["vc"]), r.get("bt", x["bt"]), r.get("sl", x["sl"]),
                                r.get("weights", x["weights"]), r.get("keep", 500)))


def test_refusals(cuda):
    """What the operators cannot run raises before anything is launched, and leaves everything as it was."""
    x = make_all(cuda, 171)
    x["sel"] = torch.zeros(3, 4, 2, dtype=torch.int32, device=cuda)
    before = {k: v.clone() for k, v in x.items()}
    f = calls(x)
    q, kc = x["q"], x["kc"]
    grad = q.clone().requires_grad_()
    for name in ("norm", "write", "select", "sparse", "weighted"):
        with pytest.raises(NotImplementedError, match="gradient"):
            f[name](q=grad)
    for name in ("bounds", "sparse", "weighted", "evict"):
        with pytest.raises(NotImplementedError, match="gradient"):
            f[name](kc=kc.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="transforms"):
        torch.func.vmap(lambda t: f["sparse"](q=t))(q[None].expand(2, -1, -1, -1))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        f["weighted"]()
    for name, key, t in (("norm", "table", x["table"]), ("write", "kc", kc), ("write", "slots", x["pos"]), ("bounds", "bt", x["bt"]),
                         ("select", "sl", x["sl"]), ("sparse", "sel", x["sel"]), ("weighted", "weights", x["weights"]),
                         ("evict", "weights", x["weights"])):  # a tensor of another device
        with pytest.raises(RuntimeError):
            f[name](**{key: t.cpu()})
    bad = [
        ("norm", dict(q=q[..., :64])), ("norm", dict(q=q.double())), ("norm", dict(w=x["w"][:64])), ("norm", dict(pos=x["pos"][:2])),
        ("norm", dict(table=x["table"][:, :64])), ("norm", dict(k=q, kw=x["w"].half())), ("norm", dict(pos=x["pos"].float())),
        ("write", dict(k=q)), ("write", dict(kc=kc.half())), ("write", dict(slots=x["pos"][:2])), ("write", dict(v=q[:, :3])),
        ("write", dict(vc=x["vc"][1:])), ("write", dict(slots=x["pos"].float())),
        ("write", dict(kc=kc[:1].expand(5, -1, -1, -1), vc=kc[:1].expand(5, -1, -1, -1))),
        ("bounds", dict(bounds=x["bounds"].half())), ("bounds", dict(bounds=x["bounds"][1:])), ("bounds", dict(sl=x["sl"][:2])),
        ("bounds", dict(bounds=x["bounds"][:, :1].expand(-1, 4, -1, -1))), ("bounds", dict(kc=kc[:, :8])),
        ("select", dict(bounds=x["bounds"].half())), ("select", dict(q=q[:, :3])), ("select", dict(bs=24)),
        ("select", dict(bt=x["bt"][:2])), ("select", dict(keep=2)), ("select", dict(keep=0)),
        ("sparse", dict(q=q.half())), ("sparse", dict(sel=x["sel"].long())), ("sparse", dict(sel=x["sel"][:, :2])),
        ("sparse", dict(sel=x["sel"][..., :0])), ("sparse", dict(vc=x["vc"][:, :, :2])), ("sparse", dict(q=q[:, :7])),
        ("sparse", dict(q=q.repeat(1, 6, 1))), ("sparse", dict(kc=kc.transpose(0, 1).contiguous().transpose(0, 1))),
        ("weighted", dict(span=1001)), ("weighted", dict(weights=x["weights"].double())), ("weighted", dict(span=0)),
        ("weighted", dict(weights=x["weights"][:, :1].expand(-1, 4, -1))), ("weighted", dict(weights=x["weights"][:2])),
        ("weighted", dict(q=q.float())), ("weighted", dict(sl=x["sl"][None])),
        ("evict", dict(keep=35)), ("evict", dict(weights=x["weights"][:, :3])), ("evict", dict(bt=x["bt"][0])),
        ("evict", dict(kc=kc[:1].expand(5, -1, -1, -1), vc=kc[:1].expand(5, -1, -1, -1))), ("evict", dict(vc=x["vc"].half())),
        ("evict", dict(vc=kc)), ("write", dict(vc=kc)),
    ]
    for name, wrong in bad:
        with pytest.raises((RuntimeError, ValueError, IndexError)):
            f[name](**wrong)
    torch.cuda.synchronize()
    for k, v in before.items():
        assert same(x[k], v), k
