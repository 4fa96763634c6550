"""Infinite, huge and NaN values in the decodes over uncompressed caches, against float64 (tolerances of test_gpu_cache_ops).

A key whose score is -inf has the softmax weight 0, like a token that is not there; a row whose scores are all -inf is
NaN, as the softmax's own 0 / 0. An infinite value gives an infinite result whatever its token's weight is, as long as
that is not 0: inf - inf and 0 inf are NaN."""
import math

import pytest
import torch

from starkv_serve.kernels.evict import paged_decode_weighted
from starkv_serve.kernels.sparse_decode import paged_decode_sparse
from starkv_serve.kernels.stock_decode import paged_decode_full
from test_gpu_cache_ops import BF16, D, E, F16, SCALE, attention64, check, make_caches, rows_of

pytestmark = pytest.mark.gpu

GROUPS = [1, 3, 8, 9, 16]


def decodes(q, kc, vc, bt, sl, span):
    """Both decodes over every token: (name, out, weights or None)."""
    n, Hkv, bs = q.shape[0], kc.shape[2], kc.shape[1]
    keep = -(-span // bs)
    sel = torch.arange(keep, dtype=torch.int32, device=q.device).expand(n, Hkv, keep).contiguous()
    w = torch.zeros(n, Hkv, span, device=q.device)
    return [("sparse", paged_decode_sparse(q, kc, vc, bt, sl, sel, SCALE), None),
            ("weighted", paged_decode_weighted(q, kc, vc, bt, sl, span, SCALE, w), w)]


def queries(n, heads, dt, seed, cuda):
    """Queries whose first dimension is 1."""
    q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(seed))
    q[:, :, 0] = 1
    return q.to(dt).to(cuda)


def token(cache, bt, b, t, h):
    return cache[bt[b, t // cache.shape[1]].long(), t % cache.shape[1], h]


# (length, its tokens of score -inf): a wave's only page, whole first tiles, whole waves' and splits' parts, single tokens
LOST = [(97, [96]), (40, range(32)), (97, range(64)), (33, [32]), (2, [0]), (5000, range(2500)), (5000, [*range(700), 4999]),
        (300, range(0, 300, 2)), (300, range(1, 299))]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("G", GROUPS)
def test_scores_of_minus_infinity_weigh_nothing(cuda, dt, G):
    lens = [L for L, _ in LOST]
    kc, vc, bt, sl = make_caches(cuda, lens, 1, 16, dt, 301)
    for b, (L, lost) in enumerate(LOST):
        for t in lost:
            token(kc, bt, b, t, 0)[0] = -math.inf
    q = queries(len(lens), G, dt, 302, cuda)
    for name, out, w in decodes(q, kc, vc, bt, sl, max(lens)):
        for b, (L, lost) in enumerate(LOST):
            there = sorted(set(range(L)) - set(lost))
            want, tol, p, ptol = attention64(q[b].cpu(), rows_of(kc, bt, b, 0, there), rows_of(vc, bt, b, 0, there), dt)
            check(out[b], want, tol, (name, b))
            if w is not None:
                weights, slack = torch.zeros(max(lens), dtype=torch.float64), torch.full((max(lens),), 1e-37, dtype=torch.float64)
                weights[there] = p.sum(0)
                slack[there] += ptol.sum(0) + 20 * E * p.sum(0)
                check(w[b, 0], weights, slack, (name, b, "w"))


@pytest.mark.parametrize("dt", [BF16, F16])
def test_rows_whose_scores_are_all_minus_infinity(cuda, dt):
    """NaN, in their own row: a row without tokens is zero, other heads are not touched."""
    lens = [1, 50, 3000, 0, 20]
    kc, vc, bt, sl = make_caches(cuda, lens, 2, 16, dt, 311)
    for b in (0, 1, 2):
        for t in range(lens[b]):
            token(kc, bt, b, t, 1)[0] = -math.inf
    q = queries(len(lens), 4, dt, 312, cuda)
    for name, out, w in decodes(q, kc, vc, bt, sl, 3000):
        for b, L in enumerate(lens):
            assert torch.isfinite(out[b, :2]).all(), (name, b)
            assert out[b, 2:].isnan().all() if b < 3 else torch.isfinite(out[b, 2:]).all(), (name, b)
            if w is not None:
                assert torch.isfinite(w[b, 0]).all() and (w[b, 1, L:] == 0).all()
                assert w[b, 1, :L].isnan().all() if b < 3 else torch.isfinite(w[b, 1]).all()
        assert (out[3] == 0).all()


# (length, {token: its score's distance above the others', or None for one among them}); the infinite values' tokens
INFINITE = [(1, {0: None}), (2, {1: None}), (37, {19: None}), (300, {0: None, 299: None}), (5000, {4999: None}),
            (700, {123: 30.0}), (700, {5: -30.0}), (64, {t: None for t in range(64)}), (5000, {40: -12.0, 3000: 12.0})]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("G", GROUPS)
def test_infinite_values(cuda, dt, G):
    """Dimension 0 holds +inf at the named tokens, 1 -inf, 2 NaN, 3 both infinities by turns (of a single token +inf), 127
    +inf at one that scores -inf besides. Scores below the largest by 30 leave weights that fp16 does not hold."""
    lens = [L for L, _ in INFINITE]
    kc, vc, bt, sl = make_caches(cuda, lens, 1, 16, dt, 321)
    q = queries(len(lens), G, dt, 322, cuda)
    for b, (L, at) in enumerate(INFINITE):
        for i, (t, above) in enumerate(at.items()):
            if above is not None:
                token(kc, bt, b, t, 0)[0] += above / SCALE
            row = token(vc, bt, b, t, 0)
            row[0], row[1], row[2], row[3] = math.inf, -math.inf, math.nan, -math.inf if i % 2 else math.inf
    last = len(lens) - 1
    token(kc, bt, last, 1, 0)[0] = -math.inf
    token(vc, bt, last, 1, 0)[127] = math.inf
    for name, out, w in decodes(q, kc, vc, bt, sl, max(lens)):
        for b, (L, at) in enumerate(INFINITE):
            both = len(at) > 1
            for d, want in ((0, math.inf), (1, -math.inf), (2, math.nan), (3, math.nan if both else math.inf)):
                got = out[b, :, d]
                assert got.isnan().all() if math.isnan(want) else (got == want).all(), (name, b, d)
            k, v = rows_of(kc, bt, b, 0, range(L)), rows_of(vc, bt, b, 0, range(L))
            if b == last:
                assert out[b, :, 127].isnan().all()  # 0 inf
                there = [t for t in range(L) if t != 1]
                k, v = k[there], v[there]
            want, tol, p, _ = attention64(q[b].cpu(), k, v[:, 4:127], dt)
            check(out[b, :, 4:127], want, tol, (name, b))
            if w is not None:
                assert torch.isfinite(w).all() and abs(w[b, 0].sum().item() - G) < 1e-3 * G


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("G", [1, 8, 13])
@pytest.mark.parametrize("part", [1.0, 2.0 ** -9, 2.0 ** -14])
def test_largest_values(cuda, dt, G, part):
    """A mean of the type's largest values is no larger, whatever the sums on the way to it are."""
    lens = [1, 40, 3000, 20000]
    kc, vc, bt, sl = make_caches(cuda, lens, 1, 16, dt, 331)
    vc.copy_(torch.where(vc.isnan(), vc, vc.sign() * (torch.finfo(dt).max * part)))
    vc[:, :, :, :64] = vc[:, :, :, :64].abs()
    q = queries(len(lens), G, dt, 332, cuda)
    for name, out, w in decodes(q, kc, vc, bt, sl, max(lens)):
        for b, L in enumerate(lens):
            want, tol, _, _ = attention64(q[b].cpu(), rows_of(kc, bt, b, 0, range(L)), rows_of(vc, bt, b, 0, range(L)), dt)
            top = torch.finfo(dt).max * part
            got = out[b].double().cpu()
            assert ((got - want).abs() <= tol).all(), (name, b)
            assert (got[:, :64] >= top * 0.98).all() and (got.abs() <= top).all(), (name, b)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_whole_decode_with_scores_of_minus_infinity(cuda, dt, G):
    """``paged_decode_full``: one length a call, so that every split of it is a case."""
    for L, lost in LOST:
        kc, vc, bt, sl = make_caches(cuda, [L, L], 2, 16, dt, 341)
        for t in lost:
            token(kc, bt, 0, t, 1)[0] = -math.inf
        for t in range(L):
            token(kc, bt, 1, t, 0)[0] = -math.inf
        q = queries(2, 2 * G, dt, 342, cuda)
        out = paged_decode_full(q, kc, vc, bt, sl, L, SCALE)
        there = sorted(set(range(L)) - set(lost))
        for b, h, tokens in ((0, 0, range(L)), (0, 1, there), (1, 1, range(L))):
            mine = out[b, h * G:(h + 1) * G]
            want, tol, _, _ = attention64(q[b, h * G:(h + 1) * G].cpu(), rows_of(kc, bt, b, h, tokens), rows_of(vc, bt, b, h, tokens), dt)
            check(mine, want, tol, (L, b, h))
        assert out[1, :G].isnan().all()
