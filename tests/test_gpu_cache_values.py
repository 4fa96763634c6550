"""Infinite, huge and NaN values in the decodes over uncompressed caches, against float64 (tolerances of test_gpu_cache_ops).

A key whose score is -inf has the softmax weight 0, like a token that is not there; a row whose scores are all -inf is
NaN, as the softmax's own 0 / 0. An infinite value gives an infinite result whatever its token's weight is, as long as
that is not 0: inf - inf and 0 inf are NaN."""
import math

import pytest
import torch

from starkv_serve.kernels.evict import paged_decode_weighted
from starkv_serve.kernels.sparse_decode import paged_decode_sparse
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
