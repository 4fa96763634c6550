"""How exact the softmax weights are that the decodes over uncompressed caches multiply values by, against float64.

Outputs in 16 bits hide what a weight lost, so the first test makes them small: two tokens, values 1 and minus the
second's weight rounded, whose sum leaves the rounding. e = 2^-24. Scores are one exact product; the scale's and the
score's rounding and that of its distance from the reference (below 9, in units of log2: 16 e of it) leave a weight off
by 3 e + 8 e ln 2 x 2, its exponential by 4 e: below 20 e. The sums of two tokens' products, of at most three values of a
weight each, of 4 waves, and the quotient are at most 14 roundings of at most a whole step, 2 e. tol = 48 e sum p |v| + the
result's own rounding.

The second: values of one sign, so that nothing a weight lost cancels. A score's error ds as in test_gpu_cache_ops; at
most two products of 32 terms a tile and a whole step each term, 4 t e, and joins of up to 4 waves and 128 splits, 300 e."""
import math

import pytest
import torch

from starkv_serve.kernels.evict import paged_decode_weighted
from starkv_serve.kernels.sparse_decode import paged_decode_sparse
from test_gpu_cache_ops import BF16, D, E, F16, SCALE, check, half_step, make_caches, rows_of

pytestmark = pytest.mark.gpu


def both(q, kc, vc, bt, sl, span, scale):
    n, Hkv, bs = q.shape[0], kc.shape[2], kc.shape[1]
    keep = -(-span // bs)
    sel = torch.arange(keep, dtype=torch.int32, device=q.device).expand(n, Hkv, keep).contiguous()
    w = torch.zeros(n, Hkv, span, device=q.device)
    return (("sparse", paged_decode_sparse(q, kc, vc, bt, sl, sel, scale)),
            ("weighted", paged_decode_weighted(q, kc, vc, bt, sl, span, scale, w)))


def lossy_scores(dt, count=24):
    """Scores (log2) whose weights leave most when they are cut to two values of bf16, or to one of fp16."""
    s = -torch.arange(1, 128, dtype=torch.float64) / 128  # exact in both types
    x = torch.exp2(s).float()
    if dt == F16:
        left = (x - x.half().float()).abs()
    else:
        cut = lambda v: (v.view(torch.int32) & -65536).view(torch.float32)
        left = x - cut(x)
        left = left - cut(left)
    return s[(left / x).sort(descending=True).indices[:count]]


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("G", [1, 8, 9, 16])
def test_weights_keep_their_bits(cuda, dt, G):
    s = lossy_scores(dt)
    n = len(s)
    kc, vc, bt, sl = make_caches(cuda, [2] * n, 1, 16, dt, 401)
    first = bt[:, 0].long()
    x = torch.exp2(s)
    v = torch.stack([-x.to(dt).double(), torch.ones_like(x)], dim=1)[:, :, None] * torch.exp2(torch.arange(D) % 5 - 2.0).double()
    kc[first, :2, 0] = 0
    kc[first, 1, 0, 0] = s.to(dt).to(cuda)
    vc[first, :2, 0] = v.to(dt).to(cuda)
    q = torch.zeros(n, G, D, dtype=dt, device=cuda)
    q[:, :, 0] = 1
    p = torch.stack([torch.ones_like(x), x], dim=1) / (1 + x)[:, None]
    want, mass = ((p[:, :, None] * t).sum(1)[:, None].expand(n, G, D) for t in (v, v.abs()))
    tol = 48 * E * mass + half_step(dt) * want.abs() * 1.01 + (2.0 ** -25 if dt == F16 else 0)
    for name, got in both(q, kc, vc, bt, sl, 2, math.log(2)):
        check(got, want, tol, name)


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("Hkv,G", [(2, 4), (1, 8), (1, 13)])
def test_values_of_one_sign(cuda, dt, Hkv, G):
    lens = [40, 300, 1000, 33]
    kc, vc, bt, sl = make_caches(cuda, lens, Hkv, 16, dt, 411)
    vc.abs_()
    q = torch.randn(len(lens), Hkv * G, D, generator=torch.Generator().manual_seed(412)).to(dt).to(cuda)
    for name, got in both(q, kc, vc, bt, sl, max(lens), SCALE):
        for b, L in enumerate(lens):
            for h in range(Hkv):
                k, v = rows_of(kc, bt, b, h, range(L)), rows_of(vc, bt, b, h, range(L))
                mine = q[b, h * G:(h + 1) * G].double().cpu()
                ds = ((128 + 4) * E * SCALE * (mine.abs() @ k.abs().t())).max().item()
                want = torch.softmax(mine @ k.t() * SCALE, dim=-1) @ v
                tol = want * (2 * ds + (4 * L + 300) * E) + half_step(dt) * want * 1.01
                if dt == F16:
                    tol = tol + L * 2.0 ** -32 * v.max() + 2.0 ** -25
                check(got[b, h * G:(h + 1) * G], want, tol, (name, b, h))
