"""8-bit caches and windows on the GPU, at the ends of what their operators take."""
import pytest
import torch

from cache8_plain import D, SCALE, Plain8
from starkv_serve import _hip
from starkv_serve.kernels.cache8 import Cache8, paged_decode_8, read_kv8, write_kv8
from starkv_serve.kernels.window import Window, paged_decode_window
from test_gpu_cache8 import rows

pytestmark = pytest.mark.gpu

BF16, I8, F8 = torch.bfloat16, torch.int8, torch.float8_e4m3fn


def test_caches_without_heads_are_refused(cuda):
    """By an error: a number of query heads is divided by theirs."""
    c = Cache8.zeros(4, 16, 0, I8, cuda)
    kc = torch.zeros(4, 16, 0, D, dtype=BF16, device=cuda)
    bt, sl = torch.zeros(2, 2, dtype=torch.int32, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    for heads in (0, 4):
        q = torch.zeros(2, heads, D, dtype=BF16, device=cuda)
        with pytest.raises(RuntimeError, match="KV heads"):
            paged_decode_8(q, c, bt, sl, 32, SCALE)
        with pytest.raises(RuntimeError, match="KV heads"):
            paged_decode_window(q, kc, kc, bt, sl, 32, SCALE, Window(8))
    rows = torch.zeros(2, 0, D, dtype=BF16, device=cuda)
    for call in (lambda: write_kv8(rows, rows, c, sl), lambda: read_kv8(c, sl)):
        with pytest.raises(RuntimeError, match="num_kv_heads"):
            call()


@pytest.mark.parametrize("code", [I8, F8])
@pytest.mark.parametrize("nb,bs,H,wide", [(70000, 64, 4, 1), (150000, 16, 8, 1), (9000, 1024, 2, 1), (300000, 16, 4, 3)])
def test_larger_writes_past_31_bits(cuda, nb, bs, H, wide, code):
    """More tokens than a workgroup looks through, into blocks at the far end of a cache of more than 2^31 bytes a tensor:
    whole blocks in any order, blocks that go on with larger values, and a token each of many blocks."""
    g = torch.Generator().manual_seed(nb + H)
    k, v = (torch.zeros(nb, H, bs, D, dtype=I8, device=cuda).view(code).transpose(1, 2) for _ in range(2))
    assert (nb - 1) * k.stride(0) > 2 ** 31
    c = Cache8(k, v, torch.full((nb, H, 2 * wide), -126, dtype=I8, device=cuda)[..., :2])
    fewest = next(n for n in range(1, 1 << 20) if _hip.lib().starkv_write_kv8_workspace_bytes(n, nb, bs) > 0)
    full = -(-(fewest + 40) // bs) + 1
    single = fewest + 76 if bs <= 64 else 0
    blocks = torch.cat([torch.tensor([nb - 1, 2, nb - 2, nb // 2]),
                        torch.randperm(nb - 2 - nb // 2 - 1, generator=g)[:full + single] + nb // 2 + 1])
    used = blocks[:full]  # of the whole writes
    small = Cache8(*(torch.zeros(len(blocks), H, bs, D, dtype=I8).view(code).transpose(1, 2) for _ in range(2)),
                   torch.full((len(blocks), H, 2), -126, dtype=I8))
    want = Plain8(small)

    def write(at, places, scale):
        """Tokens at `places` of blocks[at]."""
        n = len(at)
        assert n >= fewest
        kk, vv = rows(n, H, BF16, cuda, g, strided=False)
        kk.mul_(scale)
        write_kv8(kk, vv, c, (blocks[at] * bs + places).to(cuda))
        want.write(kk, vv, at * bs + places)
        there = blocks.to(cuda)
        assert want.same(Cache8(c.k[there], c.v[there], c.exponents[there]))

    token = torch.arange(full * bs)
    order = torch.randperm(full * bs - 7, generator=g) if bs == 16 else torch.arange(full * bs - 7)
    write(token[order] // bs, token[order] % bs, 1.0)
    later = token[token % bs >= 3]
    if len(later) >= fewest:
        write(later // bs, later % bs, 2.0 ** 5)
    if single:
        at = torch.arange(len(blocks))[-single:]
        write(at, torch.randint(0, bs, (single,), generator=g), 1.0)
        write(at, torch.randint(1, bs, (single,), generator=g), 2.0 ** 3)
    assert int((c.exponents.amax(dim=(1, 2)) > -126).sum()) == len(used) + single  # no other block was touched
