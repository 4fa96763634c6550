"""8-bit caches and attention through a window refuse what they cannot run, before anything is launched (CPU)."""
import pytest
import torch

from cache8_plain import Plain8, exponent_of, grid, nearest, visible
from starkv_serve import _hip
from starkv_serve.kernels.cache8 import Cache8, paged_decode_8, read_kv8, write_kv8
from starkv_serve.kernels.prefill import prefill_attention
from starkv_serve.kernels.window import Window, paged_decode_window

BF16, I8, F8 = torch.bfloat16, torch.int8, torch.float8_e4m3fn


def test_a_new_cache_holds_zeros():
    for dtype in (I8, F8):
        c = Cache8.zeros(5, 32, 3, dtype, "cpu")
        assert c.k.shape == c.v.shape == (5, 32, 3, 128) and c.dtype == dtype and c.exponents.shape == (5, 3, 2)
        assert c.k.stride() == c.v.stride() == (3 * 32 * 128, 128, 32 * 128, 1)  # a head's rows of a block lie together
        assert (c.exponents == -126).all() and (Plain8(c).rows(0, torch.arange(160)) == 0).all()
    for dtype in (torch.uint8, torch.float16, torch.float8_e5m2):
        with pytest.raises(ValueError, match="int8"):
            Cache8.zeros(5, 32, 3, dtype, "cpu")
    for size in (8, 24, 2048, 0):
        with pytest.raises(ValueError, match="blocks of"):
            Cache8.zeros(5, size, 3, I8, "cpu")


def test_windows():
    assert visible(10, Window(3, 2)) == [0, 1, 7, 8, 9] and visible(2, Window(3, 2)) == [0, 1] and visible(0, Window(1)) == []
    for args in ((0, 0), (-1, 2), (4, -1), (2 ** 31, 0), (4, 2 ** 31)):
        with pytest.raises(ValueError):
            Window(*args)


def test_the_plain_quantiser():
    """The tests' own quantiser against torch's conversions and small cases by hand."""
    assert [exponent_of(x, I8) for x in (0.0, 1.0, 127.0, 127.5, 2.0 ** -130)] == [-126, -6, 0, 1, -126]
    assert [exponent_of(x, F8) for x in (448.0, 449.0, 1.75, 3.4e38)] == [0, 1, -8, 120]
    x = torch.linspace(-460, 460, 40001, dtype=torch.float64).clamp(-448, 448)
    assert torch.equal(nearest(x, F8), x.float().to(F8).double())
    small = torch.linspace(-0.05, 0.05, 40001, dtype=torch.float64)
    assert torch.equal(nearest(small, F8), small.to(F8).double())
    y = x.clamp(-127, 127)
    assert torch.equal(nearest(y, I8), y.round())
    assert grid(F8).numel() == 253 and grid(I8).numel() == 255


def tensors(n=2, H=4, Hkv=2, bs=16, blocks=6):
    return dict(q=torch.zeros(n, H, 128, dtype=BF16), k=torch.zeros(n, Hkv, 128, dtype=BF16), c=Cache8.zeros(blocks, bs, Hkv, I8, "cpu"),
                kc=torch.zeros(blocks, bs, Hkv, 128, dtype=BF16), bt=torch.zeros(n, 3, dtype=torch.int32),
                sl=torch.ones(n, dtype=torch.int32), slots=torch.arange(n))


def test_cpu_tensors_are_refused():
    x = tensors()
    for call in (lambda: write_kv8(x["k"], x["k"], x["c"], x["slots"]), lambda: read_kv8(x["c"], x["slots"]),
                 lambda: paged_decode_8(x["q"], x["c"], x["bt"], x["sl"], 48, 0.1),
                 lambda: paged_decode_window(x["q"], x["kc"], x["kc"], x["bt"], x["sl"], 48, 0.1, Window(4)),
                 lambda: prefill_attention(x["q"], x["k"], x["k"], [2], 0.1, window=Window(4))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


# C ABI: one argument wrong at a time; nothing is launched, so the pointers need not be the GPU's.
P = 4096  # a 16-byte aligned address that is never read
GOOD = {
    "starkv_window_decode": dict(stream=None, q=P, q0=512, q1=128, k=P, v=P, c0=4096, c1=256, c2=128, dtype=2, bs=16, blocks=6, bt=P, t0=3,
                                 t1=1, width=3, lens=P, n=2, hq=4, heads=2, span=48, window=8, sinks=1, scale=0.1, out=P, o0=512, o1=128,
                                 ws=P, bytes=1 << 20),
    "starkv_prefill_window": dict(stream=None, q=P, q0=512, q1=128, dtype=2, k=P, k0=256, k1=128, kdt=1, v=P, v0=256, v1=128, cu=P, blk=P, blocks=3, hq=4, heads=2,
                                  D=128, window=8, sinks=1, scale=0.1, out=P, o0=512, o1=128, odt=2),
    "starkv_write_kv8": dict(stream=None, key=P, k0=256, k1=128, v=P, v0=256, v1=128, dtype=2, kc=P, vc=P, c0=4096, c1=256, c2=128, code=3, ex=P,
                             x0=4, x1=2, bs=16, blocks=6, slots=P, bits=64, n=2, heads=2, ws=P, bytes=1 << 20),
    "starkv_read_kv8": dict(stream=None, kc=P, vc=P, c0=4096, c1=256, c2=128, code=4, ex=P, x0=4, x1=2, bs=16, blocks=6, slots=P, bits=32, n=2,
                            heads=2, ko=P, vo=P, odt=1),
    "starkv_decode_kv8": dict(stream=None, q=P, q0=512, q1=128, dtype=2, kc=P, vc=P, c0=4096, c1=256, c2=128, code=3, ex=P, x0=4, x1=2, bs=16,
                              blocks=6, bt=P, t0=3, t1=1, width=3, lens=P, n=2, hq=4, heads=2, span=48, window=0, sinks=0, scale=0.1, out=P,
                              o0=512, o1=128, ws=P, bytes=1 << 20),
}
CACHE8 = [("code", 2, b"int8 or e4m3"), ("bs", 24, b"block_size"), ("bs", 2048, b"block_size"), ("blocks", 0, b"empty"), ("c1", 8, b"16-byte"),
          ("kc", P + 8, b"16-byte"), ("ex", None, b"null"), ("vc", None, b"null")]
DECODE = [("n", -1, b"n="), ("n", 65536, b"n="), ("span", 0, b"max_seq_len"), ("hq", 34, b"query heads"), ("hq", 3, b"query heads"),
          ("dtype", 0, b"bf16 or fp16"), ("width", 0, b"empty"), ("lens", None, b"null"), ("bytes", 16, b"workspace"), ("q0", 4, b"16-byte"),
          ("window", -1, b"window"), ("sinks", -1, b"sinks")]
BAD = {
    "starkv_window_decode": [*DECODE, ("window", 0, b"window"), ("c2", 4, b"16-byte"), ("k", P + 2, b"16-byte")],
    "starkv_prefill_window": [("window", 0, b"window"), ("sinks", -1, b"sinks"), ("D", 64, b"head_size"), ("kdt", 0, b"fp16"), ("q", None, b"null"),
                              ("k0", 128, b"share strides"), ("q0", 4, b"aligned"), ("o0", 2, b"aligned")],
    "starkv_write_kv8": [*CACHE8, ("n", -1, b"n="), ("heads", 0, b"heads"), ("heads", 65536, b"heads"), ("dtype", 0, b"bf16 or fp16"),
                         ("bits", 16, b"int32 or int64"), ("k1", 4, b"16-byte"), ("ws", P + 4, b"workspace"), ("bytes", 0, b"workspace")],
    "starkv_read_kv8": [*CACHE8, ("odt", 3, b"bf16, fp16 or fp32"), ("ko", P + 4, b"16-byte"), ("bits", 8, b"int32 or int64"), ("n", -1, b"n=")],
    "starkv_decode_kv8": [*CACHE8, *DECODE],
}


@pytest.mark.parametrize("name,change", [(n, c) for n, cs in BAD.items() for c in cs])
def test_c_abi_refuses(name, change):
    L = _hip.lib()
    key, value, message = change
    args = dict(GOOD[name])
    args["n" if "n" in args else "blocks"] = max(args.get("n", 3), 1)
    if key == "bytes" and name == "starkv_decode_kv8":
        args["span"] = 1 << 16  # several splits, which need room
    if key == "bytes" and name == "starkv_write_kv8":
        args["n"] = 1300  # the map of slots
    if key == "bytes" and name == "starkv_window_decode":
        args.update(span=1 << 16, window=1 << 15)
    args[key] = value
    assert getattr(L, name)(*args.values()) != 0
    assert message in L.starkv_last_error(), L.starkv_last_error()


def test_workspaces():
    L = _hip.lib()
    assert L.starkv_write_kv8_workspace_bytes(1024, 1000, 16) == 0
    assert L.starkv_write_kv8_workspace_bytes(1025, 1000, 16) == 64000
    assert L.starkv_write_kv8_workspace_bytes(10 ** 6, 2 ** 27, 16) == 2 ** 33
    one = L.starkv_decode_kv8_workspace_bytes(1, 32, 32, 1 << 20, 0, 0)
    assert one > L.starkv_decode_kv8_workspace_bytes(1, 32, 32, 1 << 20, 64, 4)
    for n, window, sinks in ((0, 0, 0), (1, -1, 0), (1, 4, -1)):
        assert L.starkv_decode_kv8_workspace_bytes(n, 32, 32, 100, window, sinks) == 256
