"""The operators over uncompressed caches refuse what they cannot run, before anything is launched (CPU)."""
import pytest
import torch

from starkv_serve import _hip
from starkv_serve.kernels import model_ops as mo
from starkv_serve.kernels.evict import evict, paged_decode_weighted
from starkv_serve.kernels.sparse_decode import (BlockSelection, key_bounds_like, paged_decode_sparse, select_blocks,
                                                update_key_bounds)

BF16 = torch.bfloat16


def tensors(n=2, H=4, Hkv=2, bs=16, blocks=6):
    return dict(q=torch.zeros(n, H, 128, dtype=BF16), kc=torch.zeros(blocks, bs, Hkv, 128, dtype=BF16),
                vc=torch.zeros(blocks, bs, Hkv, 128, dtype=BF16), bt=torch.zeros(n, 3, dtype=torch.int32),
                sl=torch.ones(n, dtype=torch.int32), w=torch.zeros(n, Hkv, 48),
                sel=torch.zeros(n, Hkv, 2, dtype=torch.int32))


def test_cpu_tensors_are_refused():
    x = tensors()
    b = key_bounds_like(x["kc"])
    assert b.shape == (6, 2, 2, 128) and b.dtype == BF16
    table, pos, w = torch.zeros(9, 128), torch.zeros(2, dtype=torch.int64), torch.ones(128)
    for call in (lambda: update_key_bounds(x["kc"], b, x["bt"], x["sl"], 1),
                 lambda: select_blocks(x["q"], b, x["bt"], x["sl"], 48, 16, 2),
                 lambda: paged_decode_sparse(x["q"], x["kc"], x["vc"], x["bt"], x["sl"], x["sel"], 0.1),
                 lambda: paged_decode_weighted(x["q"], x["kc"], x["vc"], x["bt"], x["sl"], 48, 0.1, x["w"]),
                 lambda: evict(x["kc"], x["vc"], x["bt"], x["sl"], x["w"], 40),
                 lambda: mo.norm_rope(pos, x["q"], None, table, w, None, 1e-6),
                 lambda: mo.norm_rope_write(pos, x["q"], x["q"][:, :2], x["q"][:, :2], table, w, w, 1e-6, x["kc"], x["vc"],
                                            pos, False, False)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_gradients_are_refused():
    with pytest.raises(NotImplementedError, match="no gradient"):
        _hip.refuse_grad("evict", torch.zeros(1), torch.zeros(1, requires_grad=True))
    with torch.no_grad():
        _hip.refuse_grad("evict", torch.zeros(1, requires_grad=True))


def test_block_selection_keeps_the_own_block():
    BlockSelection(3, 1, 2)
    for args in ((2, 1, 2), (3, 1, 0), (3, -1, 1)):
        with pytest.raises(ValueError):
            BlockSelection(*args)


# C ABI: one argument wrong at a time; nothing is launched, so the pointers need not be the GPU's.
P = 4096  # a 16-byte aligned address that is never read
GOOD = {
    "starkv_key_bounds": dict(stream=None, k=P, c0=4096, c1=256, c2=128, dtype=2, bs=16, blocks=6, bounds=P, b0=512, b1=256,
                              b2=128, bt=P, t0=3, t1=1, width=3, lens=P, n=2, heads=2, new=1),
    "starkv_select_blocks": dict(stream=None, q=P, q0=512, q1=128, bounds=P, b0=512, b1=256, b2=128, dtype=2, bs=16, blocks=6,
                                 bt=P, t0=3, t1=1, width=3, lens=P, n=2, hq=4, heads=2, span=48, keep=2, sink=1, recent=1,
                                 sel=P, ws=P, bytes=1 << 20),
    "starkv_sparse_decode": dict(stream=None, q=P, q0=512, q1=128, k=P, v=P, c0=4096, c1=256, c2=128, dtype=2, bs=16, blocks=6,
                                 bt=P, t0=3, t1=1, width=3, lens=P, n=2, hq=4, heads=2, sel=P, s0=4, s1=2, keep=2, scale=0.1,
                                 out=P, o0=512, o1=128, ws=P, bytes=1 << 20),
    "starkv_weighted_decode": dict(stream=None, q=P, q0=512, q1=128, k=P, v=P, c0=4096, c1=256, c2=128, dtype=2, bs=16,
                                   blocks=6, bt=P, t0=3, t1=1, width=3, lens=P, n=2, hq=4, heads=2, span=48, scale=0.1, w=P,
                                   w0=96, w1=48, wlen=48, out=P, o0=512, o1=128, ws=P, bytes=1 << 20),
    "starkv_evict": dict(stream=None, k=P, v=P, c0=4096, c1=256, c2=128, dtype=2, bs=16, blocks=6, bt=P, t0=3, t1=1, width=3,
                         lens=P, n=2, heads=2, w=P, w0=96, w1=48, wlen=48, keep=40, sink=4, recent=32, nl=P, nw=P, ws=P,
                         bytes=1 << 20),
}
COMMON = [("dtype", 0, b"bf16 or fp16"), ("bs", 24, b"block_size"), ("bs", 8, b"block_size"), ("blocks", 0, b"empty"),
          ("width", 0, b"empty"), ("n", -1, b"n="), ("n", 65536, b"n="), ("lens", None, b"null"), ("bt", None, b"null")]
BAD = {
    "starkv_key_bounds": [("c1", 4, b"16-byte"), ("bounds", P + 8, b"16-byte"), ("new", -1, b"max_new"), ("heads", 0, b"heads")],
    "starkv_select_blocks": [("keep", 0, b"keep"), ("recent", 2, b"keep"), ("sink", -1, b"keep"), ("hq", 5, b"query heads"),
                             ("hq", 0, b"query heads"), ("span", 0, b"max_seq_len"), ("bytes", 16, b"workspace"),
                             ("sink", 2 ** 31 - 1, b"keep"), ("q0", 4, b"16-byte")],
    "starkv_sparse_decode": [("keep", 0, b"keep"), ("hq", 34, b"query heads"), ("hq", 3, b"query heads"), ("sel", None, b"null"),
                             ("keep", 2 ** 31 - 1, b"keep"), ("c2", 4, b"16-byte"), ("k", P + 2, b"16-byte")],
    "starkv_weighted_decode": [("span", 0, b"max_seq_len"), ("wlen", 47, b"weights"), ("w", None, b"weights"),
                               ("bytes", 1024, b"workspace"), ("hq", 34, b"query heads"), ("out", None, b"null")],
    "starkv_evict": [("keep", 35, b"keep"), ("keep", 0, b"keep"), ("recent", -1, b"keep"), ("bytes", 16, b"workspace"),
                     ("wlen", 0, b"empty"), ("c0", 4, b"16-byte"), ("nw", None, b"null")],
}


@pytest.mark.parametrize("name,arg,value,message", [(n, *b) for n in GOOD for b in COMMON + BAD[n]])
def test_bad_arguments_return_errors(name, arg, value, message):
    L = _hip.lib()
    args = dict(GOOD[name])
    assert len(args) == len(_hip.SIGNATURES[name][1])
    args[arg] = value
    assert getattr(L, name)(*args.values()) != 0
    assert message in L.starkv_last_error(), L.starkv_last_error()


def test_no_requests_need_nothing():
    L = _hip.lib()
    for name, good in GOOD.items():
        assert getattr(L, name)(*dict(good, n=0).values()) == 0, name


def test_norm_rope_refuses_bad_arguments():
    L = _hip.lib()
    good = dict(stream=None, q=P, q0=512, q1=128, k=P, k0=512, k1=128, v=P, v0=512, v1=128, dtype=2, T=1, H=4, Hkv=2, qw=P,
                kw=P, wdt=2, eps=1e-6, pos=P, bits=64, cs=P, cs0=128, csdt=2, rows=9, qo=P, ko=P, kc=None, vc=None, c0=0, c1=0,
                c2=0, bs=0, nb=0, slots=None, sbits=64, k16=None, v16=None)
    assert len(good) == len(_hip.SIGNATURES["starkv_norm_rope_qkv"][1])
    for arg, value, message in (("qw", None, b"weight"), ("kw", None, b"weight"), ("wdt", 7, b"weights"), ("kw", P + 4, b"weights"),
                                ("eps", -1.0, b"eps"), ("eps", float("nan"), b"eps"), ("dtype", 9, b"bf16"), ("q0", 4, b"16-byte"),
                                ("ko", None, b"K and V"), ("kc", P, b"K and V"), ("bits", 16, b"int32"), ("rows", 0, b"null")):
        assert L.starkv_norm_rope_qkv(*dict(good, **{arg: value}).values()) != 0, arg
        assert message in L.starkv_last_error(), (arg, L.starkv_last_error())
    assert L.starkv_norm_rope_qkv(*dict(good, T=0).values()) == 0


def test_model_options_that_do_not_go_together():
    from starkv_serve import model as M

    class Compressed:
        @staticmethod
        def is_compressed(li):
            return li == 0

    shape = M.LlamaShape(hidden_size=64, num_layers=1, num_heads=1, num_kv_heads=1, intermediate_size=64, vocab_size=10)
    normed = M.LlamaShape(**{**shape.__dict__, "qk_norm": True})
    with pytest.raises(ValueError, match="sparse or weigh"):
        M.StarKVLlamaForCausalLM(shape, None, 32, "cpu", sparse=BlockSelection(4), weigh=True)
    with pytest.raises(NotImplementedError, match="qk_norm"):
        M.StarKVLlamaForCausalLM(normed, Compressed, 32, "cpu")
    with pytest.raises(NotImplementedError, match="weigh"):
        M.StarKVLlamaForCausalLM(shape, Compressed, 32, "cpu", weigh=True)
    model = M.StarKVLlamaForCausalLM(normed, None, 32, "cpu", weigh=True)
    assert model.layers[0].q_norm.shape == model.layers[0].k_norm.shape == (128,)
    with pytest.raises(ValueError, match="num_requests"):
        model.allocate_kv_cache(4)
    with pytest.raises(RuntimeError, match="weigh=True"):
        model.evict(torch.zeros(1, 2, dtype=torch.int32), torch.ones(1), 16)
    model.allocate_kv_cache(4, 16, 3)
    assert model.weights[0].shape == (3, 1, 32)
    plain = M.StarKVLlamaForCausalLM(shape, None, 32, "cpu", sparse=BlockSelection(4))
    plain.allocate_kv_cache(4)
    assert plain.key_bounds[0].shape == (4, 1, 2, 128) and plain.weights == [] and plain.layers[0].q_norm is None


def test_decode_metadata_of_cut_caches():
    from starkv_serve import model as M
    bt = torch.arange(8, dtype=torch.int32).view(2, 4)
    md = M.decode_metadata(bt, torch.tensor([50, 20]), 16, 64, torch.tensor([17, 20], dtype=torch.int32))
    assert md.slot_mapping.tolist() == [1 * 16 + 1, 5 * 16 + 4] and md.seq_lens.tolist() == [18, 21]
    assert M.decode_metadata(bt, torch.tensor([50, 20]), 16, 64).seq_lens.tolist() == [51, 21]
