"""The model over 8-bit caches and through windows: prompts, eager steps and captured ones. Caches are what the plain
quantiser makes of the step's keys and values, value for value; attention is compared with float64 over the caches as
the step left them (tolerances of test_gpu_cache8 and test_gpu_window); captured steps equal the eager ones bit for bit."""
import pytest
import torch

import test_gpu_cache8 as C8
import test_gpu_window as W
from cache8_plain import SCALE, Plain8
from starkv_serve import model as M
from starkv_serve.kernels.cache8 import Cache8
from starkv_serve.kernels.sparse_decode import BlockSelection
from starkv_serve.kernels.window import Window

pytestmark = pytest.mark.gpu

BF16, F16, I8, F8 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn
PROMPTS = [100, 9, 260]
SPAN = 512


def build(cuda, dtype=BF16, qk_norm=True, heads=(8, 2), **kw):
    shape = M.LlamaShape(hidden_size=512, num_layers=3, num_heads=heads[0], num_kv_heads=heads[1], intermediate_size=1024, vocab_size=1000,
                         qk_norm=qk_norm)
    model = M.StarKVLlamaForCausalLM(shape, None, SPAN, cuda, dtype=dtype, seed=3, **kw)
    model.allocate_kv_cache(len(PROMPTS) * SPAN // 16 + 1, 16)
    bt = (torch.randperm(len(PROMPTS) * SPAN // 16, generator=torch.Generator().manual_seed(4)) + 1).int().view(len(PROMPTS), -1).to(cuda)
    return model, bt


def prefill(model, bt, capture=None):
    md, pos = M.prefill_metadata(bt, PROMPTS, 16)
    tokens = torch.randint(0, 1000, (sum(PROMPTS),), generator=torch.Generator().manual_seed(5)).to(bt.device)
    return model.prefill_step(tokens, pos, md, capture).argmax(-1), md


@pytest.mark.parametrize("code,window,dtype,qk_norm", [(I8, None, BF16, False), (F8, Window(40, 4), F16, True), (I8, Window(16, 0), BF16, True),
                                                       (F8, None, BF16, True)])
def test_8_bit_caches(cuda, code, window, dtype, qk_norm):
    model, bt = build(cuda, dtype, qk_norm, cache8=code, window=window)
    assert all(isinstance(c, Cache8) and c.dtype == code for c in model.kv_caches)
    assert model.cache_bytes_per_token() == 3 * 2 * 2 * 128
    plain, capture = [Plain8(c) for c in model.kv_caches], []
    tokens, md = prefill(model, bt, capture)
    for c in capture:
        li = c["layer"]
        plain[li].write(c["k"], c["v"], md.slot_mapping)
        assert plain[li].same(model.kv_caches[li])
        W.prompts_close(c["out"], c["q"], c["k"], c["v"], PROMPTS, window or Window(SPAN), li)
    positions = torch.tensor(PROMPTS, device=cuda)
    for step in range(20):  # through the ends of blocks
        md, capture = M.decode_metadata(bt, positions, 16, SPAN), []
        logits = model.decode_step(tokens, positions, md, capture)
        assert logits.isfinite().all()
        lens = [L + step + 1 for L in PROMPTS]
        for c in capture:
            li = c["layer"]
            plain[li].write(c["k"], c["v"], md.slot_mapping)
            assert plain[li].same(model.kv_caches[li])
            if step in (0, 3, 4, 6, 7, 19):
                C8.close(c["out"], c["q"], model.kv_caches[li], bt, lens, window, what=(li, step))
        tokens, positions = logits.argmax(-1), positions + 1


def test_windows_of_16_bit_caches(cuda):
    w = Window(30, 3)
    model, bt = build(cuda, window=w)
    capture = []
    tokens, _ = prefill(model, bt, capture)
    for c in capture:
        W.prompts_close(c["out"], c["q"], c["k"], c["v"], PROMPTS, w, c["layer"])
    positions = torch.tensor(PROMPTS, device=cuda)
    for step in range(9):
        capture = []
        logits = model.decode_step(tokens, positions, M.decode_metadata(bt, positions, 16, SPAN), capture)
        for c in capture:
            W.close(c["out"], c["q"], *model.kv_caches[c["layer"]], bt, [L + step + 1 for L in PROMPTS], w, (c["layer"], step))
        tokens, positions = logits.argmax(-1), positions + 1


@pytest.mark.parametrize("kw", [dict(cache8=I8), dict(cache8=F8, window=Window(24, 4)), dict(window=Window(24, 4))])
def test_captured_steps_are_the_eager_ones(cuda, kw):
    runs = []
    for captured in (True, False):
        model, bt = build(cuda, **kw)
        tokens, _ = prefill(model, bt)
        positions = torch.tensor(PROMPTS, device=cuda)
        graph = M.DecodeGraph(model, bt, tokens, positions) if captured else None
        logits = []
        for _ in range(20):
            if captured:
                graph.replay()
                logits.append(graph.logits.clone())
            else:
                out = model.decode_step(tokens, positions, M.decode_metadata(bt, positions, 16, SPAN), in_graph=True)
                logits.append(out)
                tokens, positions = out.argmax(-1), positions + 1
            torch.cuda.synchronize()
        runs.append((logits, [t for c in model.kv_caches for t in (c.tensors if isinstance(c, Cache8) else c)]))
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.equal(a, b)
    for a, b in zip(runs[0][1], runs[1][1]):
        assert torch.equal(a.view(I8), b.view(I8))


def test_a_rotation_of_the_callers(cuda):
    """Rows that the caller rotates go into the 8-bit cache as they are."""
    model, bt = build(cuda, cache8=I8)
    apply = model.rotary.apply
    model.rotary.apply = lambda positions, x: apply(positions, x)
    plain, capture = [Plain8(c) for c in model.kv_caches], []
    _, md = prefill(model, bt, capture)
    for c in capture:
        plain[c["layer"]].write(c["k"], c["v"], md.slot_mapping)
        assert plain[c["layer"]].same(model.kv_caches[c["layer"]])
        W.prompts_close(c["out"], c["q"], c["k"], c["v"], PROMPTS, Window(SPAN), c["layer"])


def test_attention_only(cuda):
    """The attention ops of a step by themselves, as benchmarks run them."""
    model, bt = build(cuda, cache8=F8, window=Window(64, 2))
    prefill(model, bt)
    positions = torch.tensor(PROMPTS, device=cuda)
    hidden = torch.randn(3, 512, generator=torch.Generator().manual_seed(6)).to(BF16).to(cuda)
    md = M.decode_metadata(bt, positions, 16, SPAN)
    plain = [Plain8(c) for c in model.kv_caches]
    inputs = model.attention_inputs(hidden, positions)
    model.attention_only(hidden, inputs, md)
    for p, c, (_, k, v) in zip(plain, model.kv_caches, inputs):
        p.write(k, v, md.slot_mapping)
        assert p.same(c)


def test_a_window_of_everything_is_the_whole_attention(cuda):
    a, bt = build(cuda, qk_norm=False)
    b, _ = build(cuda, qk_norm=False, window=Window(SPAN))
    ca, cb = [], []
    prefill(a, bt, ca), prefill(b, bt, cb)
    x, y = ca[0]["out"].float(), cb[0]["out"].float()
    assert (x - y).abs().max() <= 3 * 2.0 ** -8 * x.abs().max()


def test_steps_without_requests(cuda):
    model, bt = build(cuda, cache8=I8, window=Window(8, 1))
    none = torch.zeros(0, dtype=torch.int64, device=cuda)
    assert model.decode_step(none, none, M.decode_metadata(bt[:0], none, 16, SPAN)).shape == (0, 1000)


def test_options_that_do_not_go_together():
    shape = M.LlamaShape(hidden_size=64, num_layers=1, num_heads=1, num_kv_heads=1, intermediate_size=64, vocab_size=10)
    for kw in (dict(cache8=I8, weigh=True), dict(window=Window(4), weigh=True), dict(cache8=F8, sparse=BlockSelection(4)),
               dict(window=Window(4), sparse=BlockSelection(4))):
        with pytest.raises(ValueError, match="16 bits"):
            M.StarKVLlamaForCausalLM(shape, None, 32, "cpu", **kw)
    with pytest.raises(ValueError, match="int8"):
        M.StarKVLlamaForCausalLM(shape, None, 32, "cpu", cache8=torch.uint8)


@pytest.mark.parametrize("kv_quant", [False, True])
def test_beside_compressed_layers(cuda, tmp_path, kv_quant):
    """A checkpoint's compressed layers decode as ever, its other layers over 8-bit caches through a window; captured too."""
    import numpy as np

    from starkv_serve import checkpoint as ck
    from test_gpu_decode import assert_close
    from test_gpu_model import SHAPE, decode_layer_truth
    path, w, n = str(tmp_path / "fused_weights.pt"), Window(48, 4), len(PROMPTS)
    ck.write_fused_checkpoint(path, SHAPE.num_layers, SHAPE.num_kv_heads, SHAPE.head_dim, SHAPE.hidden_size,
                              {1: ([16, 32, 16, 48], 64), 2: ([32, 16, 16, 16], 96)}, seed=11)
    c = ck.load_fused_checkpoint(path, SHAPE.num_layers, SHAPE.num_kv_heads, SHAPE.head_dim, dtype=BF16, kv_quant=kv_quant)
    models = []
    for _ in range(2):
        model = M.StarKVLlamaForCausalLM(SHAPE, c, SPAN, cuda, seed=12, cache8=I8, window=w)
        model.allocate_kv_cache(n * SPAN // 16 + 1)
        bt = (torch.randperm(n * SPAN // 16, generator=torch.Generator().manual_seed(13)) + 1).int().view(n, -1).to(cuda)
        tokens, _ = prefill(model, bt)
        models.append(model)
    model, positions = models[0], torch.tensor(PROMPTS, device=cuda)
    graph = M.DecodeGraph(models[1], bt, tokens, positions)
    for step in range(4):
        md, capture = M.decode_metadata(bt, positions, 16, SPAN), []
        logits = model.decode_step(tokens, positions, md, capture, in_graph=True)
        lens = [L + step + 1 for L in PROMPTS]
        for x in capture:
            li = x["layer"]
            if model.layers[li].compressed:
                assert_close(x["out"], decode_layer_truth(model, x, bt.cpu().numpy(), np.array(lens)), (step, li))
            else:
                C8.close(x["out"], x["q"], model.kv_caches[li], bt, lens, w, what=(step, li))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graph.logits, logits)
        tokens, positions = logits.argmax(-1), positions + 1
