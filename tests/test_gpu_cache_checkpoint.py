"""Decode steps over selected blocks in the uncompressed layers of a STAR-KV checkpoint, whose compressed layers decode as
ever: every layer's attention against its float64 form, and captured steps against eager ones."""
import numpy as np
import pytest
import torch

from starkv_serve import checkpoint as ck
from starkv_serve import model as M
from starkv_serve.kernels.sparse_decode import BlockSelection
from test_gpu_cache_ops import attention64, check, rows_of, select_plain
from test_gpu_decode import assert_close
from test_gpu_model import SHAPE, decode_layer_truth

pytestmark = pytest.mark.gpu

PROMPTS, SPAN, KEEP = [100, 37, 260], 512, 5


def build(cuda, tmp_path, kv_quant):
    path = str(tmp_path / "fused_weights.pt")
    ck.write_fused_checkpoint(path, SHAPE.num_layers, SHAPE.num_kv_heads, SHAPE.head_dim, SHAPE.hidden_size,
                              {1: ([16, 32, 16, 48], 64), 2: ([32, 16, 16, 16], 96)}, seed=11)
    c = ck.load_fused_checkpoint(path, SHAPE.num_layers, SHAPE.num_kv_heads, SHAPE.head_dim, dtype=torch.bfloat16,
                                 kv_quant=kv_quant)
    model = M.StarKVLlamaForCausalLM(SHAPE, c, SPAN, cuda, seed=12, sparse=BlockSelection(KEEP, 1, 2))
    model.allocate_kv_cache(len(PROMPTS) * SPAN // 16 + 1)
    g = torch.Generator().manual_seed(13)
    bt = (torch.randperm(len(PROMPTS) * SPAN // 16, generator=g) + 1).int().view(len(PROMPTS), -1).to(cuda)
    md, positions = M.prefill_metadata(bt, PROMPTS, 16)
    tokens = torch.randint(0, SHAPE.vocab_size, (sum(PROMPTS),), generator=g).to(cuda)
    return model, bt, model.prefill_step(tokens, positions, md).argmax(-1)


@pytest.mark.parametrize("kv_quant", [False, True])
def test_selected_blocks_beside_compressed_layers(cuda, tmp_path, kv_quant):
    model, bt, tokens = build(cuda, tmp_path, kv_quant)
    assert [b is None for b in model.key_bounds] == [False, True, True, False]
    positions = torch.tensor(PROMPTS, device=cuda)
    for step in range(3):
        md, capture = M.decode_metadata(bt, positions, 16, SPAN), []
        logits = model.decode_step(tokens, positions, md, capture)
        lens = [L + step + 1 for L in PROMPTS]
        assert torch.isfinite(logits).all() and len(capture) == SHAPE.num_layers
        for c in capture:
            li = c["layer"]
            if model.layers[li].compressed:
                truth = decode_layer_truth(model, c, bt.cpu().numpy(), np.array(lens))
                assert_close(c["out"], truth, (step, li))
                continue
            kc, vc = model.kv_caches[li]
            picks = select_plain(c["q"], model.key_bounds[li], bt, lens, SPAN, 16, KEEP, 1, 2)
            for b, L in enumerate(lens):
                for h in range(SHAPE.num_kv_heads):
                    at = [t for j in picks[b, h].tolist() if j >= 0 for t in range(16 * j, min(L, 16 * j + 16))]
                    want, tol, _, _ = attention64(c["q"][b, h:h + 1].cpu(), rows_of(kc, bt, b, h, at), rows_of(vc, bt, b, h, at),
                                                  torch.bfloat16)
                    check(c["out"][b, h:h + 1], want, tol, (step, li, b, h))
        tokens, positions = logits.argmax(-1), positions + 1


def test_captured_steps_beside_compressed_layers(cuda, tmp_path):
    model, bt, tokens = build(cuda, tmp_path, False)
    twin, _, _ = build(cuda, tmp_path, False)
    positions = torch.tensor(PROMPTS, device=cuda)
    graph = M.DecodeGraph(model, bt, tokens, positions)
    for _ in range(4):
        graph.replay()
        md = M.decode_metadata(bt, positions, 16, SPAN)
        want = twin.decode_step(tokens, positions, md, in_graph=True)
        torch.cuda.synchronize()
        assert torch.equal(graph.logits, want)
        tokens, positions = want.argmax(-1), positions + 1
