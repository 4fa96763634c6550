"""A session that cuts hold to a budget goes past max_model_len tokens, captured as eager, to the end of its rotary table."""
import pytest
import torch

from starkv_serve import model as M
from test_gpu_cache_model import PROMPTS, SPAN, build, check_attention, decode, prefill

pytestmark = pytest.mark.gpu

LAST = SPAN + 40


def test_positions_past_the_cache(cuda):
    runs = []
    for captured in (True, False):
        model, bt = build(cuda, weigh=True, max_positions=LAST)
        tokens, positions = prefill(model, bt), torch.tensor(PROMPTS, device=cuda)
        lens = model.evict(bt, positions, 40, 2, 8).long()
        positions = positions + SPAN - PROMPTS[2] - 30  # the longest session at SPAN - 30
        graph = M.DecodeGraph(model, bt, tokens, positions, lens) if captured else None
        logits = []
        for step in range(71):  # positions SPAN - 30 .. LAST
            if step % 20 == 19:
                cut = model.evict(bt, graph.lens if captured else lens, 40, 2, 8)
                lens = cut.long()
                if captured:
                    graph.lens.copy_(cut)
            if captured:
                graph.replay()
                logits.append(graph.logits.clone())
            else:
                out, capture, md = decode(model, bt, tokens, positions, lens, in_graph=True)
                if step in (29, 30, 31, 70):
                    check_attention(model, bt, capture, md.seq_lens.tolist(), torch.bfloat16)
                logits.append(out)
                tokens, positions, lens = out.argmax(-1), positions + 1, lens + 1
        with pytest.raises(ValueError, match="rotary table"):
            if captured:
                graph.replay()
            else:
                decode(model, bt, tokens, positions, lens)
        torch.cuda.synchronize()
        runs.append(logits)
    for a, b in zip(*runs):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_a_full_cache_ends_the_replays(cuda):
    model, bt = build(cuda, weigh=True, max_positions=LAST)
    tokens, positions = prefill(model, bt), torch.tensor(PROMPTS, device=cuda)
    lens = torch.tensor([SPAN - 2, 9, 100], device=cuda)
    graph = M.DecodeGraph(model, bt, tokens, positions, lens)
    graph.replay()
    graph.replay()
    with pytest.raises(ValueError, match="max_model_len"):
        graph.replay()
    graph.lens.copy_(model.evict(bt, graph.lens, 40, 2, 8))
    graph.replay()
    torch.cuda.synchronize()
    assert graph.lens.tolist() == [41, 12, 41] and torch.isfinite(graph.logits).all()


def test_a_graph_of_another_models_steps(cuda):
    """``DecodeGraph`` takes any model with ``decode_step``, ``block_size`` and ``max_model_len``."""
    model, bt = build(cuda)

    class Steps:
        block_size, max_model_len, decode_step = model.block_size, model.max_model_len, model.decode_step

    tokens, positions = prefill(model, bt), torch.tensor(PROMPTS, device=cuda)
    graph = M.DecodeGraph(Steps(), bt, tokens, positions)
    graph.replay()
    want = graph.logits.clone()
    graph.reset(tokens, positions)
    logits, _, _ = decode(model, bt, tokens, positions, in_graph=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(want, logits) and torch.equal(graph.logits, logits)
