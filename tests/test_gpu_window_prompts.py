"""Prompts through a window on the GPU: captured calls, beside test_gpu_window's eager ones (its tolerances)."""
import pytest
import torch

from cache8_plain import D, SCALE
from starkv_serve.kernels.prefill import prefill_attention, prompt_tables
from starkv_serve.kernels.window import Window
from test_gpu_window import prompts_close

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
LENS = [1, 200, 0, 330, 64]


def prompts(dt, H, G, cuda, g, lens=LENS):
    """q, k, v as views of one projection's rows."""
    T = sum(lens)
    return [t.view(T, -1, D) for t in torch.randn(T, (G + 2) * H * D, generator=g).to(dt).to(cuda).split([G * H * D, H * D, H * D], -1)]


@pytest.mark.parametrize("window", [Window(90, 5), None])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_captured_prompts(cuda, dt, window):
    """One graph, replayed over new rows, with eager calls of other prompts between its replays."""
    g = torch.Generator().manual_seed(1)
    q, k, v = prompts(dt, 2, 2, cuda, g)
    tables = prompt_tables(LENS, cuda)
    eager = prefill_attention(q, k, v, LENS, SCALE, tables=tables, window=window)
    assert torch.equal(eager, prefill_attention(q, k, v, LENS, SCALE, window=window))
    out = torch.empty_like(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prefill_attention(q, k, v, LENS, SCALE, out=out, tables=tables, window=window)
    for _ in range(4):
        for t, x in zip((q, k, v), prompts(dt, 2, 2, cuda, g)):
            t.copy_(x)
        graph.replay()
        got = out.clone()
        prefill_attention(*prompts(dt, 2, 2, cuda, g, [77, 150]), [77, 150], SCALE, window=window)
        assert torch.equal(got, prefill_attention(q, k, v, LENS, SCALE, window=window))
        if window is not None:  # the causal kernel's queries are rounded with their scale: test_gpu_prefill's bounds
            prompts_close(got, q, k, v, LENS, window)
        torch.cuda.synchronize()


@pytest.mark.parametrize("window", [Window(90, 5), None])
def test_a_capture_takes_tables(cuda, window):
    """Without them the call is refused and the capture goes on."""
    g = torch.Generator().manual_seed(2)
    q, k, v = prompts(BF16, 1, 3, cuda, g)
    tables = prompt_tables(LENS, cuda)
    want = prefill_attention(q, k, v, LENS, SCALE, window=window)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="tables="):
            prefill_attention(q, k, v, LENS, SCALE, out=out, window=window)
        prefill_attention(q, k, v, LENS, SCALE, out=out, tables=tables, window=window)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
