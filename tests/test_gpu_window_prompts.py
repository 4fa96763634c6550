"""Prompts through a window on the GPU: captured calls, beside test_gpu_window's eager ones (its tolerances), and bf16 values
over their whole range.

The tolerance of the latter, as test_gpu_window's but for the values' own roundings, R the values that a row sees: bf16 values
are exact in fp16 from 2^-17 on (8 bits above its step of 2^-24) up to 65504; smaller ones are off by 2^-25, where the largest
value of the workgroup's tokens (128 queries' and what they see) is 2^-10 at least, and not at all where it is less. Weights in
fp16 are off by 2^-11, and by 2^-25 below its range, times the values that it holds; in two bf16 values by 2^-17.
"""
import math
import threading

import pytest
import torch

import test_gpu_cache8_model as CM
from cache8_plain import D, E, SCALE
from starkv_serve.kernels.prefill import prefill_attention, prompt_tables
from starkv_serve.kernels.window import Window
from test_gpu_window import prompts_close

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
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


def whole_range_close(got, q, k, v, lens, w, what=""):
    """Rows whose values are finite, against float64."""
    G, u, o = q.shape[1] // k.shape[1], torch.finfo(got.dtype).eps / 2, 0
    for L in filter(None, lens):
        t = torch.arange(L)
        sees = (t[None, :] <= t[:, None]) & ((t[:, None] - t[None, :] < w.size) | (t[None, :] < w.sinks))
        for h in range(q.shape[1]):
            x, K, V = q[o:o + L, h].cpu().double(), k[o:o + L, h // G].cpu().double(), v[o:o + L, h // G].cpu().double()
            s = (x @ K.t() * SCALE).masked_fill(~sees, -math.inf)
            p = torch.softmax(s, dim=-1)
            ds = 2 * 132 * E * SCALE * (x.abs() @ K.abs().t()).masked_fill(~sees, 0).amax(-1, keepdim=True)
            most = s.masked_fill(~sees, 0).abs().amax(-1, keepdim=True)
            n = sees.sum(-1, keepdim=True)
            out, mass = p @ V, p @ V.abs()
            held = torch.where(V.abs() <= 65504, V.abs(), 0.0).max()  # of the first tiles' products in fp16
            tol = (mass * (ds + 8 * E * (most / math.log(2) + 24) + 2.0 ** -11 + (n + 16) * E) + n * 2.0 ** -25 * held
                   + (2.0 ** -25 if V.abs().max() >= 2.0 ** -10 else 0) + u * out.abs() * 1.01)
            off = ((got[o:o + L, h].cpu().double() - out).abs() - tol).max().item()
            assert off <= 0, (what, L, h, off)
        o += L


RANGE = [2.0 ** -100, 2.0 ** -60, 2.0 ** -30, 2.0 ** -20, 2.0 ** -14, 2.0 ** -10, 2.0 ** -8, 2.0 ** -7, 1.0, 2.0 ** 13, 2.0 ** 17, 2.0 ** 60, 2.0 ** 124]


@pytest.mark.parametrize("size", RANGE)
@pytest.mark.parametrize("dt", [BF16, F32])
def test_values_of_any_size(cuda, size, dt):
    g = torch.Generator().manual_seed(3)
    q, k, v = prompts(BF16, 2, 2, cuda, g)
    v = (v.float().clamp(-6, 6) * size).to(BF16)
    w = Window(90, 5)
    out = torch.empty(q.shape, dtype=dt, device=cuda)
    got = prefill_attention(q, k, v, LENS, SCALE, out=out, window=w)
    assert got.isfinite().all()
    whole_range_close(got, q, k, v, LENS, w, size)


def test_heads_of_unlike_sizes(cuda):
    """Heads, dimensions and prompts of very large, ordinary and very small values beside each other, and of zeros."""
    g = torch.Generator().manual_seed(4)
    q, k, v = prompts(BF16, 4, 2, cuda, g)
    by = torch.tensor([2.0 ** -40, 1.0, 2.0 ** 40, 0.0])[None, :, None].repeat(sum(LENS), 1, D)
    by[:, 1, :9] = 2.0 ** 20
    by[LENS[0] + LENS[1]:, :2] *= 2.0 ** -30
    v = (v.float().cpu() * by).to(BF16).to(cuda)
    w = Window(90, 5)
    got = prefill_attention(q, k, v, LENS, SCALE, window=w)
    whole_range_close(got, q, k, v, LENS, w)
    assert (got[:, 6:] == 0).all() and got[:, :2].abs().max() > 2.0 ** -42


@pytest.mark.parametrize("small", [False, True])
def test_large_values_of_few_tokens(cuda, small):
    """Single values past fp16's range reach the rows that see them as they are, beside infinities and NaN that reach
    theirs; out of sight they change nothing. small: among values that are not exact in fp16 either."""
    g = torch.Generator().manual_seed(5)
    lens, w = [400, 70], Window(100, 20)
    q, k, v = (t.cpu() for t in prompts(BF16, 1, 4, cuda, g, lens))
    if small:
        v = v * 2.0 ** -30
    clean = v.clone()
    large = [(3, 7, 1e5), (60, 8, -3e38), (150, 9, 3e38), (151, 9, 3e38), (250, 100, -7e4), (399, 1, 2.0 ** 127), (400 + 69, 3, 1e30)]
    for t, d, x in large:
        v[t, 0, d] = clean[t, 0, d] = x
    odd = [(61, 20, math.inf), (200, 21, math.nan), (201, 22, -math.inf), (202, 9, math.inf)]
    got = prefill_attention(q.to(cuda), k.to(cuda), v.to(cuda), lens, SCALE, window=w)
    assert got.isfinite().all()
    whole_range_close(got, q, k, v, lens, w)
    for t, d, x in odd:
        v[t, 0, d], clean[t, 0, d] = x, 0.0
    got = prefill_attention(q.to(cuda), k.to(cuda), v.to(cuda), lens, SCALE, window=w).cpu()
    t = torch.arange(400)
    sees = (t[None, :] <= t[:, None]) & ((t[:, None] - t[None, :] < w.size) | (t[None, :] < w.sinks))
    expect = torch.zeros(470, D)
    for at, d, x in odd:
        expect[:400, d] += torch.where(sees[:, at], x, 0.0)
    expect = expect[:, None].expand(-1, 4, -1)
    assert torch.equal(got.isnan(), expect.isnan()) and torch.equal(got[expect.isinf()].float(), expect[expect.isinf()])
    fine = expect == 0
    assert got[fine].isfinite().all()
    whole = prefill_attention(q.to(cuda), k.to(cuda), clean.to(cuda), lens, SCALE, window=w).cpu()
    whole_range_close(torch.where(fine, got, whole), q, k, clean, lens, w)


def test_values_of_any_strides_and_sizes(cuda):
    """bf16 keys and values in any layout, past fp16's range and below it: rows that are not 16-byte aligned, broadcast ones,
    rows of other dimensions between."""
    g = torch.Generator().manual_seed(6)
    L, w = 300, Window(70, 5)
    wide = torch.randn(L, 6, 2 * D + 8, generator=g).to(BF16).to(cuda)
    q = torch.randn(L, 4, D, generator=g).to(BF16).to(cuda)
    for size in (2.0 ** -40, 2.0 ** 40):
        x = wide * size
        y = torch.randn(L, 2, 2 * D, generator=g).to(BF16).to(cuda) * size
        for k, v in ((wide[:, 1:3, 4:4 + D], x[:, 3:5, 1:1 + D]), (wide[:, :1, :D].expand(L, 2, D), x[:, 5:, 8:8 + D].expand(L, 2, D)),
                     (wide[:, ::3, 3:3 + D], x[:1, 2:4, 2:2 + D].expand(L, 2, D)), (wide[:, :2, :D], y[:, :, ::2]), (y[:, :, 1::2] / size, y[:, :, :D])):
            whole_range_close(prefill_attention(q, k, v, [L - 20, 20], SCALE, window=w), q, k, v, [L - 20, 20], w, (size, k.stride(), v.stride()))
    k = wide[:, :2, 4:4 + D] * 1e20  # keys of any size, aligned or not
    got = prefill_attention(q, k, wide[:, 2:4, :D], [L], SCALE * 1e-20, window=w)
    assert torch.equal(got, prefill_attention(q, k.contiguous(), wide[:, 2:4, :D], [L], SCALE * 1e-20, window=w)) and got.isfinite().all()


def test_captured_values_of_any_size(cuda):
    g = torch.Generator().manual_seed(7)
    q, k, v = prompts(BF16, 2, 2, cuda, g)
    w, tables = Window(90, 5), prompt_tables(LENS, cuda)
    out = torch.empty_like(q)
    prefill_attention(q, k, v, LENS, SCALE, out=out, tables=tables, window=w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prefill_attention(q, k, v, LENS, SCALE, out=out, tables=tables, window=w)
    for size in (1.0, 2.0 ** 30, 2.0 ** -30, 1.0):
        v.copy_(torch.randn(v.shape, generator=g) * size)
        graph.replay()
        got = out.clone()
        assert torch.equal(got, prefill_attention(q, k, v, LENS, SCALE, window=w))
        whole_range_close(got, q, k, v, LENS, w, size)
        torch.cuda.synchronize()


@pytest.mark.parametrize("cache8", [None, torch.int8])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_model_prompts_have_bf16_range(cuda, cache8, qk_norm):
    """Keys of 2^20 with queries as much smaller and values of 2^20: neither fits fp16, and steps take them too."""
    w = Window(40, 4)
    model, bt = CM.build(cuda, BF16, qk_norm, cache8=cache8, window=w)
    for layer in model.layers:
        rows = layer.qkv_proj.view(-1, D, layer.qkv_proj.shape[1])  # 8 heads of queries, 2 of keys, 2 of values
        if qk_norm:
            layer.q_norm.mul_(2.0 ** -20)
            layer.k_norm.mul_(2.0 ** 20)
        else:
            rows[:8].mul_(2.0 ** -20)
            rows[8:10].mul_(2.0 ** 20)
        rows[10:].mul_(2.0 ** 20)
    capture = []
    tokens, _ = CM.prefill(model, bt, capture)
    for c in capture:
        assert c["k"].abs().max() > 65504 and c["v"].abs().max() > 65504
        CM.W.prompts_close(c["out"], c["q"], c["k"], c["v"], CM.PROMPTS, w, c["layer"])
    bare, _ = CM.prefill(model, bt)  # without a capture the same
    assert torch.equal(bare, tokens)
    positions = torch.tensor(CM.PROMPTS, device=cuda)
    assert model.decode_step(tokens, positions, CM.M.decode_metadata(bt, positions, 16, CM.SPAN)).isfinite().all()


def test_prompts_from_several_threads(cuda):
    """Each thread on a stream of its own, kernels of unlike types between each other; every call in each of them."""
    g = torch.Generator().manual_seed(8)
    calls = []
    for dt in (BF16, F16, F32):
        for odt in (BF16, F16, F32):
            for window in (Window(90, 5), None):
                q, k, v = prompts(dt, 2, 2, cuda, g) if dt != F32 else (t.float() for t in prompts(F16, 2, 2, cuda, g))
                calls.append((q, k, v, odt, window))
    def run(q, k, v, odt, window):
        return prefill_attention(q, k, v, LENS, SCALE, out=torch.empty(q.shape, dtype=odt, device=cuda), window=window)
    got, errors, start = {}, [], threading.Barrier(6)

    def work(i):
        try:
            stream = torch.cuda.Stream()
            start.wait()
            with torch.cuda.stream(stream):
                for r in range(4):
                    for j in range(len(calls)):
                        at = (j + 3 * i) % len(calls)
                        got[i, at] = run(*calls[at])
            stream.synchronize()
        except Exception as e:  # of a thread: told to the test
            errors.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    want = [run(*c) for c in calls]
    for (i, at), x in got.items():
        assert torch.equal(x, want[at]), (i, at)
