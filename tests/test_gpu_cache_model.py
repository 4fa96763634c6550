"""The options of the model's uncompressed layers, as a serving program runs them: normed queries and keys, decode steps
over selected blocks, and steps that weigh with a cut between them; prompts, eager decode steps and captured ones.
Each layer's attention is compared with the float64 form over its caches as the step left them (tolerances of
test_gpu_cache_ops); captured steps equal the eager ones bit for bit."""
import pytest
import torch
import torch.nn.functional as F

from starkv_serve import model as M
from starkv_serve.kernels.sparse_decode import BlockSelection
from test_gpu_cache_ops import D, E, attention64, check, half_step, rows_of, select_plain

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
SHAPE = M.LlamaShape(hidden_size=512, num_layers=3, num_heads=8, num_kv_heads=2, intermediate_size=1024, vocab_size=1000,
                     qk_norm=True)
PROMPTS = [100, 9, 260]
SPAN = 512
SCALE = D ** -0.5


def build(cuda, dtype=BF16, shape=SHAPE, **kw):
    model = M.StarKVLlamaForCausalLM(shape, None, SPAN, cuda, dtype=dtype, seed=3, **kw)
    g = torch.Generator().manual_seed(4)
    for layer in model.layers:
        if layer.q_norm is not None:
            layer.q_norm, layer.k_norm = ((1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(cuda) for _ in range(2))
    model.allocate_kv_cache(len(PROMPTS) * SPAN // 16 + 1, 16, len(PROMPTS))
    bt = (torch.randperm(len(PROMPTS) * SPAN // 16, generator=g) + 1).int().view(len(PROMPTS), -1).to(cuda)
    return model, bt


def prefill(model, bt, capture=None):
    md, pos = M.prefill_metadata(bt, PROMPTS, 16)
    tokens = torch.randint(0, 1000, (sum(PROMPTS),), generator=torch.Generator().manual_seed(5)).to(bt.device)
    return model.prefill_step(tokens, pos, md, capture).argmax(-1)


def decode(model, bt, tokens, positions, lens=None, in_graph=False):
    md = M.decode_metadata(bt, positions, 16, SPAN, lens)
    capture = []
    logits = model.decode_step(tokens, positions, md, capture, in_graph)
    return logits, capture, md


@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_normed_rows(cuda, dtype):
    model, bt = build(cuda, dtype)
    capture = []
    tokens = prefill(model, bt, capture)
    pos = torch.cat([torch.arange(L) for L in PROMPTS])
    table, u = model.rotary.cos_sin_cache.double().cpu(), half_step(dtype)
    for c in capture:
        layer, h = model.layers[c["layer"]], c["h"].double().cpu()
        W = layer.qkv_proj.double().cpu()
        x, size = h @ W.t(), h.abs() @ W.abs().t()
        off = u * x.abs() + 520 * E * size  # of the rounded product: 512 products in fp32, its rounding
        for name, heads, at, w in (("q", 8, 0, layer.q_norm), ("k", 2, 8 * D, layer.k_norm)):
            xs, offs = (t[:, at:at + heads * D].view(-1, heads, D) for t in (x, off))
            rms = (xs.square().mean(-1, keepdim=True) + 1e-5).sqrt()
            y = xs / rms * w.double().cpu()
            ye = (offs / rms + xs.abs() / rms * (offs.norm(dim=-1, keepdim=True) / (rms * D ** 0.5))) * w.double().cpu().abs() * 1.05
            cos, sin = (t[:, None] for t in table[pos].chunk(2, dim=-1))
            (a, b), (ea, eb) = y.chunk(2, dim=-1), ye.chunk(2, dim=-1)
            z = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
            terms = torch.cat([(a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()], dim=-1)
            err = torch.cat([ea * cos.abs() + eb * sin.abs(), eb * cos.abs() + ea * sin.abs()], dim=-1) + 20 * E * terms
            check(c[name], z, err + u * (z.abs() + err) + 2.0 ** -25, (c["layer"], name))
        kc, vc = model.kv_caches[c["layer"]]
        for b, L in enumerate(PROMPTS):
            o = sum(PROMPTS[:b])
            for hd in range(2):
                assert torch.equal(rows_of(kc, bt, b, hd, range(L)), c["k"][o:o + L, hd].double().cpu())
                assert torch.equal(rows_of(vc, bt, b, hd, range(L)), c["v"][o:o + L, hd].double().cpu())
    positions = torch.tensor(PROMPTS, device=cuda)
    logits, capture, _ = decode(model, bt, tokens, positions)
    assert torch.isfinite(logits).all()
    for c in capture:  # every normed and rotated row has its norm's length
        for name, w in (("q", "q_norm"), ("k", "k_norm")):
            one = c[name].double().cpu().square().mean(-1).sqrt()
            most = getattr(model.layers[c["layer"]], w).abs().max().item()
            assert (one <= most * 1.01).all() and (one > 0.3).all()
    check_attention(model, bt, capture, [L + 1 for L in PROMPTS], dtype)


def check_attention(model, bt, capture, lens, dtype, chosen=None):
    for c in capture:
        kc, vc = model.kv_caches[c["layer"]]
        for b, L in enumerate(lens):
            for h in range(2):
                tokens = range(L)
                if chosen is not None:
                    tokens = [t for j in chosen(c, b, h) for t in range(16 * j, min(L, 16 * j + 16))]
                k, v = rows_of(kc, bt, b, h, tokens), rows_of(vc, bt, b, h, tokens)
                out, tol, _, _ = attention64(c["q"][b, 4 * h:4 * h + 4].cpu(), k, v, dtype)
                check(c["out"][b, 4 * h:4 * h + 4], out, tol, (c["layer"], b, h))


@pytest.mark.parametrize("keep", [3, 5, 40])
def test_decode_over_selected_blocks(cuda, keep):
    model, bt = build(cuda, sparse=BlockSelection(keep, 1, 2))
    tokens, positions = prefill(model, bt), torch.tensor(PROMPTS, device=cuda)
    for step in range(9):  # past the end of the second request's first block
        logits, capture, md = decode(model, bt, tokens, positions)
        lens = [L + step + 1 for L in PROMPTS]
        if step in (0, 6, 7, 8):
            picks = {}
            for c in capture:
                kc = model.kv_caches[c["layer"]][0]
                bounds = torch.zeros_like(model.key_bounds[c["layer"]])
                for b, L in enumerate(lens):
                    for j in range((L + 15) // 16):
                        for h in range(2):
                            rows = rows_of(kc, bt, b, h, range(16 * j, min(L, 16 * j + 16)))
                            bounds[bt[b, j].long(), h] = torch.stack([rows.amin(0), rows.amax(0)]).to(BF16).to(cuda)
                used = bt[torch.arange(3).repeat_interleave(torch.tensor([(L + 15) // 16 for L in lens])),
                          torch.cat([torch.arange((L + 15) // 16) for L in lens])].long()
                assert torch.equal(bounds[used], model.key_bounds[c["layer"]][used])
                picks[c["layer"]] = select_plain(c["q"], bounds, bt, lens, SPAN, 16, keep, 1, 2)
            check_attention(model, bt, capture, lens, BF16, lambda c, b, h: [j for j in picks[c["layer"]][b, h].tolist() if j >= 0])
        tokens, positions = logits.argmax(-1), positions + 1


def sums64(model, bt, capture, li, lens, weights, tol):
    """weights and tol [3][2][SPAN] advanced by one token a request, from the captured queries of layer li."""
    q = next(c["q"] for c in capture if c["layer"] == li)
    kc, vc = model.kv_caches[li]
    for b, (row, L) in enumerate(lens):
        if L == 0:
            continue
        for h in range(2):
            k, v = rows_of(kc, bt, b, h, range(L)), rows_of(vc, bt, b, h, range(L))
            _, _, p, pt = attention64(q[row, 4 * h:4 * h + 4].cpu(), k, v, BF16)
            weights[b, h, L - 1], tol[b, h, L - 1] = 0, 0
            weights[b, h, :L] += p.sum(0)
            tol[b, h, :L] += pt.sum(0) + 6 * E * weights[b, h, :L]


def test_weighing_and_cuts(cuda):
    model, bt = build(cuda, weigh=True)
    capture = []
    tokens, positions = prefill(model, bt, capture), torch.tensor(PROMPTS, device=cuda)
    want = [torch.zeros(3, 2, SPAN, dtype=torch.float64) for _ in model.layers]
    tol = [torch.zeros(3, 2, SPAN, dtype=torch.float64) for _ in model.layers]
    for li in range(3):
        for back in range(M.OBSERVED - 1, -1, -1):
            rows = [(sum(PROMPTS[:b + 1]) - 1 - back, L - back) if L > back else (0, 0) for b, L in enumerate(PROMPTS)]
            sums64(model, bt, capture, li, rows, want[li], tol[li])
        check(model.weights[li], want[li], tol[li] + 1e-37, li)
    lens = torch.tensor(PROMPTS, device=cuda)
    for step in range(12):
        if step in (3, 8):  # cut, and cut again
            before = [(k.clone(), v.clone(), w.clone()) for (k, v), w in zip(model.kv_caches, model.weights)]
            old = lens.clone()
            lens = model.evict(bt, lens, 40, 4, 8)
            assert lens.tolist() == [min(L, 40) for L in old.tolist()]
            for li, (k, v, w) in enumerate(before):
                for b, L in enumerate(old.tolist()):
                    for h in range(2):
                        kept = list(range(L))
                        if L > 40:
                            mid = sorted(range(4, L - 8), key=lambda i: (-w[b, h, i].item(), i))[:28]
                            kept = [*range(4), *sorted(mid), *range(L - 8, L)]
                        for now, then in zip(model.kv_caches[li], (k, v)):
                            assert torch.equal(rows_of(now, bt, b, h, range(len(kept))), rows_of(then, bt, b, h, kept))
                        got = model.weights[li][b, h]
                        assert torch.equal(got[:len(kept)], w[b, h, kept]) and (got[len(kept):] == 0).all()
                want[li], tol[li] = model.weights[li].double().cpu(), torch.zeros(3, 2, SPAN, dtype=torch.float64)
        logits, capture, md = decode(model, bt, tokens, positions, lens)
        lens = lens + 1
        assert md.seq_lens.tolist() == lens.tolist()
        check_attention(model, bt, capture, lens.tolist(), BF16)
        for li in range(3):
            sums64(model, bt, capture, li, list(enumerate(lens.tolist())), want[li], tol[li])
            check(model.weights[li], want[li], tol[li] + 1e-37, (step, li))
        tokens, positions = logits.argmax(-1), positions + 1


def test_prompts_of_a_later_batch_take_their_rows(cuda):
    """A prompt that joins running sessions sets its own row of the weights and no other."""
    model, bt = build(cuda, weigh=True)
    prefill(model, bt)
    before = [w.clone() for w in model.weights]
    md, pos = M.prefill_metadata(bt[1:2], [50], 16)
    model.prefill_step(torch.arange(50, device=cuda), pos, md, rows=torch.tensor([1]))
    for w, old in zip(model.weights, before):
        assert torch.equal(w[0], old[0]) and torch.equal(w[2], old[2]) and not torch.equal(w[1], old[1])
        assert (w[1, :, :50] > 0).all() and (w[1, :, 50:] == 0).all()
        assert ((w[1].sum(-1) - 4 * M.OBSERVED).abs() < 4 * M.OBSERVED).all()


@pytest.mark.parametrize("mode", ["norm", "sparse", "weigh"])
def test_captured_steps_are_the_eager_ones(cuda, mode):
    """A captured step of each option, replayed with cuts between the replays where it weighs, against eager steps of a
    twin model over the same span."""
    kw = dict(norm={}, sparse=dict(sparse=BlockSelection(4, 1, 2)), weigh=dict(weigh=True))[mode]
    runs = []
    for captured in (True, False):
        model, bt = build(cuda, **kw)
        tokens, positions = prefill(model, bt), torch.tensor(PROMPTS, device=cuda)
        lens = positions.clone() if mode == "weigh" else None
        graph = M.DecodeGraph(model, bt, tokens, positions, lens) if captured else None
        logits = []
        for step in range(8):
            if mode == "weigh" and step in (2, 5):
                cut = model.evict(bt, graph.lens if captured else lens, 30, 2, 8)
                if captured:
                    graph.lens.copy_(cut)
                else:
                    lens = cut.long()
            if captured:
                graph.replay()
                logits.append(graph.logits.clone())
            else:
                out, _, _ = decode(model, bt, tokens, positions, lens, in_graph=True)
                logits.append(out)
                tokens, positions = out.argmax(-1), positions + 1
                lens = None if lens is None else lens + 1
            torch.cuda.synchronize()
        runs.append((logits, model.kv_caches, model.weights, model.key_bounds))
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.equal(a, b)
    for i in (1, 2, 3):
        for a, b in zip(runs[0][i], runs[1][i]):
            for x, y in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
                assert torch.equal(x, y)


def test_a_rotation_of_the_callers_takes_normed_rows(cuda):
    model, bt = build(cuda)
    apply, seen = model.rotary.apply, []

    def mine(positions, x):
        seen.append(x)
        return apply(positions, x)

    model.rotary.apply = mine
    capture = []
    prefill(model, bt, capture)
    assert len(seen) == 6
    q = capture[0]["h"] @ model.layers[0].qkv_proj[:8 * D].t()
    want = F.rms_norm(q.view(-1, 8, D).float(), (D,), model.layers[0].q_norm.float(), 1e-5)
    assert (seen[0].float() - want).abs().max() < 0.05


def test_an_unnormed_model_is_the_stock_one(cuda):
    """Without the options nothing changes, and a selection of every block is the whole attention."""
    shape = M.LlamaShape(**{**SHAPE.__dict__, "qk_norm": False})
    stock, bt = build(cuda, shape=shape)
    sparse, _ = build(cuda, shape=shape, sparse=BlockSelection(40, 1, 2))
    a, b = prefill(stock, bt), prefill(sparse, bt)
    assert torch.equal(a, b)
    positions = torch.tensor(PROMPTS, device=cuda)
    _, ca, _ = decode(stock, bt, a, positions)
    _, cb, _ = decode(sparse, bt, b, positions)
    lens = [L + 1 for L in PROMPTS]
    check_attention(stock, bt, ca, lens, BF16)
    check_attention(sparse, bt, cb, lens, BF16)
