"""STAR-KV Llama for decode steps, without vLLM.

Restates the serving model of the reference (starkv_serve/model.py:18-106 there) over
this library: a stock Llama whose compressed layers (those the fused checkpoint holds
factors for, checkpoint.py:74-93) attend over the STAR-KV cache and whose other layers
keep full K/V.

- A compressed layer's ``qkv_proj`` keeps only its Q rows (model.py:68-74 there; the
  checkpoint has no K/V projection for it). Its cache row is written straight from the
  layer input (``StarKVAttentionImpl.forward_from_hidden``: the codes' GEMM
  ``hidden @ [k_down; v_down]^T`` fused with the scatter or 3.2-bit pack), then the
  decode runs over the paged cache.
- An uncompressed layer is vLLM's LlamaAttention (model.py:77-81 there): QKV, RoPE on q
  and k, k and v into paged key / value caches [num_blocks, block_size, H_kv, 128]
  (``write_kv_full``, one launch, as vLLM's reshape_and_cache), and paged decode
  attention over them (``paged_decode_full``).
- Everything else is the stock Llama decoder: RMSNorm, SiLU-gated MLP, residuals, the
  final norm and the LM head.

The weights of everything but the attention factors are random-init here (the harness
measures decode steps; there is no network for real checkpoints). The factors come from
a fused checkpoint through ``load_fused_checkpoint``, as the reference loads them.

Two kinds of step: ``decode_step`` (every request contributes its one next token) and
``prefill_step`` (whole prompts, each from position 0, as the reference serves them: a
compressed layer writes the prompt's codes and runs its dense prefill,
attention.py:219-251; a full layer writes K/V and runs causal attention over the prompt,
here on this library's prefill kernel where vLLM would run FlashAttention).

Three options of the uncompressed layers that the reference does not have:

- ``LlamaShape.qk_norm``: an RMS norm of each query and key head in front of the rotation, in the rotation's launch
  (``model_ops.norm_rope_write``). A compressed layer's keys are lifted from codes as a linear map, which a norm of
  each key is not: such a shape takes no compressed layer.
- ``sparse``: decode steps attend to the blocks of each request whose key bounds promise the largest scores
  (``kernels/sparse_decode.py``); every step keeps the bounds of the blocks it writes.
- ``weigh``: steps sum up what each cached token weighs (``kernels/evict.py``); ``evict`` cuts the caches of all layers
  to the tokens that weigh most. After a cut a request's next position is no longer its cache length:
  ``decode_metadata`` and ``DecodeGraph`` take the lengths apart. Positions then go on past ``max_model_len`` while the
  cache does not; ``max_positions`` says how far, and a step past it raises.
"""
import math
from dataclasses import dataclass
from typing import List, Optional

import torch
import torch.nn.functional as F

from starkv_serve.attention import StarKVAttentionImpl, StarKVMetadata
from starkv_serve.checkpoint import StarKVCheckpoint
from starkv_serve.kernels import model_ops
from starkv_serve.kernels.evict import evict, paged_decode_weighted
from starkv_serve.kernels.prefill import prefill_attention
from starkv_serve.kernels.sparse_decode import (BlockSelection, key_bounds_like, paged_decode_sparse, select_blocks,
                                                update_key_bounds)
from starkv_serve.kernels.stock_decode import paged_decode_full, write_kv_full
from starkv_serve.workloads import cos_sin_table


@dataclass(frozen=True)
class LlamaShape:
    hidden_size: int = 4096
    num_layers: int = 32
    num_heads: int = 32
    num_kv_heads: int = 32
    head_dim: int = 128
    intermediate_size: int = 11008
    vocab_size: int = 32000
    rms_norm_eps: float = 1e-5
    rope_theta: float = 10000.0
    qk_norm: bool = False  # an RMS norm of each query and key head (uncompressed layers only)


LLAMA2_7B = LlamaShape()

FEW_MAX_TOKENS = 16  # decode steps up to this many tokens take few_linear
OBSERVED = 16        # a prompt's last tokens, whose attention a model that weighs sums up first


class Rotary:
    """What StarKVAttentionImpl reads of vLLM's RotaryEmbedding (``cos_sin_cache``
    [max_pos, head_dim] = cat(cos, sin)), plus NeoX rotate-half on q and k."""

    def __init__(self, max_pos: int, dtype: torch.dtype, device, base: float):
        self.cos_sin_cache = cos_sin_table(max_pos, dtype, device, base)

    def apply(self, positions: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
        """x [T, H, D] rotated at `positions` [T] (fp32 arithmetic, x's dtype out)."""
        if model_ops.rope_fits(self.cos_sin_cache, positions, x):
            return model_ops.rope(positions, x, self.cos_sin_cache)
        cos, sin = self.cos_sin_cache[positions].float().chunk(2, dim=-1)
        cos, sin = cos[:, None, :], sin[:, None, :]
        x1, x2 = x.float().chunk(2, dim=-1)
        return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)


@dataclass
class Layer:
    ln1: torch.Tensor
    ln2: torch.Tensor
    o_proj: torch.Tensor          # [hidden, H * D]
    gate_up: torch.Tensor         # [2 * intermediate, hidden]
    down: torch.Tensor            # [hidden, intermediate]
    q_proj: Optional[torch.Tensor] = None    # compressed: [H * D, hidden]
    impl: Optional[StarKVAttentionImpl] = None
    qkv_proj: Optional[torch.Tensor] = None  # uncompressed: [(H + 2 H_kv) * D, hidden]
    q_norm: Optional[torch.Tensor] = None    # qk_norm: [D]
    k_norm: Optional[torch.Tensor] = None

    @property
    def compressed(self) -> bool:
        return self.impl is not None


class StarKVLlamaForCausalLM:
    """Decode steps of a Llama with STAR-KV attention in its compressed layers."""

    def __init__(self, shape: LlamaShape, starkv: Optional[StarKVCheckpoint], max_model_len: int, device,
                 dtype: torch.dtype = torch.bfloat16, seed: int = 0, stock: bool = False,
                 sparse: Optional[BlockSelection] = None, weigh: bool = False, max_positions: Optional[int] = None):
        """`starkv` = None or `stock` = True: every layer uncompressed (the stock model). `sparse`: decode steps of
        the uncompressed layers read selected blocks. `weigh`: steps sum up their tokens' weights, for ``evict``.
        `max_positions`: the last position of a session whose cuts keep its cache within max_model_len tokens
        (max_model_len, and never less)."""
        compressed = starkv is not None and not stock and any(map(starkv.is_compressed, range(shape.num_layers)))
        if sparse is not None and weigh:
            raise ValueError("sparse or weigh: a decode over selected blocks does not weigh the others' tokens")
        if compressed and shape.qk_norm:
            raise NotImplementedError("qk_norm: a compressed layer's keys are a linear map of its codes, not normed ones")
        if compressed and weigh:
            raise NotImplementedError("weigh: a compressed layer's cache row holds every head's codes and is not cut by head")
        self.shape, self.device, self.dtype = shape, torch.device(device), dtype
        self.sparse, self.weigh = sparse, weigh
        self.max_model_len = max_model_len
        H, Hkv, D, hid = shape.num_heads, shape.num_kv_heads, shape.head_dim, shape.hidden_size
        self.scale = D ** -0.5
        self.rotary = Rotary(max(max_model_len, max_positions or 0) + 1, dtype, self.device, shape.rope_theta)
        g = torch.Generator(device=self.device).manual_seed(seed)

        def w(*size, fan_in):
            t = torch.empty(*size, device=self.device, dtype=dtype)
            t.normal_(0.0, fan_in ** -0.5, generator=g)
            return t

        self.embed = w(shape.vocab_size, hid, fan_in=1)
        self.norm = torch.ones(hid, device=self.device, dtype=dtype)
        self.lm_head = w(shape.vocab_size, hid, fan_in=hid)
        self.layers: List[Layer] = []
        for li in range(shape.num_layers):
            lw = None if (starkv is None or stock or not starkv.is_compressed(li)) else starkv.layers[li]
            layer = Layer(ln1=torch.ones(hid, device=self.device, dtype=dtype),
                          ln2=torch.ones(hid, device=self.device, dtype=dtype),
                          o_proj=w(hid, H * D, fan_in=H * D),
                          gate_up=w(2 * shape.intermediate_size, hid, fan_in=hid),
                          down=w(hid, shape.intermediate_size, fan_in=shape.intermediate_size))
            if lw is not None:
                layer.q_proj = w(H * D, hid, fan_in=hid)
                layer.impl = StarKVAttentionImpl(H, D, self.scale, Hkv, starkv_layer=lw, rotary_emb=self.rotary,
                                                 max_model_len=max_model_len)
                layer.impl.to_device(self.device, dtype)
            else:
                layer.qkv_proj = w((H + 2 * Hkv) * D, hid, fan_in=hid)
                if shape.qk_norm:
                    layer.q_norm, layer.k_norm = (torch.ones(D, device=self.device, dtype=dtype) for _ in range(2))
            self.layers.append(layer)
        self.kv_caches: List = []
        self.key_bounds: List = []  # sparse: per layer, None for a compressed one
        self.weights: List = []     # weigh: per layer [requests, H_kv, max_model_len], in the order of a step's rows

    # -- caches ---------------------------------------------------------------------------
    def cache_bytes_per_token(self) -> int:
        """KV-cache bytes per token over all layers."""
        s = self.shape
        total = 0
        for layer in self.layers:
            if layer.compressed:
                imp = layer.impl
                total += imp.row.nbytes if imp.row is not None else (imp.k_width + imp.w.v_rank) * 2
            else:
                total += 2 * s.num_kv_heads * s.head_dim * 2
        return total

    def allocate_kv_cache(self, num_blocks: int, block_size: int = 16, num_requests: int = 0) -> None:
        """`num_requests`: the most rows of a step of a model that weighs; a request keeps its row of the weights from its
        prompt on (decode steps take rows 0 .. n - 1)."""
        s = self.shape
        if self.weigh and num_requests < 1:
            raise ValueError("a model that weighs needs num_requests")
        self.block_size = block_size
        self.kv_caches, self.key_bounds, self.weights = [], [], []
        for layer in self.layers:
            if layer.compressed:
                imp = layer.impl
                if imp.row is not None:
                    c = torch.zeros(num_blocks, block_size, imp.row.nbytes, dtype=torch.uint8, device=self.device)
                else:
                    c = torch.zeros(num_blocks, block_size, imp.k_width + imp.w.v_rank, dtype=self.dtype,
                                    device=self.device)
                self.kv_caches.append(c)
            else:
                kc = torch.zeros(num_blocks, block_size, s.num_kv_heads, s.head_dim, dtype=self.dtype,
                                 device=self.device)
                self.kv_caches.append((kc, torch.zeros_like(kc)))
            if self.sparse is not None:
                self.key_bounds.append(None if layer.compressed else key_bounds_like(kc))
            if self.weigh:
                self.weights.append(torch.zeros(num_requests, s.num_kv_heads, self.max_model_len, device=self.device))

    @torch.no_grad()
    def evict(self, block_table: torch.Tensor, seq_lens: torch.Tensor, keep: int, sink: int = 4,
              recent: int = 32) -> torch.Tensor:
        """The caches of every layer cut to `keep` tokens a request and KV head (``kernels.evict.evict``; rows of
        `block_table` and `seq_lens` as in the steps), their summed weights with them. Returns the cache lengths
        [n] int32, which the next step takes apart from the positions."""
        if not self.weights:
            raise RuntimeError("evict: a model built with weigh=True, its caches allocated")
        n = seq_lens.shape[0]
        lens = seq_lens
        for (kc, vc), weights in zip(self.kv_caches, self.weights):
            lens, kept = evict(kc, vc, block_table[:n], seq_lens, weights[:n], keep, sink, recent)
            weights[:n].copy_(kept)
        return lens

    # -- the step ---------------------------------------------------------------------------
    def _attention(self, li: int, x: torch.Tensor, positions: torch.Tensor, md: StarKVMetadata,
                   capture: Optional[list], in_graph: bool, few: bool, observed=None) -> torch.Tensor:
        """The layer's attention from its residual stream x [T, hidden], up to o_proj's input.
        Inside a graph (`in_graph`) no launch depends on the step's lengths: every layer
        decodes over the span max_model_len, the lengths are read on the device."""
        s, layer = self.shape, self.layers[li]
        T = x.shape[0]
        H, Hkv, D = s.num_heads, s.num_kv_heads, s.head_dim
        k = v = None
        if layer.compressed:
            h, q = self._norm_linear(x, layer.ln1, layer.q_proj, few, True)
            q = self.rotary.apply(positions, q.view(T, H, D))
            out = torch.empty(T, H * D, dtype=self.dtype, device=self.device)
            layer.impl.forward_from_hidden(q.view(T, H * D), h, self.kv_caches[li], md, out, in_full_graph=in_graph)
        else:
            h, qkv = self._norm_linear(x, layer.ln1, layer.qkv_proj, few, capture is not None)
            q, k, v = (t.view(T, n, D) for t, n in zip(qkv.split([H * D, Hkv * D, Hkv * D], dim=-1), (H, Hkv, Hkv)))
            kc, vc = self.kv_caches[li]
            ka, va = k, v  # the prefill attention's operands
            slots = md.slot_mapping[:T]
            if self._own_rotation() and model_ops.rope_write_fits(self.rotary.cos_sin_cache, positions, q, k, v, kc, vc, slots):
                if layer.q_norm is None:
                    q, k, ka, va = model_ops.rope_write(positions, q, k, v, self.rotary.cos_sin_cache, kc, vc, slots,
                                                        capture is not None, bool(md.num_prefills))
                else:
                    q, k, ka, va = model_ops.norm_rope_write(positions, q, k, v, self.rotary.cos_sin_cache, layer.q_norm,
                                                             layer.k_norm, s.rms_norm_eps, kc, vc, slots,
                                                             capture is not None, bool(md.num_prefills))
            else:
                q, k = self._normed(layer, q, k)
                q, k = self.rotary.apply(positions, q), self.rotary.apply(positions, k)
                ka = k
                write_kv_full(k, v, kc, vc, slots)
            if md.num_prefills:  # whole prompts only (prefill_step): causal attention over each prompt
                out = prefill_attention(q, ka, va, md.prefill_seq_lens_cpu, self.scale).view(T, H * D)
                if self.sparse is not None:
                    update_key_bounds(kc, self.key_bounds[li], md.block_table[:md.num_prefills], md.seq_lens,
                                      md.max_seq_len)
                if self.weigh:
                    self._observe(li, q, md, observed)
            else:
                span = self.max_model_len if in_graph else max(md.max_seq_len, 1)
                out = self._decode_attention(li, q, md, span).view(T, H * D)
        if capture is not None:
            capture.append(dict(layer=li, q=q.view(T, H, D), out=out.view(T, H, D), h=h, k=k, v=v))
        return out

    def _own_rotation(self) -> bool:
        """Whether rows are rotated by the rotary table, not by a rotation of the caller's."""
        return getattr(self.rotary.apply, "__func__", None) is Rotary.apply

    def _check_positions(self, positions: torch.Tensor, md: StarKVMetadata) -> None:
        """Refuses positions behind the rotary table, where the kernels would end the launch and the process with it. The
        block table bounds a position that is its cache's length; one that lies apart is read here where the
        caller gives no bound (a wait for the device; inside a capture ``DecodeGraph.replay`` counts)."""
        if not (md.positions_apart or md.max_position is not None) or not self._own_rotation():
            return
        top, rows = md.max_position, self.rotary.cos_sin_cache.shape[0]
        if top is None:
            if not positions.numel() or positions.is_cuda and torch.cuda.is_current_stream_capturing():
                return
            top = int(positions.max())
        if top >= rows:
            raise ValueError(f"position {top} is behind the rotary table's {rows} rows (max_positions)")

    def _normed(self, layer: Layer, q: torch.Tensor, k: torch.Tensor) -> tuple:
        """q and k behind their norms, where a rotation of the caller's follows (rounded between the two)."""
        if layer.q_norm is None:
            return q, k
        eps, D = self.shape.rms_norm_eps, self.shape.head_dim
        return F.rms_norm(q, (D,), layer.q_norm, eps), F.rms_norm(k, (D,), layer.k_norm, eps)

    def _decode_attention(self, li: int, q: torch.Tensor, md: StarKVMetadata, span: int) -> torch.Tensor:
        """An uncompressed layer's attention of a decode step, its keys and values written."""
        T = q.shape[0]
        kc, vc = self.kv_caches[li]
        table, lens = md.block_table[:T], md.seq_lens[:T]
        if self.sparse is not None:
            update_key_bounds(kc, self.key_bounds[li], table, lens, 1)
            sel = select_blocks(q, self.key_bounds[li], table, lens, span, self.block_size, self.sparse.keep,
                                self.sparse.sink, self.sparse.recent)
            return paged_decode_sparse(q, kc, vc, table, lens, sel, self.scale)
        if self.weigh:
            return paged_decode_weighted(q, kc, vc, table, lens, span, self.scale, self.weights[li][:T])
        return paged_decode_full(q, kc, vc, table, lens, span, self.scale)

    @staticmethod
    def _observed_rows(md: StarKVMetadata, device) -> list:
        """The last tokens of each prompt in their order: (their rows of the step, the tokens they see), 0 tokens where
        the prompt is shorter."""
        ends = torch.tensor(md.prefill_query_start_loc_cpu[1:])
        lens = torch.tensor(md.prefill_seq_lens_cpu)
        back = torch.arange(OBSERVED - 1, -1, -1)[:, None]
        seen = (lens - back).clamp(min=0)
        rows = (ends - 1 - torch.minimum(back, lens - 1)).to(device, non_blocking=True)
        return list(zip(rows, seen.to(torch.int32).to(device, non_blocking=True)))

    def _prompt_rows(self, n: int, rows) -> torch.Tensor:
        """`rows` of n prompts on the device. One outside the weights would end the process there, and of two prompts with
        one row either might win: refused before the step writes anything."""
        if not self.weights:
            raise RuntimeError("prompts of a model that weighs need allocate_kv_cache first")
        have, dev = self.weights[0].shape[0], self.weights[0].device
        if n > have:
            raise ValueError(f"{n} prompts for {have} rows of weights (num_requests of allocate_kv_cache)")
        if rows is None:
            return torch.arange(n, device=dev)
        rows = torch.as_tensor(rows)
        whole = not rows.is_floating_point() and rows.dtype != torch.bool and rows.shape == (n,)
        at = rows.tolist() if whole else []
        if len(set(at)) != n or min(at) < 0 or max(at) >= have:
            raise ValueError(f"prefill_step: rows {rows.tolist()} of {n} prompts: each one of its own of 0 .. {have - 1}")
        return rows.to(dev, torch.int64)

    def _observe(self, li: int, q: torch.Tensor, md: StarKVMetadata, observed: tuple) -> None:
        """The weights of prompts just written: what their last ``OBSERVED`` tokens give, a decode form each."""
        kc, vc = self.kv_caches[li]
        n = md.num_prefills
        steps, rows = observed
        weights = torch.zeros(n, *self.weights[li].shape[1:], device=q.device)
        for at, seen in steps:
            paged_decode_weighted(q[at], kc, vc, md.block_table[:n], seen, md.max_seq_len, self.scale, weights)
        self.weights[li].index_copy_(0, rows, weights)

    # -- the weight products ------------------------------------------------------------------
    def _few(self, T: int, md: StarKVMetadata) -> bool:
        """Whether this step's weight products run on ``few_linear``: a decode step of few tokens,
        where the weights' bytes are the time. Llama-2-7B's widths at 16 tokens, us, against the
        library's products with torch's norm, gate and sum: q 14 / 21, qkv 35 / 35, o 12 / 18, gate and
        up 53 / 67, down 30 / 41, the head 74 / 68; the kernel's matrix tile holds 16 tokens."""
        return (self.device.type == "cuda" and not md.num_prefills and 1 <= T <= FEW_MAX_TOKENS
                and self.dtype in (torch.bfloat16, torch.float16))

    def _norm_linear(self, x: torch.Tensor, ln: torch.Tensor, w: torch.Tensor, few: bool, want_h: bool) -> tuple:
        """(the normalised x, when wanted, its product with w)."""
        s = self.shape
        if few and self.dtype == torch.bfloat16 and model_ops.few_fits(x, w, ln):
            h = torch.empty_like(x) if want_h else None
            return h, model_ops.few_linear(x, w, ln, s.rms_norm_eps, h)
        h = F.rms_norm(x, (s.hidden_size,), ln, s.rms_norm_eps)
        return h, model_ops.few_linear(h, w) if few and model_ops.few_fits(h, w) else F.linear(h, w)

    def _mlp(self, x: torch.Tensor, layer: Layer, few: bool) -> torch.Tensor:
        """x plus the gated MLP of its norm."""
        s = self.shape
        if few and self.dtype == torch.bfloat16 and model_ops.few_fits(x, layer.gate_up, layer.ln2):
            a = model_ops.few_linear(x, layer.gate_up, layer.ln2, s.rms_norm_eps, gate=True)
        else:
            gu = self._norm_linear(x, layer.ln2, layer.gate_up, few, False)[1]
            if gu.is_cuda and gu.dtype in (torch.bfloat16, torch.float16) and s.intermediate_size % 8 == 0:
                a = model_ops.silu_mul(gu)
            else:
                gate, up = gu.chunk(2, dim=-1)
                a = F.silu(gate) * up
        return self._add_linear(x, a, layer.down, few)

    @staticmethod
    def _add_linear(x: torch.Tensor, a: torch.Tensor, w: torch.Tensor, few: bool) -> torch.Tensor:
        return model_ops.few_linear(a, w, residual=x) if few and model_ops.few_fits(a, w, residual=x) else x + F.linear(a, w)

    @torch.no_grad()
    def attention_inputs(self, hidden: torch.Tensor, positions: torch.Tensor) -> List[tuple]:
        """Per layer, what its attention op takes for one step with input `hidden`: the
        rotated queries, and for an uncompressed layer the rotated keys and the values (a
        compressed layer takes `hidden` itself: its write computes the codes)."""
        s = self.shape
        T = hidden.shape[0]
        H, Hkv, D = s.num_heads, s.num_kv_heads, s.head_dim
        res = []
        for layer in self.layers:
            if layer.compressed:
                q = self.rotary.apply(positions, F.linear(hidden, layer.q_proj).view(T, H, D))
                res.append((q.reshape(T, H * D), None, None))
            else:
                q, k, v = F.linear(hidden, layer.qkv_proj).split([H * D, Hkv * D, Hkv * D], dim=-1)
                q, k = self._normed(layer, q.reshape(T, H, D), k.reshape(T, Hkv, D))
                res.append((self.rotary.apply(positions, q), self.rotary.apply(positions, k),
                            v.reshape(T, Hkv, D).contiguous()))
        return res

    @torch.no_grad()
    def attention_only(self, hidden: torch.Tensor, inputs: List[tuple], md: StarKVMetadata,
                       in_graph: bool = False) -> None:
        """The attention ops of every layer for one step (the "attention per step" figure:
        the cache write and the attention, summed over the layers, as the reference's
        benchmark sums its two attention ops, bench_serving.py:62-115; the projections and
        RoPE are outside, as there). `inputs` from attention_inputs. A compressed layer's
        write includes its codes' GEMM (hidden @ kv_down^T), which the reference runs
        outside the attention op (model.py:71)."""
        T = hidden.shape[0]
        for li, layer in enumerate(self.layers):
            q, k, v = inputs[li]
            if layer.compressed:
                out = torch.empty(T, q.shape[1], dtype=self.dtype, device=self.device)
                layer.impl.forward_from_hidden(q, hidden, self.kv_caches[li], md, out, in_full_graph=in_graph)
            else:
                kc, vc = self.kv_caches[li]
                write_kv_full(k, v, kc, vc, md.slot_mapping[:T])
                self._decode_attention(li, q, md, self.max_model_len if in_graph else max(md.max_seq_len, 1))

    @torch.no_grad()
    def _layers(self, x: torch.Tensor, positions: torch.Tensor, md: StarKVMetadata, capture: Optional[list],
                in_graph: bool, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        few = self._few(x.shape[0], md)
        observed = None
        if self.weigh and md.num_prefills:
            observed = self._observed_rows(md, x.device), rows
        for li, layer in enumerate(self.layers):
            a = self._attention(li, x, positions, md, capture, in_graph, few, observed)
            x = self._add_linear(x, a, layer.o_proj, few)
            x = self._mlp(x, layer, few)
        return x

    def _logits(self, x: torch.Tensor, few: bool) -> torch.Tensor:
        return self._norm_linear(x, self.norm, self.lm_head, few, False)[1]

    def decode_step(self, tokens: torch.Tensor, positions: torch.Tensor, md: StarKVMetadata,
                    capture: Optional[list] = None, in_graph: bool = False) -> torch.Tensor:
        """Logits [n, vocab] for one new token per request: tokens [n] at `positions` [n];
        `md` has every row as a decode (slot_mapping the new tokens' slots, seq_lens the cached
        tokens with them: positions + 1, fewer where caches were cut)."""
        self._check_positions(positions, md)
        x = self._layers(self.embed[tokens], positions, md, capture, in_graph)
        return self._logits(x, self._few(x.shape[0], md))

    @torch.no_grad()
    def prefill_step(self, tokens: torch.Tensor, positions: torch.Tensor, md: StarKVMetadata,
                     capture: Optional[list] = None, rows=None) -> torch.Tensor:
        """Logits [P, vocab] at the last token of each of P whole prompts: tokens [T] and
        positions [T] (0 .. L - 1 per prompt) laid end to end, `md` from
        ``prefill_metadata``. Every layer writes the prompts' cache rows (compressed: the
        codes through the fused write; full: K and V), so decode steps can follow. `rows` [P]: the
        prompts' rows of a weighing model's weights (0 .. P - 1; a list or a tensor, which is read back)."""
        if md.num_decodes or not md.num_prefills:
            raise ValueError("prefill_step: a prompts-only batch (prefill_metadata)")
        if self.weigh:
            rows = self._prompt_rows(md.num_prefills, rows)
        x = self._layers(self.embed[tokens], positions, md, capture, False, rows)
        last = torch.tensor([e - 1 for e in md.prefill_query_start_loc_cpu[1:]]).to(x.device, non_blocking=True)
        return self._logits(x[last], False)


class DecodeGraph:
    """Greedy decode steps of `n` sessions captured once in a HIP graph: each replay runs
    one whole step (metadata from the positions, the 32 layers, the LM head, argmax) and
    advances the static tokens and positions in place, so consecutive replays decode
    consecutive tokens with no host work between them; `logits` holds the last replay's
    logits. The block table is static: its rows must cover every position the replays
    reach (up to max_model_len - 1). `lens`: cached tokens of each session where they are not its
    positions (``StarKVLlamaForCausalLM.evict`` cut its caches; ``lens`` of the graph takes what a later
    cut returns); they advance with the positions, and ``replay`` raises before a length passes max_model_len or a
    position the rotary table."""

    def __init__(self, model: StarKVLlamaForCausalLM, block_table: torch.Tensor, tokens: torch.Tensor,
                 positions: torch.Tensor, lens: Optional[torch.Tensor] = None):
        if model.max_model_len > block_table.shape[1] * model.block_size:
            raise ValueError("the block table's rows must cover max_model_len positions")
        self.model, self.block_table = model, block_table
        self.tokens = tokens.clone()
        self.positions = positions.clone().long()
        self.lens = None if lens is None else lens.clone().long()
        if lens is not None:
            self._steps_left()
        self.graph = torch.cuda.CUDAGraph()
        weights = getattr(model, "weights", [])  # any model with these steps will do
        kept = [w.clone() for w in weights]
        self._body()  # eager first: every lazy initialisation outside the capture
        for w, before in zip(weights, kept):  # that step is run again: its weights count once
            w.copy_(before)
        self.reset(tokens, positions, lens)
        torch.cuda.synchronize()
        with torch.cuda.graph(self.graph):
            self._body()

    @torch.no_grad()
    def _body(self) -> None:
        m = self.model
        md = decode_metadata(self.block_table, self.positions, m.block_size, m.max_model_len, self.lens)
        self.logits = m.decode_step(self.tokens, self.positions, md, in_graph=True)
        if model_ops.greedy_fits(self.logits, self.tokens):
            model_ops.greedy_step(self.logits, self.tokens, self.positions)
        else:
            self.tokens.copy_(self.logits.argmax(-1))
            self.positions.add_(1)
        if self.lens is not None:
            self.lens.add_(1)

    def reset(self, tokens: torch.Tensor, positions: torch.Tensor, lens: Optional[torch.Tensor] = None) -> None:
        if (lens is None) != (self.lens is None):
            raise ValueError("a graph of sessions with lengths of their own takes them at every reset, another none")
        self.tokens.copy_(tokens)
        self.positions.copy_(positions)
        if lens is not None:
            self.lens.copy_(lens)
        self._left = 0

    def _steps_left(self) -> int:
        """Replays that stay in the cache and the rotary table; raises where there are none."""
        m = self.model
        length, top = int(self.lens.max()), int(self.positions.max())
        if length >= m.max_model_len:
            raise ValueError(f"a session's cache holds {length} tokens, the model's max_model_len; cut it or reset")
        left = m.max_model_len - length
        if m._own_rotation():
            rows = m.rotary.cos_sin_cache.shape[0]
            if top >= rows:
                raise ValueError(f"position {top} is behind the rotary table's {rows} rows (max_positions)")
            left = min(left, rows - top)
        return left

    def replay(self) -> None:
        if self.lens is not None:
            # Counted on the host and read from the device only where the count runs out: a cut since shortened lengths.
            self._left = (self._left or self._steps_left()) - 1
        self.graph.replay()


def decode_metadata(block_table: torch.Tensor, positions: torch.Tensor, block_size: int,
                    max_seq_len: int, lens: Optional[torch.Tensor] = None,
                    max_position: Optional[int] = None) -> StarKVMetadata:
    """A decode-only batch's metadata: request b's new token at positions[b] (slot from its
    block-table row), seq_lens = positions + 1. `lens` [n]: the tokens cached before it, where a cut left fewer than
    positions[b]; the slot and seq_lens go by them. `max_position`: an upper bound of positions that lie apart from
    `lens`, so that the step need not read them back to see that they are in the rotary table."""
    n, apart = positions.shape[0], lens is not None
    if lens is not None:
        positions = lens.long()
    if max_seq_len > block_table.shape[1] * block_size:
        raise ValueError(f"positions up to {max_seq_len - 1} need more than the block table's "
                         f"{block_table.shape[1]} blocks of {block_size}")
    if model_ops.slots_fit(block_table, positions):
        slots, seq_lens = model_ops.decode_slots(block_table, positions, block_size)
    else:
        rows = torch.arange(n, device=positions.device)
        slots = block_table[rows, positions // block_size].long() * block_size + positions % block_size
        seq_lens = (positions + 1).to(torch.int32)
    return StarKVMetadata(num_actual_tokens=n, num_decodes=n, num_decode_tokens=n, num_prefills=0,
                          max_seq_len=int(max_seq_len), seq_lens=seq_lens, block_table=block_table, slot_mapping=slots,
                          positions_apart=apart, max_position=max_position)


def prefill_metadata(block_table: torch.Tensor, prompt_lens: List[int], block_size: int):
    """A prompts-only batch's metadata and positions: prompt b's tokens at positions
    0 .. L_b - 1, their slots from block-table row b, laid end to end. Returns (md,
    positions [T])."""
    lens = [int(L) for L in prompt_lens]
    if not lens or min(lens) < 1:
        raise ValueError("prefill_metadata: every prompt needs at least one token")
    if max(lens) > block_table.shape[1] * block_size:
        raise ValueError(f"a prompt of {max(lens)} tokens needs more than the block table's "
                         f"{block_table.shape[1]} blocks of {block_size}")
    dev = block_table.device
    rows = torch.cat([torch.full((L,), b, dtype=torch.long) for b, L in enumerate(lens)]).to(dev)
    positions = torch.cat([torch.arange(L) for L in lens]).to(dev)
    slots = block_table[rows, positions // block_size].long() * block_size + positions % block_size
    qsl = [0]
    for L in lens:
        qsl.append(qsl[-1] + L)
    md = StarKVMetadata(num_actual_tokens=qsl[-1], num_decodes=0, num_decode_tokens=0, num_prefills=len(lens),
                        max_seq_len=max(lens), seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                        block_table=block_table, slot_mapping=slots, prefill_seq_lens_cpu=lens,
                        prefill_query_start_loc_cpu=qsl)
    return md, positions


def ranks_for_ratio(num_kv_heads: int, head_dim: int, keep: float, multiple: int, generator: torch.Generator):
    """Per-head K ranks (multiples of `multiple`) keeping about `keep` of the K dimensions
    in all, drawn around the mean (the reference's 0.75-ratio checkpoint keeps ~21.5 % of K
    and ~31.5 % of V, train.py:356-389 / README.md:87-88)."""
    total = int(round(keep * num_kv_heads * head_dim / multiple)) * multiple
    lo = max(multiple, (total // num_kv_heads) // multiple * multiple)
    ranks = [lo] * num_kv_heads
    left = (total - lo * num_kv_heads) // multiple
    for i in torch.randperm(num_kv_heads, generator=generator).tolist()[:left]:
        ranks[i] += multiple
    return ranks


def v_rank_for_ratio(num_kv_heads: int, head_dim: int, keep: float, multiple: int) -> int:
    return max(multiple, int(math.floor(keep * num_kv_heads * head_dim / multiple)) * multiple)
