"""Eviction by accumulated attention weight, for uncompressed caches on MI355X (libstarkv_hip.so): a decode that
sums up what each cached token weighs, and the cut of a cache to the tokens that weigh most.

The sums are a tensor ``[n, H_kv, tokens]`` (fp32) in the order of the block table's rows, one for each layer. A decode
step calls ``paged_decode_weighted`` where it would call ``paged_decode_full``; when caches have grown past their
budget, ``evict`` cuts them and the sums. Token positions go on counting: after a cut a request's
cache length is no longer its next position. No operator here has a gradient: calls that want one raise. The
reference has no counterpart; its uncompressed layers keep every token (starkv_serve/model.py:77-81 there).
"""
import torch

from starkv_serve import _hip
from starkv_serve.kernels.paged_decode import _as_i32


def paged_decode_weighted(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                          seq_lens: torch.Tensor, max_seq_len: int, scale: float,
                          weights: torch.Tensor) -> torch.Tensor:
    """``paged_decode_full`` (query of the cache's dtype, up to 16 query heads per KV head, any number), and weights
    [n, H_kv, >= max_seq_len] += each token's softmax weight, summed over its KV head's query heads. The newest
    token's entry (seq_lens[b] - 1) is set, as its sum starts with this step; entries behind it stay as they are.
    Lengths are cut to max_seq_len. A request without tokens gives zeros and leaves its weights; a head whose scores
    are all -inf gives NaN, and NaN weights."""
    _hip.require_cuda(query, k_cache, v_cache, block_table, seq_lens, weights)
    _hip.refuse_grad("paged_decode_weighted", query, k_cache, v_cache, weights)
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    if query.shape[0]:
        _hip.ops().weighted_decode(query, k_cache, v_cache, _as_i32(block_table), _as_i32(seq_lens), int(max_seq_len),
                                   float(scale), weights, out)
    return out


def evict(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
          weights: torch.Tensor, keep: int, sink: int = 4, recent: int = 32) -> tuple:
    """Cuts each request's cache to `keep` tokens per KV head: the first `sink`, the last `recent`, and the largest
    `weights` [n, H_kv, tokens] between (equal ones: the earlier token). The kept rows of both caches move to the
    front in place, in their order. Returns (seq_lens [n] int32, weights): new tensors, the kept tokens'
    sums in front and zeros behind.

    Requests of at most `keep` tokens keep their rows. A request that is cut owns its blocks: rows of a block that
    another request's table names too would move under it."""
    _hip.require_cuda(k_cache, v_cache, block_table, seq_lens, weights)
    _hip.refuse_grad("evict", k_cache, v_cache, weights)
    if sink < 0 or recent < 0 or keep < 1 or sink + recent > keep:
        raise ValueError(f"evict: keep={keep} tokens, sink={sink} and recent={recent} among them")
    lens = seq_lens.new_empty(seq_lens.shape, dtype=torch.int32)
    kept = torch.empty_like(weights, memory_format=torch.contiguous_format)
    if block_table.shape[0]:
        _hip.ops().evict(k_cache, v_cache, _as_i32(block_table), _as_i32(seq_lens), weights, int(keep), int(sink),
                         int(recent), lens, kept)
    return lens, kept
