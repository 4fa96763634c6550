"""Decode over a part of a long uncompressed cache on MI355X (libstarkv_hip.so): per cache block and KV head
the bounds of its keys, the choice of the blocks a query token reads by them, and the attention over those.

The caches are ``paged_decode_full``'s; beside them ``key_bounds_like`` makes the bounds ``[num_blocks, H_kv, 2, 128]``,
indexed by the same block ids, so they follow the block table wherever the caches go. A step:
``update_key_bounds`` after the cache write, ``select_blocks``, ``paged_decode_sparse``. No operator here has a
gradient: calls that want one raise. The reference has no counterpart; its uncompressed layers attend to
their whole cache (starkv_serve/model.py:77-81 there).
"""
from dataclasses import dataclass

import torch

from starkv_serve import _hip
from starkv_serve.kernels.paged_decode import _as_i32


@dataclass(frozen=True)
class BlockSelection:
    """How many cache blocks a query token of a request reads per KV head: `keep` in all, the first `sink` and
    the last `recent` always among them."""
    keep: int
    sink: int = 1
    recent: int = 2

    def __post_init__(self):
        if self.sink < 0 or self.recent < 1 or self.keep < self.sink + self.recent:
            raise ValueError(f"{self}: at least the last block (the token's own), and keep >= sink + recent")


def key_bounds_like(k_cache: torch.Tensor) -> torch.Tensor:
    """The bounds of a key cache [num_blocks, block_size, H_kv, 128], not filled."""
    return torch.zeros(k_cache.shape[0], k_cache.shape[2], 2, k_cache.shape[3], dtype=k_cache.dtype,
                       device=k_cache.device)


def update_key_bounds(k_cache: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                      max_new: int) -> None:
    """The bounds (bounds[block, head, 0]: least, [.., 1]: largest key, elementwise) of every block that holds one of
    the last `max_new` of a request's seq_lens[b] tokens, from all its tokens, in place; one launch. A decode
    step has one new token, a prefill as many as its longest prompt."""
    _hip.require_cuda(k_cache, bounds, block_table, seq_lens)
    _hip.refuse_grad("update_key_bounds", k_cache, bounds)
    if max_new < 0:
        raise ValueError(f"update_key_bounds: max_new={max_new}")
    if block_table.shape[0]:
        _hip.ops().key_bounds(k_cache, bounds, _as_i32(block_table), _as_i32(seq_lens), int(max_new))


def select_blocks(query: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  max_seq_len: int, block_size: int, keep: int, sink: int = 1, recent: int = 2) -> torch.Tensor:
    """``[n, H_kv, keep]`` int32: per request and KV head the logical blocks (places in the request's block-table row)
    that query [n, H_q, 128] reads, ascending, -1 behind the last.

    The first `sink` and the last `recent` blocks are always read; between them the largest
    ``sum_g sum_d max(q_gd lo_d, q_gd hi_d)``, an upper bound of the block's scores summed over the KV head's query
    heads. Scores are summed in 64 bits and compared in fp32, equal ones go to the lower block, so
    the choice does not depend on batch or launch. Requests of at most `keep` blocks read all of them."""
    n = query.shape[0]
    _hip.require_cuda(query, bounds, block_table, seq_lens)
    _hip.refuse_grad("select_blocks", query, bounds)
    if sink < 0 or recent < 0 or keep < 1 or sink + recent > keep:
        raise ValueError(f"select_blocks: keep={keep} blocks, sink={sink} and recent={recent} among them")
    selected = query.new_empty((n, bounds.shape[1], int(keep)), dtype=torch.int32)
    if n:
        _hip.ops().select_blocks(query, bounds, _as_i32(block_table), _as_i32(seq_lens), int(max_seq_len),
                                 int(block_size), int(sink), int(recent), selected)
    return selected


def paged_decode_sparse(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                        seq_lens: torch.Tensor, selected: torch.Tensor, scale: float) -> torch.Tensor:
    """``[n, H_q, 128]``: ``paged_decode_full`` over the tokens of the blocks that `selected` [n, H_kv, keep] names for
    each request and KV head (each at most once; a place outside the request's blocks, such as -1, holds no
    tokens). Up to 16 query heads per KV head, any number; query of the cache's dtype. A row without
    tokens is zero, one whose scores are all -inf NaN."""
    _hip.require_cuda(query, k_cache, v_cache, block_table, seq_lens, selected)
    _hip.refuse_grad("paged_decode_sparse", query, k_cache, v_cache)
    out = torch.empty_like(query, memory_format=torch.contiguous_format)
    if query.shape[0]:
        _hip.ops().sparse_decode(query, k_cache, v_cache, _as_i32(block_table), _as_i32(seq_lens), selected,
                                 float(scale), out)
    return out
