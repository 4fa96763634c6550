"""Attention through a window on MI355X (libstarkv_hip.so): a token sees the last tokens in front of it, itself among
them, and a few first ones that stay visible.

``Window(size, sinks)``: the token at place t of its request sees place s <= t where t - s < size or s < sinks. Decode
steps take it through ``paged_decode_window`` here, over an 8-bit cache through ``cache8.paged_decode_8``, prompts
through ``prefill.prefill_attention(window=)``. No operator here has a gradient: calls that want one raise. The reference
has no counterpart; its uncompressed layers attend to their whole cache (starkv_serve/model.py:77-81 there).
"""
from dataclasses import dataclass
from typing import Optional

import torch

from starkv_serve import _hip
from starkv_serve.kernels.paged_decode import _as_i32


@dataclass(frozen=True)
class Window:
    """The last `size` tokens, the token's own among them, and the first `sinks`."""
    size: int
    sinks: int = 0

    def __post_init__(self):
        if not 1 <= self.size < 2 ** 31 or not 0 <= self.sinks < 2 ** 31:
            raise ValueError(f"{self}: at least the token itself, and 0 or more first tokens")


def sizes(window: Optional[Window]) -> tuple:
    """(size, sinks) as the operators take them; (0, 0): all tokens."""
    return (0, 0) if window is None else (int(window.size), int(window.sinks))


def paged_decode_window(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                        seq_lens: torch.Tensor, max_seq_len: int, scale: float, window: Window) -> torch.Tensor:
    """``[n, H_q, 128]``: ``paged_decode_full`` through `window`: the token at place seq_lens[b] - 1 of request b. Up to 16
    query heads per KV head, any number; query of the cache's dtype; lengths are cut to max_seq_len. Blocks of
    which nothing is seen are not read, nor their entries of the block table, so a caller may have given them
    away. A row without tokens is zero, one whose scores are all -inf NaN."""
    _hip.require_cuda(query, k_cache, v_cache, block_table, seq_lens)
    _hip.refuse_grad("paged_decode_window", query, k_cache, v_cache)
    return _hip.ops().window_decode(query, k_cache, v_cache, _as_i32(block_table), _as_i32(seq_lens), int(max_seq_len),
                                    *sizes(window), float(scale))
