"""8-bit caches of uncompressed layers on MI355X (libstarkv_hip.so): keys and values quantised as they are written, read
back, and one token's attention over them.

``Cache8`` holds codes of one byte in the shape of ``paged_decode_full``'s caches and, for each block and KV head, an
exponent of the keys and one of the values: a value is code * 2^exponent. Codes are int8 (up to 127) or e4m3 (up to 448).
Scales are powers of two, so a code's only error is its own rounding: half a step, which is 2^-8 of the block's largest
value at least and up to 2^-7 (int8), or 2^-4 of the value itself (e4m3). Block tables, lengths and slots are
those of the 16-bit caches. No operator here has a gradient: calls that want one raise. The reference has no
counterpart; its uncompressed layers keep 16 bits (starkv_serve/model.py:77-81 there).
"""
from dataclasses import dataclass
from typing import Optional

import torch

from starkv_serve import _hip
from starkv_serve.kernels.paged_decode import _as_i32
from starkv_serve.kernels.window import Window, sizes

CODE_TYPES = (torch.int8, torch.float8_e4m3fn)
LEAST_EXPONENT = -126  # that of a block of zeros; -128 stands for NaN


@dataclass
class Cache8:
    """k and v [num_blocks, block_size, H_kv, 128] of one code type and layout (any strides that are multiples of 16
    behind the last dimension), exponents [num_blocks, H_kv, 2] int8 (of k, of v)."""
    k: torch.Tensor
    v: torch.Tensor
    exponents: torch.Tensor

    @classmethod
    def zeros(cls, num_blocks: int, block_size: int, num_kv_heads: int, dtype: torch.dtype, device,
              head_dim: int = 128) -> "Cache8":
        """A cache of zeros. A block's rows of one head lie together: a page of 16 tokens is 2 KB that a decode reads
        as one run."""
        if dtype not in CODE_TYPES:
            raise ValueError(f"8-bit caches hold torch.int8 or torch.float8_e4m3fn, not {dtype}")
        if block_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError(f"blocks of {block_size} tokens: 16 times a power of two, at most 1024")
        k, v = (torch.zeros(num_blocks, num_kv_heads, block_size, head_dim, dtype=torch.int8, device=device).view(dtype)
                .transpose(1, 2) for _ in range(2))
        return cls(k, v, torch.full((num_blocks, num_kv_heads, 2), LEAST_EXPONENT, dtype=torch.int8, device=device))

    @property
    def dtype(self) -> torch.dtype:
        return self.k.dtype

    @property
    def tensors(self) -> tuple:
        return self.k, self.v, self.exponents


def _slots(what: str, slot_mapping: torch.Tensor, n: Optional[int] = None) -> torch.Tensor:
    if slot_mapping.dim() != 1 or slot_mapping.is_floating_point() or slot_mapping.dtype == torch.bool or (
            n is not None and slot_mapping.shape[0] != n):
        raise ValueError(f"{what}: slots {tuple(slot_mapping.shape)} of {slot_mapping.dtype}"
                         + ("" if n is None else f" for {n} tokens"))
    return slot_mapping.contiguous() if slot_mapping.dtype == torch.int64 else _as_i32(slot_mapping)


def write_kv8(key: torch.Tensor, value: torch.Tensor, cache: Cache8, slot_mapping: torch.Tensor) -> None:
    """The step's ``key`` / ``value`` [n, H_kv, 128] (bf16 or fp16) into `cache` at ``slot_mapping`` [n] (distinct; one
    outside the cache, such as -1: nothing), as ``write_kv_full`` does for 16-bit caches.

    Per block, head, and of the two: a call that writes the block's first token begins the block anew, with the least
    exponent (at least -126) at which its own largest value has a code, and leaves the block's other rows as they
    are. Any other call keeps the exponent, or raises it to what its values need and rounds the codes that are there
    to it; an exponent never falls until its block begins anew. Values that are infinite or NaN give the block's head the exponent -128: all its values are NaN until it begins
    anew. Results do not depend on the order of slots, nor on how requests share a call."""
    _hip.require_cuda(key, value, *cache.tensors, slot_mapping)
    _hip.refuse_grad("write_kv8", key, value)
    slots = _slots("write_kv8", slot_mapping, key.shape[0])
    if key.shape[0]:
        _hip.ops().write_kv8(key, value, *cache.tensors, slots)


def read_kv8(cache: Cache8, slot_mapping: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> tuple:
    """The keys and values at ``slot_mapping`` [n] as (k, v) [n, H_kv, 128] of `dtype` (bf16, fp16 or fp32, rounded once);
    zeros at a slot outside the cache."""
    _hip.require_cuda(*cache.tensors, slot_mapping)
    _hip.refuse_grad("read_kv8")
    slots = _slots("read_kv8", slot_mapping)
    return _hip.ops().read_kv8(*cache.tensors, slots, dtype)


def paged_decode_8(query: torch.Tensor, cache: Cache8, block_table: torch.Tensor, seq_lens: torch.Tensor,
                   max_seq_len: int, scale: float, window: Optional[Window] = None) -> torch.Tensor:
    """``[n, H_q, 128]``: ``paged_decode_full`` over an 8-bit cache, through `window` where there is one. query [n, H_q, 128]
    (bf16 or fp16), up to 16 query heads per KV head, any number; lengths are cut to max_seq_len. A row without
    tokens is zero, one whose scores are all -inf NaN, as is one that sees a block of exponent -128. Through a window, blocks
    of which nothing is seen are not read, nor their entries of the block table."""
    _hip.require_cuda(query, *cache.tensors, block_table, seq_lens)
    _hip.refuse_grad("paged_decode_8", query)
    return _hip.ops().decode_kv8(query, *cache.tensors, _as_i32(block_table), _as_i32(seq_lens), int(max_seq_len),
                                 *sizes(window), float(scale))
