"""Dense causal prefill attention on MI355X (libstarkv_hip.so, starkv_prefill_attention).

The attention half of the STAR-KV layer's prefill (starkv_serve/attention.py:219-251 in
the reference, which hands the lifted K and V to vLLM's flash_attn_varlen_func with
causal=True): every prompt attends to itself, no cached context.
"""
import ctypes
from typing import List, Optional

import torch

from starkv_serve import _hip
from starkv_serve.kernels.window import Window, sizes


def _tables(query_lens: List[int]) -> tuple:
    """The prompts' first tokens and their ends, then the workgroup rows, as int32 in one buffer; how many of the latter."""
    cu = [0]
    for L in query_lens:
        if L < 0:
            raise ValueError(f"negative prompt length {L}")
        cu.append(cu[-1] + int(L))
    lib, P = _hip.lib(), len(cu)
    cu_c = (ctypes.c_int32 * P)(*cu)
    n = lib.starkv_prefill_block_list(cu_c, P - 1, None, 0)
    buf = (ctypes.c_int32 * (P + 2 * max(n, 1)))()
    rows = (ctypes.c_int32 * (2 * max(n, 1))).from_buffer(buf, 4 * P)
    if n < 0 or lib.starkv_prefill_block_list(cu_c, P - 1, rows, n) != n:
        raise RuntimeError("starkv_prefill_block_list failed")
    ctypes.memmove(buf, cu_c, 4 * P)
    return buf, n


def block_list(query_lens: List[int]) -> List[int]:
    """The kernel's workgroup rows, (prompt, query block) pairs flattened, from the
    library's host helper starkv_prefill_block_list (the query block size is the
    kernel's): the blocks with the most keys first."""
    buf, n = _tables(query_lens)
    P = len(query_lens) + 1
    return buf[P:P + 2 * n]


def prompt_tables(query_lens: List[int], device) -> tuple:
    """(cu_seqlens [P + 1], blocks [num_blocks, 2]) int32 on `device`, in one upload. Made before a capture: a graph would
    read them from this call's host memory again at each replay."""
    if torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("in a capture the prompts' tables are those of prompt_tables(), made before it: tables=")
    buf, n = _tables(query_lens)
    P = len(query_lens) + 1
    meta = torch.frombuffer(buf, dtype=torch.int32).to(device, non_blocking=True)
    return meta[:P], meta.as_strided((n, 2), (2, 1), P)


def prefill_lift(k_codes: torch.Tensor, v_codes: torch.Tensor, cu_seqlens: torch.Tensor, k_up: torch.Tensor,
                 k_offsets: torch.Tensor, k_widths: torch.Tensor, cos_sin: torch.Tensor) -> tuple:
    """The step's lifted keys and the V codes in fp16 (V's product's left operand), in one
    launch (starkv_prefill_lift): K [T, H_kv, 128] = RoPE(codes @ U), formed in fp32 and
    rounded once to fp16.

    k_codes [T, W], v_codes [T, r_v] (bf16, fp16 or fp32, contiguous rows); k_up [W, 128]
    fp32, rank-major; cos_sin [positions, 128] covering the longest prompt. fp16 V codes
    are returned as they are."""
    T = k_codes.shape[0]
    _hip.require_cuda(k_codes, v_codes, cu_seqlens, k_up, k_offsets, k_widths, cos_sin)
    key = torch.empty(T, k_offsets.numel(), 128, dtype=torch.float16, device=k_codes.device)
    if v_codes.dtype != k_codes.dtype:
        v_codes = v_codes.to(torch.float16)
    v16 = None
    if v_codes.dtype != torch.float16:
        v16 = torch.empty(v_codes.shape, dtype=torch.float16, device=v_codes.device)
    _hip.ops().prefill_lift(k_codes, v_codes, cu_seqlens, k_up, k_offsets, k_widths, cos_sin, key, v16)
    return key, v_codes if v16 is None else v16


def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, query_lens: List[int], scale: float,
                      out: Optional[torch.Tensor] = None, tables: Optional[tuple] = None,
                      window: Optional[Window] = None) -> torch.Tensor:
    """Causal attention of each prompt to itself, through `window` where there is one (which has no gradient: calls that want
    one raise).

    q [T, H_q, 128] (bf16, fp16 or fp32; to fp16 in the kernel); k, v [T, H_kv, 128] (converted to fp16 once here when they
    are not: values past its range become infinite, those below 2^-14 lose bits). Through a window bf16 q, k and v go as they
    are, over bf16's whole range: a value below 2^-17 among larger ones (2^-10 or more) is off by 2^-25 at most. query_lens: the
    prompts' token counts (host ints, summing to T); tables: their ``prompt_tables``, when the caller has them (in a capture
    it must). Returns ``out`` [T, H_q, 128] (new, in q's dtype, when not given)."""
    T, Hq, D = q.shape
    assert D == 128 and k.shape == v.shape and k.shape[0] == T and k.shape[2] == D and Hq % k.shape[1] == 0
    assert sum(query_lens) == T
    if window is not None:
        _hip.refuse_grad("prefill_attention through a window", q, k, v)
    if out is None:
        out = torch.empty_like(q)
    if T == 0:
        return out
    _hip.require_cuda(q, k, v, out)
    # Through a window rows of one type go as they are: bf16 over its whole range (keys 16-byte aligned), fp16 where keys and
    # values share their strides. All others become fp16.
    rows = window is not None and q.dtype == k.dtype == v.dtype
    aligned = rows and k.stride(-1) == v.stride(-1) == 1 and k.stride(0) % 8 == k.stride(1) % 8 == k.data_ptr() % 16 == 0 and k.stride(0) < 1 << 23
    if rows and k.dtype == torch.bfloat16:
        if not aligned:
            k, v = (t.clone(memory_format=torch.contiguous_format) for t in (k, v))
    elif not (aligned and k.dtype == torch.float16 and k.stride() == v.stride() and v.data_ptr() % 16 == 0):
        if k.dtype == v.dtype and k.dtype in (torch.bfloat16, torch.float32) and k.stride(-1) == v.stride(-1) == 1:
            kv = torch.empty((2, *k.shape), dtype=torch.float16, device=k.device)
            _hip.ops().prefill_to_half(k, v, kv[0], kv[1])
            k, v = kv[0], kv[1]
        k, v = k.to(torch.float16), v.to(torch.float16)
        k, v = k.contiguous(), v.contiguous()
    q = q if q.stride(-1) == 1 else q.contiguous()
    if window is not None:
        if tables is None and min(query_lens) < 0:
            raise ValueError(f"negative prompt length {min(query_lens)}")
        cu_d, blk_d = (None, None) if tables is None else tables
        _hip.ops().prefill_window(q, k, v, cu_d, blk_d, list(map(int, query_lens)) if tables is None else [], *sizes(window), float(scale), out)
        return out
    cu_d, blk_d = prompt_tables(query_lens, q.device) if tables is None else tables
    _hip.ops().prefill(q, k, v, cu_d, blk_d, float(scale), out)
    return out
