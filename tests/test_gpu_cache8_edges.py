"""8-bit caches and windows on the GPU, at the ends of what their operators take."""
import pytest
import torch

from cache8_plain import D, SCALE
from starkv_serve.kernels.cache8 import Cache8, paged_decode_8, read_kv8, write_kv8
from starkv_serve.kernels.window import Window, paged_decode_window

pytestmark = pytest.mark.gpu

BF16, I8, F8 = torch.bfloat16, torch.int8, torch.float8_e4m3fn


def test_caches_without_heads_are_refused(cuda):
    """By an error: a number of query heads is divided by theirs."""
    c = Cache8.zeros(4, 16, 0, I8, cuda)
    kc = torch.zeros(4, 16, 0, D, dtype=BF16, device=cuda)
    bt, sl = torch.zeros(2, 2, dtype=torch.int32, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    for heads in (0, 4):
        q = torch.zeros(2, heads, D, dtype=BF16, device=cuda)
        with pytest.raises(RuntimeError, match="KV heads"):
            paged_decode_8(q, c, bt, sl, 32, SCALE)
        with pytest.raises(RuntimeError, match="KV heads"):
            paged_decode_window(q, kc, kc, bt, sl, 32, SCALE, Window(8))
    rows = torch.zeros(2, 0, D, dtype=BF16, device=cuda)
    for call in (lambda: write_kv8(rows, rows, c, sl), lambda: read_kv8(c, sl)):
        with pytest.raises(RuntimeError, match="num_kv_heads"):
            call()
