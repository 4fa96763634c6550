"""Prompts through a window: what is refused before anything is launched (CPU)."""
import pytest
import torch

from starkv_serve import _hip
from starkv_serve.kernels.prefill import prompt_tables


def test_tables_are_not_made_in_a_capture(monkeypatch):
    """A graph would upload them from memory that is gone by its first replay."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for device in ("cuda", torch.device("cuda", 0)):
        with pytest.raises(RuntimeError, match="tables="):
            prompt_tables([3, 4], device)
    cu, blocks = prompt_tables([3, 0, 140], "cpu")
    assert cu.tolist() == [0, 3, 3, 143] and blocks.tolist() == [[2, 1], [2, 0], [0, 0]]


P = 4096  # a 16-byte aligned address that is never read
GOOD = dict(stream=None, q=P, q0=512, q1=128, k=P, k0=256, k1=128, v=P + 2, v0=256, v1=128, cu=P, blk=P, blocks=3, tokens=300, hq=4, heads=2, D=128,
            window=8, sinks=1, scale=0.1, out=P, o0=512, o1=128, odt=2, ws=P, bytes=2 * (300 * 256 + 304))


@pytest.mark.parametrize("key,value,message", [("window", 0, b"window"), ("sinks", -1, b"sinks"), ("D", 64, b"head_size"), ("q", None, b"null"),
                                               ("k", None, b"null"), ("v", None, b"null"), ("v", P + 1, b"odd"), ("out", None, b"null"), ("ws", None, b"null"),
                                               ("ws", P + 8, b"odd"), ("bytes", 2 * (300 * 256 + 304) - 1, b"workspace"), ("hq", 5, b"heads"), ("heads", 0, b"heads"),
                                               ("tokens", -1, b"tokens"), ("q0", 4, b"aligned"), ("k1", 4, b"aligned"), ("k0", 1 << 24, b"stride"), ("o0", 2, b"aligned"),
                                               ("odt", 3, b"dtypes"), ("blocks", -1, b"num_blocks")])
def test_bf16_prompts_refuse(key, value, message):
    """Before anything is launched."""
    L = _hip.lib()
    assert L.starkv_prefill_window_bf16_workspace_bytes(300, 2) == 2 * (300 * 256 + 304)
    args = dict(GOOD, **{key: value})
    assert L.starkv_prefill_window_bf16(*args.values()) != 0
    assert message in L.starkv_last_error(), L.starkv_last_error()


def test_no_tokens():
    assert _hip.lib().starkv_prefill_window_bf16(*dict(GOOD, tokens=0, blocks=0, bytes=0).values()) == 0


def test_conversion_takes_keys_and_values():
    """The operator that makes fp16 rows has both."""
    schema = str(_hip.ops().prefill_to_half.default._schema)
    assert schema == "starkv::prefill_to_half(Tensor key, Tensor value, Tensor(a!) key_out, Tensor(b!) value_out) -> ()"
    L = _hip.lib()
    assert L.starkv_prefill_to_half(None, None, 0, 0, None, P, 256, 128, P, 2, 4, 2) != 0 and b"null" in L.starkv_last_error()
