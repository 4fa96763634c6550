"""Prompts through a window: what is refused before anything is launched (CPU)."""
import pytest
import torch

from starkv_serve.kernels.prefill import prompt_tables


def test_tables_are_not_made_in_a_capture(monkeypatch):
    """A graph would upload them from memory that is gone by its first replay."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    for device in ("cuda", torch.device("cuda", 0)):
        with pytest.raises(RuntimeError, match="tables="):
            prompt_tables([3, 4], device)
    cu, blocks = prompt_tables([3, 0, 140], "cpu")
    assert cu.tolist() == [0, 3, 3, 143] and blocks.tolist() == [[2, 1], [2, 0], [0, 0]]
