"""The operators over uncompressed caches on a stream of the caller's: their inputs are written there, behind work that
keeps it busy, over other inputs that are as valid. A launch on any other stream would read those, and results are copied
on the caller's stream too."""
import pytest
import torch

from test_gpu_cache_ops import make_all, run_all, same

pytestmark = pytest.mark.gpu


def test_inputs_written_on_the_callers_stream(cuda):
    source, x = make_all(cuda, 151), make_all(cuda, 152)
    assert all(x[k].shape == source[k].shape and not same(x[k], source[k]) for k in ("q", "kc", "vc", "weights", "table", "w"))
    want = run_all(make_all(cuda, 151))
    busy = torch.randn(4096, 4096, device=cuda)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(30):
            busy = busy @ busy * 1e-3
        for k, t in x.items():
            t.copy_(source[k])
        got = [t.clone() for t in run_all(x)]
    stream.synchronize()
    for a, b in zip(got, want):
        assert same(a, b)
