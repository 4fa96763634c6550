"""Limits that the host keeps before anything is launched (CPU): positions of sessions whose caches are cut, which the
cache's length no longer bounds, and the rows that prompts take of a weighing model's sums."""
import pytest
import torch

from starkv_serve import model as M

SHAPE = M.LlamaShape(hidden_size=64, num_layers=1, num_heads=1, num_kv_heads=1, intermediate_size=64, vocab_size=10)
TABLE = torch.arange(8, dtype=torch.int32).view(2, 4)


def weighing(monkeypatch, **kw):
    """A model whose layers do nothing: what reaches them has passed the checks."""
    model = M.StarKVLlamaForCausalLM(SHAPE, None, 64, "cpu", weigh=True, **kw)
    model.allocate_kv_cache(9, 16, 2)
    model.ran = []
    monkeypatch.setattr(model, "_layers", lambda x, positions, *a: model.ran.append(positions) or x)
    return model


def step(model, positions, lens, **kw):
    md = M.decode_metadata(TABLE, torch.tensor(positions), 16, 64, None if lens is None else torch.tensor(lens), **kw)
    return model.decode_step(torch.zeros(len(positions), dtype=torch.int64), torch.tensor(positions), md)


def test_positions_stay_in_the_rotary_table(monkeypatch):
    model = weighing(monkeypatch)
    assert model.rotary.cos_sin_cache.shape[0] == 65
    step(model, [64, 3], [20, 3])
    with pytest.raises(ValueError, match="position 65 .* 65 rows"):
        step(model, [3, 65], [3, 20])
    with pytest.raises(ValueError, match="position 90"):  # by the caller's bound, without a look at the positions
        step(model, [3, 4], [3, 4], max_position=90)
    step(model, [3, 64], [3, 20], max_position=64)
    step(model, [63, 3], None)
    assert len(model.ran) == 3


def test_a_model_takes_more_positions_than_its_caches_hold(monkeypatch):
    model = weighing(monkeypatch, max_positions=1000)
    assert model.rotary.cos_sin_cache.shape[0] == 1001 and model.max_model_len == 64
    step(model, [1000, 3], [20, 3])
    with pytest.raises(ValueError, match="position 1001"):
        step(model, [1001, 3], [20, 3])
    assert torch.equal(model.rotary.cos_sin_cache[:65], weighing(monkeypatch).rotary.cos_sin_cache)
    assert weighing(monkeypatch, max_positions=5).rotary.cos_sin_cache.shape[0] == 65  # no fewer than before


def test_a_rotation_of_the_callers_has_its_own_limit(monkeypatch):
    model = weighing(monkeypatch)
    model.rotary.apply = lambda positions, x: x
    step(model, [700, 3], [20, 3])
    assert len(model.ran) == 1


class Replays:
    """A graph's host side, without a device."""

    def __init__(self, graph):
        self.graph, self.n = graph, 0

    def replay(self):
        self.n += 1
        self.graph.positions += 1
        if self.graph.lens is not None:
            self.graph.lens += 1


def graph_of(model, positions, lens):
    g = M.DecodeGraph.__new__(M.DecodeGraph)
    g.model, g.block_table = model, TABLE
    g.tokens, g.positions = torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    g.lens = None if lens is None else torch.zeros(2, dtype=torch.int64)
    g.graph = Replays(g)
    g.reset(g.tokens, torch.tensor(positions), None if lens is None else torch.tensor(lens))
    return g


def test_replays_stay_in_the_rotary_table(monkeypatch):
    model = weighing(monkeypatch, max_positions=100)
    g = graph_of(model, [90, 5], [10, 5])
    for _ in range(11):  # positions 90 .. 100
        g.replay()
    with pytest.raises(ValueError, match="position"):
        g.replay()
    assert g.graph.n == 11 and g.positions.tolist() == [101, 16]
    g.reset(g.tokens, torch.tensor([99, 5]), torch.tensor([10, 5]))
    g.replay()
    g.replay()
    with pytest.raises(ValueError, match="position"):
        g.replay()


def test_replays_stay_in_the_cache_and_go_on_after_a_cut(monkeypatch):
    model = weighing(monkeypatch, max_positions=1000)
    g = graph_of(model, [60, 30], [60, 30])
    for _ in range(4):  # lengths 60 .. 63 before the token
        g.replay()
    with pytest.raises(ValueError, match="64 tokens"):
        g.replay()
    g.lens.copy_(torch.tensor([20, 20]))  # a cut
    for _ in range(44):
        g.replay()
    with pytest.raises(ValueError, match="64 tokens"):
        g.replay()
    assert g.graph.n == 48 and g.positions.tolist() == [108, 78]


def test_replays_without_lengths_are_not_counted(monkeypatch):
    g = graph_of(weighing(monkeypatch), [60, 30], None)
    for _ in range(3):
        g.replay()
    assert g.graph.n == 3


def test_a_graph_does_not_start_behind_the_limits(monkeypatch):
    model = weighing(monkeypatch)
    tokens = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="64 tokens"):
        M.DecodeGraph(model, TABLE, tokens, torch.tensor([64, 3]), torch.tensor([64, 3]))
    with pytest.raises(ValueError, match="position 70"):
        M.DecodeGraph(model, TABLE, tokens, torch.tensor([70, 3]), torch.tensor([20, 3]))
    assert not model.ran


def prompts(model, lens, **kw):
    table = torch.arange(4 * len(lens), dtype=torch.int32).view(len(lens), 4)
    md, positions = M.prefill_metadata(table, lens, 16)
    return model.prefill_step(torch.zeros(sum(lens), dtype=torch.int64), positions, md, **kw)


@pytest.mark.parametrize("lens,rows,message", [
    ([5, 3, 4], None, "3 prompts"), ([5, 3], [0, 2], "rows"), ([5, 3], torch.tensor([0, 7]), "rows"),
    ([5, 3], [-1, 0], "rows"), ([5, 3], [1, 1], "rows"), ([5, 3], [0], "rows"), ([5], torch.tensor([0, 1]), "rows"),
    ([5, 3], torch.tensor([[0, 1]]), "rows"), ([5, 3], torch.tensor([0.0, 1.0]), "rows"), ([5, 3], [True, False], "rows")])
def test_prompts_take_rows_that_are_there(monkeypatch, lens, rows, message):
    model = weighing(monkeypatch)
    with pytest.raises(ValueError, match=message):
        prompts(model, lens, rows=rows)
    assert not model.ran


def test_prompts_rows(monkeypatch):
    model = weighing(monkeypatch)
    for lens, rows in (([5, 3], None), ([5, 3], [1, 0]), ([5], torch.tensor([1])), ([5], (0,)),
                       ([5, 3], torch.tensor([1, 0], dtype=torch.int32))):
        prompts(model, lens, rows=rows)
    assert len(model.ran) == 5
    with pytest.raises(RuntimeError, match="allocate_kv_cache"):
        prompts(M.StarKVLlamaForCausalLM(SHAPE, None, 64, "cpu", weigh=True), [5])
