"""Replays of captured calls and prefill: what the device holds decides, not which calls Python has seen."""

import pytest
import torch

import sink_window_attention as swa

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def cache(storage=None):
    return swa.SinkWindowStreamingAttention(32, 32, streams=2, heads=4, kv_heads=2, window=24, sinks=2, storage=storage,
                                            dtype=torch.bfloat16, device=DEV)


def rows(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(2, h, n, 32, generator=g).bfloat16().to(DEV) for h in (4, 2, 2)]


def captured(f):
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = f()
    return graph, out


def test_prefill_sees_replayed_tokens():
    a = cache()
    q, k, v = rows(30, 1)
    graph, _ = captured(lambda: a.step(q[:, :, 0], k[:, :, 0], v[:, :, 0]))
    a.reset()
    graph.replay()
    with pytest.raises(ValueError, match="empty state"):
        a.prefill(q, k, v)
    assert a.lengths.tolist() == [1, 1]
    a.reset()
    assert torch.equal(a.prefill(q, k, v), cache().prefill(q, k, v))
    a.reset([0])  # the other stream still holds its tokens
    with pytest.raises(ValueError, match="empty state"):
        a.prefill(q, k, v)


def test_prefill_after_a_replayed_reset():
    a = cache()
    q, k, v = rows(30, 2)
    graph, _ = captured(a.reset)
    a.extend(k, v)
    with pytest.raises(ValueError, match="empty state"):
        a.prefill(q, k, v)
    graph.replay()
    assert torch.equal(a.prefill(q, k, v), cache().prefill(q, k, v))
    state = cache().state_dict()
    a.load_state_dict(state)
    assert torch.equal(a.prefill(q, k, v), cache().prefill(q, k, v))


@pytest.mark.parametrize("storage", [None, "fp4"])
def test_captured_prefill_starts_from_an_empty_state(storage):
    a = cache(storage)
    q, k, v = rows(40, 3)
    counts = torch.tensor([40, 17], dtype=torch.int32, device=DEV)
    graph, out = captured(lambda: a.prefill(q, k, v, counts=counts))
    for seed in (4, 5, 6):
        new = rows(41, seed)
        for x, y in zip((q, k, v), new):
            x.copy_(y[:, :, :40])
        graph.replay()
        b = cache(storage)
        assert torch.equal(out, b.prefill(q, k, v, counts=counts))
        token = [x[:, :, 40] for x in new]
        for _ in range(2):
            assert torch.equal(a.step(*token), b.step(*token))
        assert torch.equal(a.lengths, b.lengths)
