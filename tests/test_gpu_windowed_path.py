"""The windowed operators together, as a model's layer uses them: norm and rotation, attention over a prompt, the prompt
into the cache, and token after token from there; and a training step through all of it."""

import math
import threading

import pytest
import torch

import benchmark_attention as bench_mod
import qk_rotary as qkr
import sink_window_attention as swa
import window_reference as ref

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.mark.parametrize("storage", [None, "fp4"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_prompt_then_tokens(dtype, storage):
    s, h, hk, d, window, sinks = 3, 4, 2, 64, 48, 4
    prompt = [90, 1, 37]
    steps = 60
    total = max(prompt) + steps
    g = torch.Generator().manual_seed(3)
    q0, k0, v0 = (torch.randn(s, x, total, d, generator=g).to(dtype).to(DEV) for x in (h, hk, hk))
    w = [(torch.rand(d, generator=g) + 0.5).to(DEV) for _ in range(2)]
    table = qkr.rotary_table(total, d, device=DEV)
    # every token's rows at once, then the same rows as a server sees them
    q, k = qkr.qk_norm_rotary(q0, k0, table, q_weight=w[0], k_weight=w[1])
    rows = max(prompt)
    a = swa.SinkWindowStreamingAttention(d, d, streams=s, heads=h, kv_heads=hk, window=window, sinks=sinks, dtype=dtype,
                                         storage=storage, device=DEV)
    counts = torch.tensor(prompt, dtype=torch.int32, device=DEV)
    pq, pk = qkr.qk_norm_rotary(q0[:, :, :rows], k0[:, :, :rows], table, q_weight=w[0], k_weight=w[1])
    out = a.prefill(pq, pk, v0[:, :, :rows], counts=counts)
    want = ref.window_attention(q.cpu()[:, :, :rows], k.cpu()[:, :, :rows], v0.cpu()[:, :, :rows], window=window,
                                sinks=sinks, lengths=prompt)
    assert ref.over(out, want["out"]) <= 1.0
    cache = ref.TokenCache(s, window, sinks, storage)
    for i in range(s):
        for p in range(prompt[i]):
            cache.put(i, k[i, :, p].cpu(), v0[i, :, p].cpu())
    pick = torch.arange(s, device=DEV)
    for t in range(steps):
        at = counts.long() + t
        tq, tk, tv = (x[pick, :, at] for x in (q0, k0, v0))
        tq, tk = qkr.qk_norm_rotary(tq, tk, table, q_weight=w[0], k_weight=w[1], positions=at)
        assert torch.equal(tq, q[pick, :, at]) and torch.equal(tk, k[pick, :, at])
        out = a.step(tq, tk, tv)
        for i in range(s):
            cache.put(i, tk[i].cpu(), tv[i].cpu())
            assert ref.over(out[i], cache.query(i, tq[i].cpu(), a.scale, dtype)) <= 1.0
    assert a.lengths.tolist() == [p + steps for p in prompt]
    with pytest.raises(ValueError, match="empty state"):
        a.prefill(pq, pk, v0[:, :, :rows])


def test_steps_equal_the_prompts_rows():
    """Exact storage: a step's output is the prompt's row, up to the order of its sums."""
    s, h, d, n, window, sinks = 2, 2, 64, 300, 64, 4
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(s, h, n, d, generator=g).to(DEV) for _ in range(3))
    out = swa.sink_window_causal_attention(q, k, v, window=window, sinks=sinks)
    bound = ref.window_attention(q.cpu(), k.cpu(), v.cpu(), window=window, sinks=sinks)["out"][1].to(DEV)
    a = swa.SinkWindowStreamingAttention(d, d, streams=s, heads=h, window=window, sinks=sinks, device=DEV)
    for i in range(n):
        o = a.step(q[:, :, i], k[:, :, i], v[:, :, i])
        assert ((o - out[:, :, i]).abs() <= 2.1 * bound[:, :, i]).all()


def test_training_step_through_both():
    """Gradients of q, k, v and the weights through rotation and attention, against float64 autograd."""
    b, h, hk, n, d = 2, 4, 2, 150, 32
    g = torch.Generator().manual_seed(5)
    x = [torch.randn(b, m, n, d, generator=g) for m in (h, hk, hk)] + [torch.rand(d, generator=g) + 0.5 for _ in range(2)]
    go = torch.randn(b, h, n, d, generator=g)
    table = qkr.rotary_table(n, d)
    mine = [t.to(DEV).requires_grad_() for t in x]
    q, k = qkr.qk_norm_rotary(mine[0], mine[1], table.to(DEV), q_weight=mine[3], k_weight=mine[4])
    out = swa.sink_window_causal_attention(q, k, mine[2], window=40, sinks=3)
    got = torch.autograd.grad(out, mine, go.to(DEV))
    want_in = [t.double().requires_grad_() for t in x]
    cos, sin = table.double().chunk(2, -1)

    def turn(t, w):
        t = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        a_, b_ = t.chunk(2, -1)
        return torch.cat([a_ * cos - b_ * sin, b_ * cos + a_ * sin], -1)

    qd, kd = turn(want_in[0], want_in[3]), turn(want_in[1], want_in[4])
    see = ref.visible(n, n, 40, 3)
    p = (qd @ kd.repeat_interleave(2, 1).transpose(-1, -2) / math.sqrt(d)).masked_fill(~see, -math.inf).softmax(-1)
    want = torch.autograd.grad(p @ want_in[2].repeat_interleave(2, 1), want_in, go.double())
    for y, z in zip(got, want):
        # logits up to 10 off by 32 2^-23 of that, 4e-5 of a weight at most, and sums of 43 such weights: relative to
        # the tensor's size, 1e-5 is above what they leave on average (sqrt(43) terms of 4e-5 / sqrt(32) over 43)
        assert (y.double().cpu() - z).norm() <= 1e-5 * z.norm()


def test_two_objects_and_streams():
    """Two caches stepped on two streams at once do not meet."""
    g = torch.Generator().manual_seed(6)
    make = lambda: swa.SinkWindowStreamingAttention(64, 64, streams=1, heads=4, kv_heads=1, window=4000, sinks=4,
                                                    dtype=torch.bfloat16, storage="fp4", device=DEV)
    a, b, a1, b1 = make(), make(), make(), make()
    x = [torch.randn(1, m, 3000, 64, generator=g).to(torch.bfloat16).to(DEV) for m in (1, 1, 1, 1)]
    a.extend(x[0], x[1]), a1.extend(x[0], x[1]), b.extend(x[2], x[3]), b1.extend(x[2], x[3])
    q = [torch.randn(1, 4, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(20)]
    k = [torch.randn(1, 1, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(20)]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for i in range(20):
        for j, obj in enumerate((a, b)):
            with torch.cuda.stream(side[j]):
                outs[j].append(obj.step(q[i], k[i], k[19 - i]))
    torch.cuda.synchronize()
    for i in range(20):
        assert torch.equal(outs[0][i], a1.step(q[i], k[i], k[19 - i]))
        assert torch.equal(outs[1][i], b1.step(q[i], k[i], k[19 - i]))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_benchmark_command(tmp_path, capsys, dtype):
    """--window adds its columns behind the others, which stay as they are without it; a window as long as the sequence
    is exact attention."""
    plain = bench_mod.main(["--sweep-n", "96", "--repeats", "1", "--csv", str(tmp_path / "a.csv"), "--dtype", dtype])
    assert list(plain[0]) == list(bench_mod.COLUMNS) and "window" not in capsys.readouterr().out
    rows = bench_mod.main(["--sweep-n", "96", "300", "--repeats", "1", "--csv", str(tmp_path / "b.csv"), "--dtype", dtype,
                           "--window", "100", "--sinks", "3"])
    assert capsys.readouterr().out.splitlines()[1].endswith("coreset_items | window_rel_l2 | window_ms | window_state")
    header, *lines = (tmp_path / "b.csv").read_text().splitlines()
    assert header == ",".join(bench_mod.COLUMNS + bench_mod.WINDOW_COLUMNS) and len(lines) == 2
    elem = 4 if dtype == "float32" else 2
    assert [r["window_state_bytes"] for r in rows] == [96 * 64 * elem, 103 * 64 * elem]
    # both round their outputs once (and 16-bit weights once more), the fp32 ones sum 96 products
    assert rows[0]["window_rel_l2"] <= (1e-5 if dtype == "float32" else 4 * 2.0 ** -8)
    assert rows[1]["window_rel_l2"] > rows[0]["window_rel_l2"] and rows[1]["window_best_ms"] > 0


def test_second_derivatives_are_refused():
    """A graph of the gradients may be asked for; a derivative of them is an error and not a silent zero."""
    q, k, v = (torch.randn(1, 2, 40, 32, device=DEV).requires_grad_() for _ in range(3))
    table = qkr.rotary_table(64, 32, device=DEV)
    for out in (swa.sink_window_causal_attention(q, k, v, window=8), qkr.qk_norm_rotary(q, k, table)[0]):
        plain = torch.autograd.grad(out.square().sum(), q, retain_graph=True)[0]
        dq = torch.autograd.grad(out.square().sum(), q, create_graph=True)[0]
        assert torch.equal(plain, dq)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            dq.sum().backward()


@pytest.mark.parametrize("storage", [None, "fp4"])
def test_two_captured_objects(storage):
    """Steps of two objects in graphs of their own, both with split queries, replayed in turn and on two streams at once."""
    g = torch.Generator().manual_seed(31)
    size = dict(streams=1, heads=4, kv_heads=1, window=3000, sinks=4, dtype=torch.bfloat16, storage=storage, device=DEV)
    objects, eager, graphs, inputs, outs = [], [], [], [], []
    for i in range(2):
        pair = [swa.SinkWindowStreamingAttention(64, 48, **size) for _ in range(2)]
        k, v = (torch.randn(1, 1, 2990, d, generator=g).bfloat16().to(DEV) for d in (64, 48))
        for a in pair:
            a.extend(k, v)
        x = [torch.zeros(1, h, d, dtype=torch.bfloat16, device=DEV) for h, d in ((4, 64), (1, 64), (1, 48))]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pair[0].step(*x))
        objects.append(pair[0])
        eager.append(pair[1])
        graphs.append(graph)
        inputs.append(x)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for n in range(20):
        for x in inputs:
            for t in x:
                t.copy_(torch.randn(t.shape, generator=g))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i if n % 2 else 0]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], eager[i].step(*inputs[i])), (n, i)
    for a, b in zip(objects, eager):
        for x, y in zip(a.items(), b.items()):
            assert torch.equal(x, y)


def test_calls_from_two_threads():
    """Forward and backward passes of two threads at once, each on a stream of its own, give what they give alone."""
    def inputs(i):
        g = torch.Generator().manual_seed(40 + i)
        return [torch.randn(2, 4, 300 + 77 * i, 64, generator=g).to(DEV, (torch.bfloat16, torch.float32)[i]) for _ in range(4)]

    table = qkr.rotary_table(512, 64, device=DEV)

    def work(q, k, v, go):
        q, k, v = (t.clone().requires_grad_() for t in (q, k, v))
        x, y = qkr.qk_norm_rotary(q, k, table)
        out = swa.sink_window_causal_attention(x, y, v, window=50)
        return [t.detach() for t in (out, *torch.autograd.grad(out, (q, k, v), go))]

    data = [inputs(i) for i in range(2)]
    alone = [work(*x) for x in data]
    torch.cuda.synchronize()
    results, failures = [[], []], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    results[i].append(work(*data[i]))
            stream.synchronize()
        except Exception as e:  # reported in the test's own thread
            failures.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    torch.cuda.synchronize()
    for i in range(2):
        assert len(results[i]) == 10
        for got in results[i]:
            for x, y in zip(got, alone[i]):
                assert torch.equal(x, y)


def test_lengths_outside_the_rows():
    """Lengths and counts outside 0 .. N are taken as the nearest of them."""
    g = torch.Generator().manual_seed(50)
    q, k, v, go = (torch.randn(3, 2, 150, 32, generator=g).to(DEV) for _ in range(4))
    far = torch.tensor([-7, 2 ** 31 - 1, 151], dtype=torch.int32, device=DEV)
    near = torch.tensor([0, 150, 150], dtype=torch.int32, device=DEV)
    got, want = [], []
    for lengths, to in ((far, got), (near, want)):
        out, lse = swa.sink_window_forward(q, k, v, window=20, sinks=2, lengths=lengths)
        to += [out, lse, *swa.sink_window_backward(go, q, k, v, out, lse, window=20, sinks=2, lengths=lengths)]
        a = swa.SinkWindowStreamingAttention(32, 32, streams=3, heads=2, window=20, sinks=2, device=DEV)
        to.append(a.prefill(q, k, v, counts=lengths))
        to += [a.lengths, *a.items(), a.step(q[:, :, 0], k[:, :, 0], v[:, :, 0])]
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert got[0][0].count_nonzero() == 0 and got[6].tolist() == [1, 151, 151]  # a view: the step counts
