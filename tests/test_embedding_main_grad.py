"""``weight.main_grad`` over passes on several streams: sums one behind the other, and the caller behind them, as autograd orders the
gradients that it accumulates itself."""

import copy
import pickle

import pytest
import torch

from kareus_amd import LanguageModelEmbedding, LayerConfig
from kareus_amd.partitions.streams import use_stream_api
from kareus_amd.schedule_check import RecordingStreams

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def embedding(backend, dtype, device, rows=1000, hidden=256):
    cfg = LayerConfig(hidden, 4, 2, 64, 328, backend=backend, params_dtype=dtype)
    return LanguageModelEmbedding(cfg, rows, device=device, generator=torch.Generator().manual_seed(1), main_grad=True)


def ids(seed, device, rows=1000):
    return torch.randint(0, rows, (2, 50), generator=torch.Generator().manual_seed(seed)).to(device)


class OnStream(torch.autograd.Function):
    """The backward pass goes on on another stream from here, as autograd does where the forward pass ran there."""

    @staticmethod
    def forward(ctx, x, rec, stream):
        ctx.rec, ctx.stream = rec, stream
        return x.clone()

    @staticmethod
    def backward(ctx, dy):
        ctx.rec._current[-1] = ctx.stream
        return dy, None, None


def test_sums_of_one_pass_and_the_caller_are_in_order():
    rec = RecordingStreams()
    with use_stream_api(rec):
        caller, a, b = rec.current_stream(), rec.new_stream(), rec.new_stream()
        emb = embedding("eager", torch.float32, "cpu")
        loss = OnStream.apply(emb(ids(1, "cpu")), rec, a).sum() + OnStream.apply(emb(ids(2, "cpu")), rec, b).sum()
        rec.edges.clear()
        order = []
        loss.register_hook(lambda g: order.append(rec._current[-1]) or torch.autograd.Variable._execution_engine.queue_callback(
            lambda: rec._current.__setitem__(-1, caller)))
        loss.backward()
    assert order == [caller] and not rec.violations
    waits = [(x[0], y[0]) for x, y in rec.edges]
    assert (a.sid, b.sid) in waits or (b.sid, a.sid) in waits        # the second sum behind the first
    assert (a.sid, caller.sid) in waits and (b.sid, caller.sid) in waits


def test_sums_of_passes_on_two_streams_are_in_order():
    rec = RecordingStreams()
    with use_stream_api(rec):
        a, b = rec.new_stream(), rec.new_stream()
        emb = embedding("eager", torch.float32, "cpu")
        for s in (a, b, b, a):
            with rec.stream(s):
                emb(ids(1, "cpu")).sum().backward()
    assert not rec.violations
    assert [(x[0], y[0]) for x, y in rec.edges] == [(a.sid, b.sid), (b.sid, a.sid)]


def test_modules_are_copied_and_saved_between_passes():
    emb = embedding("eager", torch.float32, "cpu")
    emb(ids(1, "cpu")).sum().backward()
    for other in (copy.deepcopy(emb), pickle.loads(pickle.dumps(emb))):
        other.weight.main_grad = None
        other(ids(1, "cpu")).sum().backward()
        assert torch.equal(other.weight.main_grad, emb.weight.main_grad)


@on_gpu
def test_passes_on_streams_with_work_in_front():
    """Forward passes on three streams, each backward behind work of its own length: read at once on the caller's stream, several times."""
    emb = embedding("hip", torch.bfloat16, "cuda", rows=32000, hidden=1024)
    sets = [torch.randint(0, 32000, (2, 2000), generator=torch.Generator().manual_seed(i)).cuda() for i in range(3)]
    grads = [torch.randn(2000, 2, 1024, generator=torch.Generator().manual_seed(9 + i)).bfloat16().cuda() for i in range(3)]

    class Late(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, cycles):
            ctx.cycles = cycles
            return x.clone()

        @staticmethod
        def backward(ctx, dy):
            torch.cuda._sleep(ctx.cycles)
            return dy, None

    def total(streams):
        emb.weight.main_grad = None
        outs = []
        for i, (s, x) in enumerate(zip(streams, sets)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(Late.apply(emb(x), 400000 * (3 - i)))
        torch.autograd.backward(outs, grads)
        return emb.weight.main_grad.clone()

    caller = torch.cuda.current_stream()
    want = total([caller] * 3)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        got = total(streams)
        # (the order of the three sums is the engine's: fp32 sums of three terms each way)
        assert torch.allclose(got, want, rtol=0, atol=3 * 2.0 ** -24 * 3 * want.abs().max().item() * 4)
        torch.cuda.synchronize()


@on_gpu
def test_a_pass_in_a_graph_behind_eager_ones_on_another_stream():
    emb = embedding("hip", torch.bfloat16, "cuda")
    x, go = ids(1, "cuda"), torch.randn(50, 2, 256, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        emb(x).backward(go)
    torch.cuda.synchronize()
    once = emb.weight.main_grad.clone()
    emb.weight.main_grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        emb(x).backward(go)
    main = emb.weight.main_grad
    for r in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(main, (r + 1) * once) or torch.allclose(main, (r + 1) * once, rtol=4 * 2.0 ** -24, atol=0)
    with torch.cuda.stream(side):
        emb(x).backward(go)
    torch.cuda.synchronize()
    assert torch.allclose(main, 5 * once, rtol=5 * 2.0 ** -24, atol=0)
