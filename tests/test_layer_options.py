"""Layers with a layer norm, a window with sinks and rotary positions on several axes, through the partition engine and with both ends
of the model, and the end of the step: against plain autograd."""

import dataclasses

import pytest
import torch

from kareus_amd import GPTModelShard, LayerConfig, LayerStack, clip_grad_norm, grad_norm
from kareus_amd.partitions.partition_base import _build_overlap_slots
from kareus_amd.partitions.streams import use_stream_api
from kareus_amd.rotary_axes import axis_of_frequency
from kareus_amd.schedule_check import RecordingStreams

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]
OPTIONS = {"norm": dict(normalization="LayerNorm"), "window": dict(attention_window=19, attention_sinks=3),
           "axes": dict(rotary_sections=(8, 12, 12)), "in turn": dict(rotary_sections=(12, 10, 10), rotary_interleaved=True),
           "all": dict(normalization="LayerNorm", attention_window=19, attention_sinks=3, rotary_sections=(8, 12, 12)),
           "heads": dict(normalization="LayerNorm", attention_window=40, rotary_sections=(8, 12, 12), qk_layernorm=True)}


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def config(backend, dtype, n=1, layers=2, **kw):
    return LayerConfig(256, 4, 2, 64, 328, num_layers=layers, num_nanobatches=n, backend=backend, params_dtype=dtype, rotary_base=10000.0, **kw)


def stir(model):
    """Norm weights and biases other than ones and zeros."""
    gen = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if p.dim() == 1:
                p.add_((0.2 * torch.randn(p.shape, generator=gen)).to(p.device, p.dtype))
    return model


def positions(s, b, n, device):
    gen = torch.Generator().manual_seed(3)
    return torch.randint(0, 5000, (n, b, s), generator=gen).to(device)


def norm(x, op, c):
    if c.normalization == "LayerNorm":
        return torch.nn.functional.layer_norm(x, (x.shape[-1],), op.weight, op.bias, c.layernorm_epsilon)
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + c.layernorm_epsilon) * op.weight


def plain_layer(x, layer, c, at):
    """One layer in x's type by autograd; at: [axes, b, s], or None for the place in the sequence."""
    s, b, _ = x.shape
    ng, per, hd = c.num_query_groups, c.num_attention_heads // c.num_query_groups, c.kv_channels
    mixed = (norm(x, layer.input_layernorm, c) @ layer.linear_qkv.weight.t()).view(s, b, ng, per + 2, hd)
    q, k, v = mixed[:, :, :, :per], mixed[:, :, :, per:per + 1], mixed[:, :, :, per + 1:]
    if c.qk_layernorm:
        q, k = (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + c.layernorm_epsilon) * o.weight
                for t, o in ((q, layer.qkv_postprocess.q_layernorm), (k, layer.qkv_postprocess.k_layernorm)))
    inv = c.rotary_base ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=x.device) / hd)
    if c.rotary_sections is None:
        place = torch.arange(s, device=x.device).expand(hd // 2, b, s)
    else:
        place = at[axis_of_frequency(c.rotary_sections, c.rotary_interleaved, x.device)]
    angle = (place.double() * inv[:, None, None]).permute(2, 1, 0)[:, :, None, None]
    cos, sin = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
    turn = lambda t: torch.cat((t[..., :hd // 2] * cos - t[..., hd // 2:] * sin, t[..., hd // 2:] * cos + t[..., :hd // 2] * sin), -1)  # noqa: E731
    q, k = turn(q), turn(k)
    heads = lambda t: t.permute(1, 2, 3, 0, 4)   # noqa: E731  [b, ng, per or 1, s, hd]
    i = torch.arange(s, device=x.device)
    back = i[:, None] - i
    seen = back >= 0
    if c.attention_window:
        seen &= (back < c.attention_window) | (i < c.attention_sinks)
    p = (heads(q) @ heads(k).transpose(-1, -2) / hd ** 0.5).masked_fill(~seen, -torch.inf).softmax(-1)
    o = (p @ heads(v)).permute(3, 0, 1, 2, 4).reshape(s, b, ng * per * hd)
    x = x + o @ layer.linear_proj.weight.t()
    gate, up = (norm(x, layer.pre_mlp_layernorm, c) @ layer.linear_fc1.weight.t()).chunk(2, -1)
    return x + (torch.nn.functional.silu(gate) * up) @ layer.linear_fc2.weight.t()


def reference(model, x, dy, at):
    """Output, input gradient and parameter gradients of a stack in fp32 on the model's values."""
    twin = LayerStack(dataclasses.replace(model.config, backend="eager", params_dtype=torch.float32, num_nanobatches=1,
                                          nanobatch_streams=None, made_streams=None), device=x.device)
    twin.load_state_dict({n: t.float() for n, t in model.state_dict().items()})
    x = x.detach().float().requires_grad_(True)
    y = x
    for layer in twin.layers:
        y = plain_layer(y, layer, model.config, at)
    y.backward(dy.float())
    return y.detach(), x.grad, {n: p.grad for n, p in twin.named_parameters()}


def run(model, x, dy, at):
    for p in model.parameters():
        p.grad = None
    x = x.detach().clone().requires_grad_(True)
    y = model(x, position_ids=at)
    y.backward(dy)
    return y.detach(), x.grad, {n: p.grad for n, p in model.named_parameters()}


def near(got, want, tol):
    for name, a, b in (("y", got[0], want[0]), ("dx", got[1], want[1]), *[(n, got[2][n], want[2][n]) for n in want[2]]):
        assert a.shape == b.shape
        off = (a.float() - b.float()).abs().max() / b.float().abs().max()
        assert float(off) <= tol, (name, float(off))


@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("option", OPTIONS)
def test_the_eager_engine(option, n):
    """fp32 against fp32: what is left is the order of sums."""
    c = config("eager", torch.float32, n, **OPTIONS[option])
    model = stir(LayerStack(c, seed=1))
    gen = torch.Generator().manual_seed(5)
    x, dy = torch.randn(48, 2, 256, generator=gen), torch.randn(48, 2, 256, generator=gen)
    at = positions(48, 2, 3, "cpu") if c.rotary_sections else None
    near(run(model, x, dy, at), reference(model, x, dy, at), 2e-4)


def test_without_positions_every_axis_has_the_place_in_the_sequence():
    c = config("eager", torch.float32, 2, **OPTIONS["axes"])
    model = stir(LayerStack(c, seed=1))
    plain = LayerStack(config("eager", torch.float32, 2), seed=1)
    plain.load_state_dict(model.state_dict())
    x = torch.randn(40, 2, 256, generator=torch.Generator().manual_seed(5))
    with torch.no_grad():
        assert torch.allclose(model(x), plain(x), rtol=0, atol=1e-4)


def test_recomputation_and_streams_on_the_host():
    """Positions reach the recomputed forward pass, and the plan of streams has no violation."""
    rec = RecordingStreams()
    with use_stream_api(rec):
        c = config("eager", torch.float32, 2, checkpoint_activations=True, **OPTIONS["all"])
        model = stir(LayerStack(c, seed=1))
        gen = torch.Generator().manual_seed(5)
        x, dy = torch.randn(32, 4, 256, generator=gen), torch.randn(32, 4, 256, generator=gen)
        at = positions(32, 4, 3, "cpu")
        near(run(model, x, dy, at), reference(model, x, dy, at), 2e-4)
    assert not rec.violations


@pytest.mark.parametrize("again", [False, True])
def test_positions_that_change_before_the_backward_pass(again):
    """A buffer of positions that is filled for the next microbatch in between: refused, not turned by the wrong angles."""
    c = config("eager", torch.float32, 2, checkpoint_activations=again, **OPTIONS["axes"])
    model = stir(LayerStack(c, seed=1))
    gen = torch.Generator().manual_seed(5)
    x, dy = torch.randn(16, 2, 256, generator=gen), torch.randn(16, 2, 256, generator=gen)
    at = positions(16, 2, 3, "cpu")
    y = model(x.requires_grad_(True), position_ids=at)
    at.copy_(at + 1)
    with pytest.raises(RuntimeError, match="positions"):
        y.backward(dy)
    with torch.inference_mode():
        frozen = at.clone()
    near(run(model, x, dy, frozen), run(model, x, dy, at), 0.0)


def test_slots_and_refusals():
    c = config("eager", torch.float32, layers=1, **OPTIONS["all"])
    model = LayerStack(c, seed=1)
    plain = LayerStack(config("eager", torch.float32, layers=1), seed=1)
    for a, b in zip(model.forward_partitions + model.backward_partitions, plain.forward_partitions + plain.backward_partitions):
        assert _build_overlap_slots(a.comp_ops) == _build_overlap_slots(b.comp_ops)     # the schedules' names
    x = torch.randn(8, 2, 256)
    at = positions(8, 2, 3, "cpu")
    for bad in (at[:2], at[:, :1], at.int(), at[:, :, :4]):
        with pytest.raises(ValueError, match="position"):
            model(x, position_ids=bad)
    with pytest.raises(NotImplementedError):
        plain(x, position_ids=at)
    with pytest.raises(NotImplementedError):
        model(x, rotary_pos_emb=plain.rotary_pos_emb(8), position_ids=at)
    for kw in (dict(normalization="BatchNorm"), dict(attention_window=-1), dict(attention_sinks=4), dict(attention_window=4, attention_sinks=-1)):
        with pytest.raises(ValueError):
            LayerStack(config("eager", torch.float32, **kw))
    with pytest.raises(RuntimeError):
        LayerStack(config("eager", torch.float32, rotary_sections=(8, 8)))


def test_the_estimate_of_a_nanobatch_counts_what_its_window_leaves():
    whole, part = (config("hip", torch.bfloat16, 2, streams_are_own=True, in_line_below_ms=0.5, **kw) for kw in ({}, dict(attention_window=64)))
    assert not whole.nanobatches_in_line(16384, 1) and part.nanobatches_in_line(4096, 1)
    assert any(part.nanobatches_in_line(s, 1) and not whole.nanobatches_in_line(s, 1) for s in range(1024, 16384, 1024))


@on_gpu
@pytest.mark.parametrize("n,streams", [(1, False), (2, False), (2, True), (4, True)])
@pytest.mark.parametrize("option", OPTIONS)
def test_the_layers_on_the_device(option, n, streams):
    """bf16 results to 2e-2 of the largest, as the plain layers' are."""
    kw = dict(in_line_below_ms=0.0) if streams else {}
    c = config("hip", torch.bfloat16, n, **OPTIONS[option], **kw)
    model = stir(LayerStack(c, device="cuda", seed=1))
    gen = torch.Generator().manual_seed(5)
    x, dy = (torch.randn(200, 4, 256, generator=gen).to("cuda", torch.bfloat16) for _ in range(2))
    at = positions(200, 4, 3, "cuda") if c.rotary_sections else None
    near(run(model, x, dy, at), reference(model, x, dy, at), 2e-2)


@on_gpu
def test_recomputed_layers_on_the_device():
    gen = torch.Generator().manual_seed(5)
    x, dy = (torch.randn(132, 4, 256, generator=gen).to("cuda", torch.bfloat16) for _ in range(2))
    at = positions(132, 4, 3, "cuda")
    results = []
    for again in (False, True):
        model = stir(LayerStack(config("hip", torch.bfloat16, 2, checkpoint_activations=again, in_line_below_ms=0.0, **OPTIONS["all"]),
                                device="cuda", seed=1))
        results.append(run(model, x, dy, at))
    near(results[1], results[0], 1e-2)
    assert torch.equal(results[0][0], results[1][0])


def shard(backend, dtype, device, n=2, **kw):
    c = config(backend, dtype, n, **OPTIONS["all"])
    return stir(GPTModelShard(c, 512, device=device, seed=1, **kw))


def a_step(model, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ids, labels = (torch.randint(0, 512, (4, 40), generator=gen).to(device) for _ in range(2))
    loss = model(ids, labels, position_ids=positions(40, 4, 3, device)).mean()
    loss.backward()
    return loss


def test_a_step_on_the_host():
    """Embedding, layers, final norm, loss, backward and clipping; the embedding's gradient in fp32."""
    model = shard("eager", torch.float32, "cpu", embedding_main_grad=True)
    a_step(model, "cpu")
    assert model.embedding.weight.grad is None and model.final_layernorm_bias.grad is not None
    found = {n: (p.main_grad if n == "embedding.weight" else p.grad).clone() for n, p in model.named_parameters()}
    want = float(sum(g.double().square().sum() for g in found.values())) ** 0.5
    norm = model.clip_grad_norm(0.25 * want, eps=0.0)
    assert abs(float(norm) - want) <= 1e-6 * want
    for n, p in model.named_parameters():
        g = p.main_grad if n == "embedding.weight" else p.grad
        assert torch.allclose(g, 0.25 * found[n], rtol=1e-6, atol=0)
    assert abs(float(grad_norm(model.parameters(), backend="eager")) - 0.25 * want) <= 1e-5 * want


@on_gpu
def test_a_step_on_the_device():
    model = shard("hip", torch.bfloat16, "cuda", embedding_main_grad=True)
    twin = shard("eager", torch.float32, "cpu", embedding_main_grad=True)
    twin.load_state_dict({n: t.float().cpu() for n, t in model.state_dict().items()})
    loss, want = a_step(model, "cuda"), a_step(twin, "cpu")
    assert abs(float(loss.detach()) - float(want.detach())) <= 2e-2 * float(want.detach())
    norm = float(grad_norm(twin.parameters(), backend="eager"))
    before = [p.main_grad.clone() if n == "embedding.weight" else p.grad.clone() for n, p in model.named_parameters()]
    assert abs(float(model.clip_grad_norm(0.5 * norm)) - norm) <= 2e-2 * norm
    after = [p.main_grad if n == "embedding.weight" else p.grad for n, p in model.named_parameters()]
    exact = float(sum(g.double().square().sum() for g in before)) ** 0.5
    for a, b in zip(after, before):
        assert bool(((a.double() - b.double() * (0.5 * norm / (exact + 1e-6))).abs() <= 1.01 * 2.0 ** -8 * b.abs() + 1e-12).all())
    out = [torch.empty(g.shape, device="cuda") for g in after]
    clip_grad_norm(model.parameters(), 1e9, out=out)
    assert all(torch.equal(o, g.float()) for o, g in zip(out, after))


@on_gpu
def test_a_step_captured_and_replayed():
    """Forward, backward and clipping in a graph, beside eager steps of the same model."""
    model = shard("hip", torch.bfloat16, "cuda", n=1)
    gen = torch.Generator().manual_seed(0)
    ids, labels = (torch.randint(0, 512, (4, 40), generator=gen).to("cuda") for _ in range(2))
    at = positions(40, 4, 3, "cuda")

    def step():
        for p in model.parameters():
            p.grad = None
        loss = model(ids, labels, position_ids=at).mean()
        grads = torch.autograd.grad(loss, list(model.parameters()))
        for p, g in zip(model.parameters(), grads):
            p.grad = g
        return loss.detach(), model.clip_grad_norm(0.01), [p.grad for p in model.parameters()]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    for p in model.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, norm, grads = step()
    for seed in (1, 2, 3):
        gen = torch.Generator().manual_seed(seed)
        ids.copy_(torch.randint(0, 512, (4, 40), generator=gen).to("cuda"))
        at.copy_(torch.randint(0, 999, at.shape, generator=gen).to("cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = (loss.clone(), norm.clone(), [g.clone() for g in grads])
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and all(torch.equal(a, b) for a, b in zip(got[2], want[2]))


@pytest.mark.parametrize("sections,had", [((12, 10, 10), True), ((11, 11, 10), True), ((16, 16), True), ((32,), True), ((17, 15), True), ((8, 12, 12), False),
                                          ((2, 14, 16), False), ((15, 17), False), ((0, 16, 16), False)])
def test_sections_in_turn_are_what_the_axes_get(sections, had):
    """Dealt in turn an axis has at most every n-th frequency: a layer refuses sections that say more."""
    counts = torch.bincount(axis_of_frequency(sections, True), minlength=len(sections)).tolist()
    assert (counts == list(sections)) == had
    LayerStack(config("eager", torch.float32, layers=1, rotary_sections=sections))
    c = config("eager", torch.float32, layers=1, rotary_sections=sections, rotary_interleaved=True)
    if had:
        LayerStack(c)
    else:
        with pytest.raises(RuntimeError, match="in turn"):
            LayerStack(c)


def test_sections_are_looked_at_without_a_device():
    """Layers are made under any default device, whose tensors may hold no values."""
    with torch.device("meta"):
        LayerStack(config("eager", torch.float32, layers=1, rotary_sections=(12, 10, 10), rotary_interleaved=True))
        with pytest.raises(RuntimeError, match="in turn"):
            LayerStack(config("eager", torch.float32, layers=1, rotary_sections=(8, 12, 12), rotary_interleaved=True))
