"""Decoder layers and model shards over 8-bit blocks (LayerConfig.linear_format) and with the scaled, sorted embedding: the engine against
the same operators composed by hand, on one stream and on several, with recomputation and without gradients; refusals."""

import pytest
import torch

from kareus_amd import GPTModelShard, LanguageModelEmbedding, LayerConfig, LayerStack
from kareus_amd.backend import get_backend
from kareus_amd.operators import BlockColumnParallelLinearOp, BlockRowParallelLinearOp
from kareus_amd.partitions.op_context import OperationContext

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]
LINEARS = ("linear_qkv", "linear_proj", "linear_fc1", "linear_fc2")


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def config(backend, dtype, **kw):
    sizes = dict(hidden_size=256, num_attention_heads=4, num_query_groups=2, kv_channels=64, ffn_hidden_size=328)
    return LayerConfig(**{**sizes, **kw}, params_dtype=dtype, backend=backend, linear_format="fp8_blocks")


def batch(s, b, h, device, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(s, b, h, generator=g).to(device, dtype).requires_grad_(True), torch.randn(s, b, h, generator=g).to(device, dtype))


def step(model, x, go):
    for p in model.parameters():
        p.grad = None
    x.grad = None
    y = model(x)
    y.backward(go)
    return [y.detach(), x.grad] + [p.grad for p in model.parameters()]


# ---- one operator ----------------------------------------------------------------------------------
def check_operator(cls, device, dtype, backend):
    be = get_backend(backend)
    op = cls(264, 136, device=device, dtype=dtype, backend=backend)
    x, dy = batch(37, 3, 264, device, dtype)[0].detach(), batch(37, 3, 136, device, dtype, 5)[1]
    ctx = OperationContext()
    y, _ = op.fuser_forward([ctx], x, basic_op_extra_inputs=[()], basic_op_prev_ops=[None], basic_op_next_ops=[None], basic_op_kwargs=[{}])
    ctx.saved_tensors = ctx.to_save
    dx, [(dw,)], _ = op.fuser_backward([ctx], dy, basic_op_grad_extra_outputs=[()])
    q = be.quantize_blocks(x.view(-1, 264), True, True)
    w = be.quantize_blocks(op.weight.detach(), True, True, tiles=True)
    d = be.quantize_blocks(dy.view(-1, 136), True, True)
    assert torch.equal(y.view(-1, 136), be.block_matmul(q.by_row, w.by_row, dtype=dtype))
    assert torch.equal(dx.view(-1, 264), be.block_matmul(d.by_row, w.by_col, dtype=dtype))
    assert torch.equal(dw, be.block_matmul(d.by_col, q.by_col, dtype=dtype))
    with pytest.raises(ValueError, match="in_features"):
        op.fuser_forward([OperationContext()], dy, basic_op_extra_inputs=[()], basic_op_prev_ops=[None], basic_op_next_ops=[None],
                         basic_op_kwargs=[{}])
    # a frozen weight: no gradient, nothing saved for it
    op.weight.requires_grad_(False)
    ctx = OperationContext()
    op.fuser_forward([ctx], x, basic_op_extra_inputs=[()], basic_op_prev_ops=[None], basic_op_next_ops=[None], basic_op_kwargs=[{}])
    ctx.saved_tensors = ctx.to_save
    dx2, [(none,)], _ = op.fuser_backward([ctx], dy, basic_op_grad_extra_outputs=[()])
    assert none is None and ctx.saved_tensors[0] is None and torch.equal(dx2, dx)


@pytest.mark.parametrize("cls", [BlockColumnParallelLinearOp, BlockRowParallelLinearOp])
def test_eager_operator(cls):
    check_operator(cls, "cpu", torch.float32, "eager")


@pytest.mark.parametrize("cls", [BlockColumnParallelLinearOp, BlockRowParallelLinearOp])
@on_gpu
def test_operator(cls):
    check_operator(cls, "cuda", torch.bfloat16, "hip")


# ---- layers ----------------------------------------------------------------------------------------
def test_eager_nanobatches_and_recomputation():
    """Row blocks do not see how a batch is cut into nanobatches: outputs and input gradients are the whole batch's, up to the order of
    the eager products' fp32 sums (each off by at most 2^-24 of the magnitudes per term), which a rounding to 8 bits behind them can
    turn into one of its steps; weight gradients are those of the nanobatches' own columns."""
    x, go = batch(24, 4, 256, "cpu", torch.float32)
    whole = LayerStack(config("eager", torch.float32, num_nanobatches=1), seed=7)
    want = step(whole, x, go)
    for kw in (dict(num_nanobatches=1, checkpoint_activations=True), dict(num_nanobatches=2), dict(num_nanobatches=4, checkpoint_activations=True)):
        model = LayerStack(config("eager", torch.float32, **kw), seed=7)
        got = step(model, x, go)
        if kw["num_nanobatches"] == 1:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        else:
            for a, b in zip(got, want):
                # 1 in 32 values a step of 2^-3 off would be 2^-3 / sqrt(32) = 0.022 of the norm; weight gradients are of other column
                # blocks: two roundings of 2^-4 / sqrt(3) each in either product
                assert ((a - b).norm() / b.norm()).item() < 0.08
    with torch.no_grad():
        assert torch.equal(whole(x), want[0])




@pytest.mark.parametrize("sizes", [dict(), dict(hidden_size=512, num_attention_heads=8, num_query_groups=2, kv_channels=128, ffn_hidden_size=1376)])
@on_gpu
def test_layer_near_the_layer_in_fp32(sizes):
    """Against the same layer on the eager backend in fp32.  bf16 roundings between the operators (2^-9 relative, rms 2^-9 / sqrt(3)) move
    a value over a border between e4m3 values in at most one of 16 cases (the spacing is 2^-4 of the value at least), by 2^-3 of it at
    most: 2^-3 / sqrt(16) = 0.03 of the norm for each rounding to 8 bits, two in a product; through a layer whose branches add to the
    residual that stays under 0.1."""
    s, b = 200, 4
    x, go = batch(s, b, sizes.get("hidden_size", 256), "cuda", torch.bfloat16)
    model = LayerStack(config("hip", torch.bfloat16, num_nanobatches=1, **sizes), device="cuda", seed=7)
    got = step(model, x, go)
    ref = LayerStack(config("eager", torch.float32, num_nanobatches=1, **sizes), seed=7)
    ref.load_state_dict({k: v.float().cpu() for k, v in model.state_dict().items()})
    want = step(ref, x.detach().float().cpu().requires_grad_(True), go.float().cpu())
    for a, c in zip(got, want):
        assert ((a.float().cpu() - c).norm() / c.norm()).item() < 0.1


@on_gpu
def test_streams_in_line_and_recomputation_agree():
    """Two and four nanobatches on streams, in line, recomputed, in row runs: the same bits every way, and again."""
    s, b, h = 160, 4, 512
    sizes = dict(hidden_size=h, num_attention_heads=4, num_query_groups=2, kv_channels=128, ffn_hidden_size=712, num_layers=2)
    x, go = batch(s, b, h, "cuda", torch.bfloat16)
    one = step(LayerStack(config("hip", torch.bfloat16, num_nanobatches=1, **sizes), device="cuda", seed=7), x, go)
    for n in (2, 4):
        first = None
        for kw in (dict(in_line_below_ms=0.0), dict(), dict(use_streams=False), dict(in_line_below_ms=0.0, checkpoint_activations=True),
                   dict(checkpoint_activations=True)):
            model = LayerStack(config("hip", torch.bfloat16, num_nanobatches=n, **sizes, **kw), device="cuda", seed=7)
            for _ in range(2):
                got = step(model, x, go)
                torch.cuda.synchronize()
                if first is None:
                    first = [t.clone() for t in got]
                assert all(torch.equal(a, c) for a, c in zip(got, first)), (n, kw)
        # (row blocks do not see the nanobatches: the products in front of the attention are the whole batch's, bit for bit; whole layers
        # differ by the attention's order of sums, and weight gradients by their column blocks)
        for a, c in zip(first, one):
            assert ((a.float() - c.float()).norm() / c.float().norm()).item() < 0.08


@on_gpu
def test_layer_with_dropout_and_head_norms_trains():
    """The other options of a layer beside the format: gradients of every parameter, finite, and the same from the same seed."""
    sizes = dict(hidden_size=512, num_attention_heads=4, num_query_groups=2, kv_channels=128, ffn_hidden_size=768)
    x, go = batch(128, 2, 512, "cuda", torch.bfloat16)
    model = LayerStack(config("hip", torch.bfloat16, num_nanobatches=2, hidden_dropout=0.1, qk_layernorm=True, **sizes), device="cuda", seed=7)
    runs = []
    for _ in range(2):
        torch.manual_seed(5)
        runs.append([t.clone() for t in step(model, x, go)])
    assert all(t.isfinite().all() and t.any() for t in runs[0])
    assert all(torch.equal(a, c) for a, c in zip(*runs))
    with torch.no_grad():
        model.eval()
        assert model(x).isfinite().all()


@on_gpu
def test_one_stream_step_in_a_graph():
    s, b, h = 96, 2, 512
    sizes = dict(hidden_size=h, num_attention_heads=4, num_query_groups=2, kv_channels=128, ffn_hidden_size=768)
    model = LayerStack(config("hip", torch.bfloat16, num_nanobatches=1, **sizes), device="cuda", seed=7)
    sets = [batch(s, b, h, "cuda", torch.bfloat16, i) for i in range(3)]
    with torch.no_grad():
        want = [model(x).clone() for x, _ in sets]
        held = sets[0][0].detach().clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = model(held)
        for r in range(4):
            held.copy_(sets[r % 3][0])
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[r % 3])
            assert torch.equal(model(sets[0][0]), want[0])


@on_gpu
def test_forward_and_backward_in_a_graph():
    s, b, h = 96, 2, 512
    sizes = dict(hidden_size=h, num_attention_heads=4, num_query_groups=2, kv_channels=128, ffn_hidden_size=768)
    model = LayerStack(config("hip", torch.bfloat16, num_nanobatches=1, **sizes), device="cuda", seed=7)
    weights = list(model.parameters())
    sets = [batch(s, b, h, "cuda", torch.bfloat16, i) for i in range(3)]

    def step(x, go):
        return torch.autograd.grad(model(x), [x] + weights, go)

    want = [[t.clone() for t in step(x.detach().clone().requires_grad_(True), go)] for x, go in sets]
    held, held_go = sets[0][0].detach().clone().requires_grad_(True), sets[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held, held_go)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held, held_go)
    for r in range(4):
        with torch.no_grad():
            held.copy_(sets[r % 3][0])
            held_go.copy_(sets[r % 3][1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want[r % 3]))
        eager = step(sets[1][0].detach().clone().requires_grad_(True), sets[1][1])
        assert all(torch.equal(a, c) for a, c in zip(eager, want[1]))


@pytest.mark.parametrize("key,slot", [("fwd_attn", "attn_0"), ("fwd_mlp", "linear_0"), ("bwd_mlp", "linear_0"), ("bwd_attn", "attn_0")])
@on_gpu
def test_profiled_partitions(key, slot):
    """A partition alone, run twice on the same saved tensors."""
    from kareus_amd.profiling import PartitionTest

    cfg = config("hip", torch.bfloat16, hidden_size=512, num_attention_heads=4, num_query_groups=2, kv_channels=128, ffn_hidden_size=768)
    t = PartitionTest(key, cfg, 2, 128, device="cuda")
    for _ in range(2):
        grads = t.test_config((slot, "none"), (16, 1024))
        torch.cuda.synchronize()
        if key.startswith("bwd"):
            assert all(g is None or g.isfinite().all() for op in grads.values() for g in op)


# ---- model shards ------------------------------------------------------------------------------------
def shard(backend, dtype, device=None, **kw):
    return GPTModelShard(config(backend, dtype, num_nanobatches=2), vocab_rows=104, device=device, seed=11, **kw)


def ids_and_labels(device, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 104, (4, 40), generator=g)
    ids[:, -9:] = 3                                              # padding
    return ids.to(device), torch.randint(0, 104, (4, 40), generator=g).to(device)


def check_shard(backend, dtype, device):
    ids, labels = ids_and_labels(device)
    plain = shard(backend, dtype, device, embedding_scale=8.0)
    plain(ids, labels).mean().backward()
    whole = plain.embedding.weight.grad
    assert whole is not None and not whole[~torch.isin(torch.arange(104, device=device), ids)].any()
    kept = shard(backend, dtype, device, embedding_scale=8.0, embedding_main_grad=True)
    assert kept.embedding.weight.main_grad is None
    kept(ids, labels).mean().backward()
    main = kept.embedding.weight.main_grad
    assert kept.embedding.weight.grad is None and main.dtype == torch.float32 and torch.equal(main.to(dtype), whole)
    once = main.clone()
    kept(ids, labels).mean().backward()                          # a second microbatch of the same tokens: twice the sum, exactly
    assert kept.embedding.weight.main_grad is main and torch.equal(main, 2 * once)
    kept.embedding.weight.main_grad = None
    kept(ids, labels).mean().backward()
    assert torch.equal(kept.embedding.weight.main_grad, once)


def test_eager_shard():
    check_shard("eager", torch.float32, "cpu")


@on_gpu
def test_shard():
    check_shard("hip", torch.bfloat16, "cuda")


def check_embedding(backend, dtype, device):
    """The sorted gradient is the gradient of scale * rows: by the formula, and by a difference along one element."""
    cfg = config(backend, dtype)
    ids, _ = ids_and_labels(device)
    g = torch.Generator().manual_seed(2)
    go = torch.randn(40, 4, 256, generator=g).to(device, dtype)
    emb = LanguageModelEmbedding(cfg, 104, device=device, generator=torch.Generator().manual_seed(1), scale=4.0)
    emb(ids).backward(go)
    want = torch.zeros(104, 256, dtype=torch.float64, device=device).index_add_(0, ids.t().reshape(-1), go.reshape(-1, 256).double()) * 4.0
    eps = torch.finfo(dtype).eps / 2
    mags = torch.zeros(104, 256, dtype=torch.float64, device=device).index_add_(0, ids.t().reshape(-1), go.reshape(-1, 256).double().abs()) * 4.0
    assert ((emb.weight.grad.double() - want).abs() <= want.abs() * eps + mags * 64 * 2.0 ** -24).all()
    w = emb.weight.detach().double()
    moved = w.clone()
    moved[3, 17] += 0.5
    slope = ((4.0 * (moved - w))[ids.t()] * go.double()).sum() / 0.5
    assert abs(emb.weight.grad[3, 17].double() - slope) <= abs(slope) * eps + mags[3, 17] * 64 * 2.0 ** -24


def test_eager_embedding_gradient():
    check_embedding("eager", torch.float32, "cpu")


@on_gpu
def test_embedding_gradient():
    check_embedding("hip", torch.bfloat16, "cuda")


@on_gpu
def test_sorted_gradient_of_the_plain_embedding():
    """sorted_gradient alone: the lookup's bits, and a gradient within the roundings of the one by vocabulary rows."""
    cfg = config("hip", torch.bfloat16)
    ids, _ = ids_and_labels("cuda")
    go = torch.randn(40, 4, 256, generator=torch.Generator().manual_seed(2)).to("cuda", torch.bfloat16)
    outs, grads = [], []
    for kw in (dict(), dict(sorted_gradient=True)):
        emb = LanguageModelEmbedding(cfg, 104, device="cuda", generator=torch.Generator().manual_seed(1), **kw)
        out = emb(ids)
        out.backward(go)
        outs.append(out.detach())
        grads.append(emb.weight.grad.double())
    assert torch.equal(*outs)
    # (two roundings to bf16 of fp32 sums: a step of 2^-7 at most, and the sums' own 64 * 2^-24 of the magnitudes)
    assert ((grads[0] - grads[1]).abs() <= grads[0].abs() * 2.0 ** -7 + 64 * 64 * 2.0 ** -24).all()


def test_refusals():
    with pytest.raises(ValueError, match="linear_format"):
        LayerStack(LayerConfig(256, 4, 2, 64, 328, backend="eager", params_dtype=torch.float32, linear_format="fp8"))


def test_slots_of_a_schedule_are_those_of_the_bf16_layer():
    from kareus_amd.partitions.partition_base import _build_overlap_slots  # noqa: F401
    plain = LayerStack(LayerConfig(256, 4, 2, 64, 328, backend="eager", params_dtype=torch.float32, fuse_forward_epilogues=False))
    blocks = LayerStack(config("eager", torch.float32))
    for a, b in zip(plain.forward_partitions + plain.backward_partitions, blocks.forward_partitions + blocks.backward_partitions):
        assert a._overlap_slots == b._overlap_slots
