"""The weight gradient of an 8-bit layer over several nanobatches: one sum over all their tokens, rounded once, launched where the bf16 layers
launch theirs; and the product over pairs of operands that it runs on."""

import ctypes

import pytest
import torch

from kareus_amd import BlockOperand, LayerConfig, LayerStack
from kareus_amd.backend import get_backend, reserve_compute_units
from kareus_amd.block_scaled import blocks_of
from kareus_amd.operators import BlockColumnParallelLinearOp
from kareus_amd.partitions.op_context import OperationContext
from kareus_amd.partitions.streams import use_stream_api
from kareus_amd.schedule_check import RecordingStreams

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


# ---- one layer, several nanobatches -------------------------------------------------------------------
def gradients_over(op, be, device, n, seed, **sink):
    """(what the nanobatches' backward passes return as dW, the operands of each product)."""
    g = torch.Generator().manual_seed(seed)
    n_out, n_in = op.weight.shape
    shared, got, operands = dict(n=n, turn=[0], defer=True, pending=None, in_line=True, **sink), [], []
    for i in range(n):
        t = 40 + 13 * i
        x, dy = (torch.randn(t, 1, w, generator=g).to(device, torch.bfloat16) for w in (n_in, n_out))
        ctx = OperationContext()
        op.fuser_forward([ctx], x, basic_op_extra_inputs=[()], basic_op_prev_ops=[None], basic_op_next_ops=[None], basic_op_kwargs=[{}])
        ctx.saved_tensors, ctx.wgrad_sink, ctx.nanobatch_index, ctx.alone = ctx.to_save, shared, i, True
        _, [(dw,)], _ = op.fuser_backward([ctx], dy, basic_op_grad_extra_outputs=[()])
        got.append(dw)
        operands.append((be.quantize_blocks(dy.view(t, n_out), False, True).by_col, be.quantize_blocks(x.view(t, n_in), False, True).by_col))
        for held in ctx.saved_tensors:          # (as the engine does)
            if held is not None:
                held.data = held.new_empty(0)
    return got, operands


def stands_for(t):
    """What an operand stands for, in 64 bits."""
    nb = blocks_of(t.length)
    e = torch.exp2(t.scales[:nb, :t.rows].t().double() - 127)
    return (t.data[:, :nb * 128].double().view(t.rows, nb, 128) * e[..., None]).view(t.rows, -1)[:, :t.length]


@pytest.mark.parametrize("n", [2, 4])
def test_eager_gradient_is_rounded_once(n):
    be = get_backend("eager")
    op = BlockColumnParallelLinearOp(136, 72, device="cpu", dtype=torch.bfloat16, backend="eager")
    got, operands = gradients_over(op, be, "cpu", n, 3)
    assert [dw is None for dw in got] == [True] * (n - 1) + [False]
    assert torch.equal(got[-1], sum(be.block_matmul(*o, dtype=torch.float32) for o in operands).bfloat16())


def product_bound(want, mags, steps):
    """test_block_scaled.py's: half a bf16 step, the groups' cut, and the fp32 sums of `steps` halves of a block and 16 cuts."""
    return want.abs() * 2.0 ** -8 + mags * (7 * 2.0 ** -13 + steps * 9 * 2.0 ** -23 + 16 * 2.0 ** -24)


@pytest.mark.parametrize("n", [2, 4, 18])
@on_gpu
def test_gradient_over_nanobatches(n):
    """Within the bound of one sum, and rounded once.  A sum off by d falls to another bf16 neighbour with the probability |d| / u (u: a
    step, 2^-8 to 2^-7 of the value).  The matrix unit's cuts are off by less than 2^-13 of a group's largest product each, with either
    sign: in the norm at most 2^-13 / sqrt(3) * 2 = 1.4e-4 of the sum's, |d| / u below 0.03.  A part that was rounded by itself is off by
    u' / 4 on average, u' its own step, u / 2 and more where it is half the sum: 0.12 and more."""
    be = get_backend("hip")
    op = BlockColumnParallelLinearOp(520, 264, device="cuda", dtype=torch.bfloat16, backend="hip")
    got, operands = gradients_over(op, be, "cuda", n, 3)
    assert [dw is None for dw in got] == [True] * (n - 1) + [False]
    pairs = [(stands_for(d).contiguous(), stands_for(x).t().contiguous()) for d, x in operands]
    want, mags = sum(d @ x for d, x in pairs), sum(d.abs() @ x.abs() for d, x in pairs)
    err = (got[-1].double() - want).abs()
    assert (err <= product_bound(want, mags, 2 * sum(blocks_of(d.length) for d, _ in operands))).all()
    assert (got[-1] != want.float().bfloat16()).double().mean().item() < 0.05


def config(backend, dtype, **kw):
    sizes = dict(hidden_size=256, num_attention_heads=4, num_query_groups=2, kv_channels=64, ffn_hidden_size=328)
    return LayerConfig(**{**sizes, **kw}, params_dtype=dtype, backend=backend, linear_format="fp8_blocks")


def record(be, monkeypatch):
    """Calls of the product over pairs, and of the accumulating one, as the layers make them."""
    calls = {"pairs": [], "added": 0}
    whole, one = be.block_matmul_segments, be.block_matmul

    def segments(a, b, out=None, **kw):
        got = whole(a, b, out=out, **kw)
        calls["pairs"].append(([(x, y) for x, y in zip(a, b)], got))
        return got

    def single(a, b, out=None, accumulate=False, **kw):
        calls["added"] += bool(accumulate)
        return one(a, b, out=out, accumulate=accumulate, **kw)

    monkeypatch.setattr(be, "block_matmul_segments", segments, raising=False)
    monkeypatch.setattr(be, "block_matmul", single, raising=False)
    return calls


@pytest.mark.parametrize("kw,launches,added", [(dict(), 4, 0), (dict(wgrad_launches_at_end=True), 4, 0),
                                               (dict(wgrad_over_all_nanobatches=False), 0, 4)])
def test_one_product_per_layer_and_pass(monkeypatch, kw, launches, added):
    """Two nanobatches of a layer's four weights: a launch each, or as the configuration asks."""
    calls = record(get_backend("eager"), monkeypatch)
    model = LayerStack(config("eager", torch.float32, num_nanobatches=2, **kw), seed=7)
    x = torch.randn(24, 4, 256, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
    model(x).sum().backward()
    assert len(calls["pairs"]) == launches and calls["added"] == added
    assert all(len(pairs) == 2 for pairs, _ in calls["pairs"])


@pytest.mark.parametrize("at_end", [True, False])
def test_nanobatches_wait_for_each_other_as_the_bf16_layers_do(at_end):
    """On streams: a backward pass has the waits between the nanobatches' streams that the bf16 layer has, none for sums of its own."""
    waits = []
    for form in ("bf16", "fp8_blocks"):
        rec = RecordingStreams()
        with use_stream_api(rec):
            cfg = config("eager", torch.float32, num_nanobatches=2, wgrad_launches_at_end=at_end, fuse_forward_epilogues=False)
            cfg.linear_format = form
            cfg.nanobatch_streams = [rec.new_stream(), rec.new_stream()]
            model = LayerStack(cfg, seed=7)
            x = torch.randn(24, 4, 256, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
            y = model(x).sum()
            rec.edges.clear()
            y.backward()
        assert not rec.violations
        sids = [s.sid for s in cfg.nanobatch_streams]
        waits.append([(sids.index(a[0]), sids.index(b[0])) for a, b in rec.edges if a[0] in sids and b[0] in sids and a[0] != b[0]])
    assert waits[0] == waits[1] and waits[0]


@pytest.mark.parametrize("kw", [dict(in_line_below_ms=0.0), dict(), dict(wgrad_launches_at_end=True, in_line_below_ms=0.0),
                                dict(checkpoint_activations=True, in_line_below_ms=0.0)])
@pytest.mark.parametrize("n", [2, 4])
@on_gpu
def test_layers_gradient_over_nanobatches(monkeypatch, n, kw):
    """What autograd gets is the product over all nanobatches, on streams and in line."""
    calls = record(get_backend("hip"), monkeypatch)
    model = LayerStack(config("hip", torch.bfloat16, hidden_size=512, num_attention_heads=4, kv_channels=128, ffn_hidden_size=712,
                              num_nanobatches=n, **kw), device="cuda", seed=7)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(160, 4, 512, generator=g).to("cuda", torch.bfloat16).requires_grad_(True)
    model(x).backward(torch.randn(160, 4, 512, generator=g).to("cuda", torch.bfloat16))
    torch.cuda.synchronize()
    assert len(calls["pairs"]) == 4 and not calls["added"]
    kept = {id(p.grad.untyped_storage()) for p in model.parameters()}
    assert len(kept) == len(list(model.parameters()))
    grads = [p.grad for name, p in model.named_parameters() if "linear" in name]
    for pairs, got in calls["pairs"]:
        assert len(pairs) == n
        parts = [(stands_for(d).contiguous(), stands_for(v).t().contiguous()) for d, v in pairs]
        want, mags = sum(d @ v for d, v in parts), sum(d.abs() @ v.abs() for d, v in parts)
        assert ((got.double() - want).abs() <= product_bound(want, mags, 2 * sum(blocks_of(d.length) for d, _ in pairs))).all()
        assert any(g.shape == got.shape and torch.equal(g, got) for g in grads)


# ---- the product over pairs ------------------------------------------------------------------------------
def whole_operand(rows, k, seed, device, pitch=0):
    """(operand of -1, 0 and 1 with scales from 2^-2 to 2^2, what it stands for in 64 bits)."""
    g = torch.Generator(device=device).manual_seed(seed)
    nb = blocks_of(k)
    v = torch.zeros(rows, nb * 128 + pitch, device=device)
    v[:, :k] = torch.randint(-1, 2, (rows, k), generator=g, device=device).float()
    v[:, nb * 128:] = float("nan")
    scales = torch.randint(125, 130, (nb, (rows + 3) // 4 * 4 + pitch), generator=g, device=device, dtype=torch.uint8)
    e = torch.exp2(scales[:, :rows].t().double() - 127)
    stands = (v[:, :nb * 128].double().view(rows, nb, 128) * e[..., None]).view(rows, -1)[:, :k]
    return BlockOperand(v.to(torch.float8_e4m3fn), scales, k), stands.contiguous()


def check_segments(be, device, m, n, lengths, out=None, dtype=torch.bfloat16):
    """Exact but for the store: see test_block_exact.py."""
    a, b, want, most = [], [], 0.0, 0.0
    for i, k in enumerate(lengths):
        (x, xv), (y, yv) = whole_operand(m, k, 2 * i, device, 16 * (i % 3)), whole_operand(n, k, 2 * i + 1, device, 32 * (i % 2))
        a.append(x)
        b.append(y)
        want, most = want + xv @ yv.t(), most + xv.abs() @ yv.abs().t()
    assert most.max() < 2.0 ** 20
    got = be.block_matmul_segments(a, b, out=out)
    assert got.dtype == dtype and torch.equal(got, want.float().to(dtype)) and (out is None or got is out)
    return a, b, got


LENGTHS = [(1,), (130, 1, 300), (128, 128, 128, 128), (257, 640, 5), tuple(range(1, 32, 2)), tuple(range(60, 77)), (40,) * 40]


@pytest.mark.parametrize("lengths", LENGTHS)
def test_eager_segments(lengths):
    check_segments(get_backend("eager"), "cpu", 33, 40, lengths)


# (the larger ones by the planner on 256 units: 256 x 256 whole and cut, 192 x 256, 256 x 128, 128 x 256, 128 x 128 whole and cut, 64 x 64 cut)
@pytest.mark.parametrize("m,n,lengths", [(m, n, k) for k in LENGTHS for m, n in ((1, 8), (33, 40), (130, 264))] + [
    (5745, 2184, (100, 161)), (401, 5552, (5000, 10129)), (1848, 5184, (129, 257)), (523, 4672, (4000, 903, 6000)), (5737, 1352, (435, 436)),
    (133, 3096, (7000, 7755)), (2960, 1368, (199,) * 4), (147, 5448, (2716, 3000)), (1753, 1776, (1, 258)), (66, 4368, (2940, 2940)),
    (4352, 4096, (300, 724)), (5000, 6144, (8, 128)), (1536, 2048, (3011, 3012))])
@on_gpu
def test_segments(m, n, lengths):
    check_segments(get_backend("hip"), "cuda", m, n, lengths)


@on_gpu
def test_segments_into_a_part_of_a_larger_matrix_and_on_fewer_units():
    be = get_backend("hip")
    whole = torch.full((300, 400), 7.0, dtype=torch.bfloat16, device="cuda")
    a, b, got = check_segments(be, "cuda", 130, 264, (300, 17, 256), out=whole[10:140, 16:280])
    rest = whole.clone()
    rest[10:140, 16:280] = 7.0
    assert (rest == 7.0).all()
    for reserved in (32, 200, 248):
        with reserve_compute_units(reserved):
            check_segments(be, "cuda", 130, 264, (300, 17, 256))
            check_segments(be, "cuda", 1536, 2048, (3011, 3012))
    # operands in tuples take the general path, with the same bits
    assert torch.equal(be.block_matmul_segments(tuple(a), tuple(b)), got)
    # a pair without tokens adds nothing, none but such pairs gives zeros
    empty = [BlockOperand(t.data[:, :0], t.scales[:0], 0) for t in (a[0], b[0])]
    assert torch.equal(be.block_matmul_segments(a + empty[:1], b + empty[1:]), got)
    assert not be.block_matmul_segments(empty[:1], empty[1:]).any()


@on_gpu
def test_segments_on_another_stream_and_in_a_graph():
    be = get_backend("hip")
    m, n, lengths = 264, 520, (300, 1000)
    sets = [[[whole_operand(rows, k, 10 * s + j + i, "cuda")[0] for j, k in enumerate(lengths)] for i, rows in ((0, m), (5, n))] for s in range(3)]
    want = [be.block_matmul_segments(*x).clone() for x in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = be.block_matmul_segments(*sets[1])
    side.synchronize()
    assert torch.equal(got, want[1])
    held = [[t._replace(data=t.data.clone(), scales=t.scales.clone()) for t in ops] for ops in sets[0]]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = be.block_matmul_segments(*held)
    for r in range(4):
        for mine, theirs in zip(held, sets[r % 3]):
            for t, u in zip(mine, theirs):
                t.data.view(torch.uint8).copy_(u.data.view(torch.uint8))
                t.scales.copy_(u.scales)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[r % 3]) and torch.equal(be.block_matmul_segments(*sets[1]), want[1])


# ---- refusals -----------------------------------------------------------------------------------------
def test_library_refuses_segments_before_anything_is_launched():
    from kareus_amd.backend import hip

    lib = hip.load_library()

    def call(m=4, n=8, nseg=2, k=(128, 5), a=(16, 32), lda=(128, 144), sa=(4, 8), lsa=(4, 8), b=(16, 16), ldb=(128, 128), sb=(4, 4), lsb=(8, 8),
             c=16, ldc=8, ws=None):
        args = []
        for v, kind in ((k, ctypes.c_int), (a, ctypes.c_void_p), (lda, ctypes.c_int64), (sa, ctypes.c_void_p), (lsa, ctypes.c_int64),
                        (b, ctypes.c_void_p), (ldb, ctypes.c_int64), (sb, ctypes.c_void_p), (lsb, ctypes.c_int64)):
            args.append(None if v is None else (kind * len(v))(*v))
        return lib.kr_block_gemm_segments(m, n, nseg, *args, c, ldc, 0, ws, 0, None)

    for kw, rc in ((dict(m=0), -1), (dict(n=0), -1), (dict(n=12), -2), (dict(nseg=0), -1), (dict(nseg=17), -2), (dict(k=None), -1),
                   (dict(k=(128, 0)), -1), (dict(k=(128, 129)), -1), (dict(a=(16, None)), -1), (dict(a=(16, 40)), -1), (dict(lda=(128, 112)), -1),
                   (dict(lda=(136, 128)), -2), (dict(lda=(128, 1 << 24)), -2), (dict(sa=(4, None)), -1), (dict(sa=(4, 6)), -1),
                   (dict(lsa=(4, 0)), -1), (dict(lsa=(4, 6)), -2), (dict(b=(None, 16)), -1), (dict(lsb=(4, 8)), -1), (dict(c=None), -1),
                   (dict(c=24), -1), (dict(ldc=0), -1), (dict(ldc=12), -2), (dict(ws=8), -1)):
        assert call(**kw) == rc, kw
    assert lib.kr_block_gemm_segments_workspace_bytes(0, 8, 8, 0) == 0
    assert lib.kr_block_gemm_segments_workspace_bytes(8, 8, 1 << 30, 0) == 0


def test_backend_refuses_segments():
    be = get_backend("hip")
    good = get_backend("eager").quantize_blocks(torch.zeros(4, 128)).by_row
    with pytest.raises(RuntimeError, match="HIP device"):
        be.block_matmul_segments([good], [good])
    with pytest.raises(RuntimeError, match="operands"):
        be.block_matmul_segments([good], [good, good])
    with pytest.raises(RuntimeError, match="operands"):
        be.block_matmul_segments([], [])
    with pytest.raises(RuntimeError, match="bf16"):
        be.block_matmul_segments([good], [good], dtype=torch.float32)
    for pair in (([good], []), ([], [])):
        with pytest.raises(RuntimeError, match="operands"):
            get_backend("eager").block_matmul_segments(*pair)


@on_gpu
def test_backend_refuses_segments_on_the_device():
    be = get_backend("hip")
    a, b = whole_operand(16, 200, 1, "cuda")[0], whole_operand(24, 200, 2, "cuda")[0]
    with pytest.raises(RuntimeError, match="contractions"):
        be.block_matmul_segments([a], [b._replace(length=199)])
    with pytest.raises(RuntimeError, match="rows behind"):
        be.block_matmul_segments([a, a], [b, a])
    with pytest.raises(RuntimeError, match="out must be"):
        be.block_matmul_segments([a], [b], out=torch.empty(16, 16, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="scales"):
        be.block_matmul_segments([a], [b._replace(scales=b.scales[:1])])
    with pytest.raises(RuntimeError, match="kr_block_gemm_segments"):      # four columns: not a multiple of 8
        be.block_matmul_segments([b], [whole_operand(4, 200, 3, "cuda")[0]])


# ---- a weight's blocks while a pass runs ----------------------------------------------------------------
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("n,kw", [(1, dict()), (2, dict()), (4, dict()), (2, dict(checkpoint_activations=True)), (1, dict(checkpoint_activations=True))])
def test_a_weights_rows_are_dropped_behind_its_last_nanobatch(monkeypatch, n, kw, grad):
    """Six layers: at no time are the rows' orientations of more than two layers' four weights alive (nanobatches run less than a layer
    apart), forward, recomputed and without gradients, and each weight is quantised once a pass."""
    import weakref

    be = get_backend("eager")
    made, alive, passes = [], [], []
    whole = be.quantize_blocks

    def quantise(x, by_row=True, by_col=False, tiles=False):
        got = whole(x, by_row, by_col, tiles)
        if tiles:
            made.append(weakref.ref(got.by_row.data))
            alive.append(sum(r() is not None for r in made))
        return got

    monkeypatch.setattr(be, "quantize_blocks", quantise, raising=False)
    model = LayerStack(config("eager", torch.float32, num_layers=6, num_nanobatches=n, **kw), seed=7)
    x = torch.randn(8, 4, 256, generator=torch.Generator().manual_seed(1)).requires_grad_(grad)
    with torch.set_grad_enabled(grad):
        y = model(x)
        passes.append(len(made))
        assert all(r() is None for r in made)
        if grad:
            y.sum().backward()
            passes.append(len(made))
    assert passes == [24] + ([48 if kw else 24] if grad else [])
    assert max(alive) <= (1 if n == 1 else 8)


# ---- streams or one behind the other ----------------------------------------------------------------------
@pytest.mark.parametrize("h,nq,nkv,hd,ffn,seq,seqs,bf16,blocks", [
    (2048, 32, 8, 64, 8192, 2048, 2, False, True), (2048, 32, 8, 64, 8192, 2048, 1, False, True), (2048, 2, 1, 128, 768, 4096, 4, False, True),
    (2048, 2, 1, 128, 768, 4096, 2, False, True), (4096, 8, 2, 128, 3584, 4096, 1, False, False), (4096, 8, 2, 128, 3584, 4096, 2, False, False),
    (4096, 32, 8, 128, 14336, 8192, 1, False, False), (512, 8, 8, 64, 1376, 128, 1, True, True)])
def test_small_nanobatches_of_8_bit_layers_run_in_line(h, nq, nkv, hd, ffn, seq, seqs, bf16, blocks):
    """By what was faster, measured: an 8-bit layer's nanobatch needs less of the device and more of the host than a bf16 layer's."""
    for form, want in (("bf16", bf16), ("fp8_blocks", blocks)):
        cfg = LayerConfig(h, nq, nkv, hd, ffn, linear_format=form, streams_are_own=True)
        assert cfg.nanobatches_in_line(seq, seqs) is want
        cfg.in_line_below_ms = 0.0
        assert cfg.nanobatches_in_line(seq, seqs) is False


@on_gpu
def test_two_nanobatches_forward_and_backward_in_a_graph():
    sizes = dict(hidden_size=512, num_attention_heads=4, num_query_groups=2, kv_channels=128, ffn_hidden_size=768)
    model = LayerStack(config("hip", torch.bfloat16, num_nanobatches=2, num_layers=2, **sizes), device="cuda", seed=7)
    weights = list(model.parameters())
    g = torch.Generator().manual_seed(1)
    sets = [[torch.randn(96, 2, 512, generator=g).to("cuda", torch.bfloat16) for _ in range(2)] for _ in range(3)]

    def step(x, go):
        return torch.autograd.grad(model(x), [x] + weights, go)

    want = [[t.clone() for t in step(x.clone().requires_grad_(True), go)] for x, go in sets]
    held, held_go = sets[0][0].clone().requires_grad_(True), sets[0][1].clone()
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
        eager = step(sets[1][0].clone().requires_grad_(True), sets[1][1])
        assert all(torch.equal(a, c) for a, c in zip(eager, want[1]))
