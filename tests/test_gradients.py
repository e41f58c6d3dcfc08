"""The global gradient norm and clipping against 64 bits.

Bounds.  Squares are exact in 64 bits and so, to some 2^-50, is their sum: the norm is one fp32 rounding off, 2^-24 of it, and the
factor another; a scaled gradient has the factor's rounding and its own: 2^-23 in fp32, 2^-8 + 2^-23 where it is rounded to bf16."""

import pytest
import torch

from kareus_amd import clip_grad_norm, grad_norm
from kareus_amd.backend import get_backend, hip

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]
U = 2.0 ** -24


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def make(sizes, size=1.0, device="cuda", seed=0):
    """Gradients of the given numbers of elements, fp32 where the number is negative."""
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(abs(n), generator=gen) * size).to(device, torch.float32 if n < 0 else torch.bfloat16) for n in sizes]


def true_norm(grads):
    return float(sum((g.double() ** 2).sum().cpu() for g in grads)) ** 0.5


def check(grads, max_norm=1.0, eps=1e-6):
    be = get_backend("hip")
    want = true_norm(grads)
    assert abs(float(be.grad_norm(grads)) - want) <= 1.01 * U * want
    factor = min(1.0, max_norm / (want + eps))
    before = [g.clone() for g in grads]
    out = [torch.full(g.shape, 9.0, device="cuda") for g in grads]
    norm = be.clip_grad_norm(grads, max_norm, eps, out=out)
    assert abs(float(norm) - want) <= 1.01 * U * want and norm.dtype == torch.float32 and norm.dim() == 0
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    for g, o in zip(before, out):
        exact = g.double() * factor
        assert bool(((o.double() - exact).abs() <= 2.02 * U * exact.abs() + 2.0 ** -149).all())
    be.clip_grad_norm(grads, max_norm, eps)
    for g, b, o in zip(grads, before, out):
        if factor == 1.0:
            assert torch.equal(g, b)
        else:
            assert torch.equal(g, o.to(g.dtype))


@on_gpu
@pytest.mark.parametrize("sizes", [[1], [-1], [7, -3], [4096], [8192], [8191, -8193], [-4097, 8200, 1], [0, 5, 0, -6, 0], [100000, -50001, 8],
                                   [3] * 127, [3] * 128, [5] * 129, [17, -9] * 150, [1 << 24, 4096, -(1 << 22)], [1 << 25, -3, 5, 1]])
@pytest.mark.parametrize("max_norm", [1.0, 1e9])
def test_sizes(sizes, max_norm):
    check(make(sizes), max_norm)


@on_gpu
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e18, 1e25])
def test_sizes_whose_squares_leave_fp32(size):
    check(make([5000, -3000], size), 0.5 * size, eps=0.0)


@on_gpu
def test_views_that_begin_anywhere():
    """Parameters one behind the other in flat buffers: nothing is aligned."""
    flat = torch.randn(40000, device="cuda")
    half = torch.randn(40000, device="cuda").bfloat16()
    grads = [flat[1:9000], flat[9000:9003].view(3, 1), half[3:20000], half[20000:38000]]
    keep = (flat.clone(), half.clone())
    check([g for g in grads])
    for whole, old, parts in ((flat, keep[0], ((0, 1), (9003, 40000))), (half, keep[1], ((0, 3), (38000, 40000)))):
        for lo, hi in parts:
            assert torch.equal(whole[lo:hi], old[lo:hi])


@on_gpu
def test_layouts():
    be = get_backend("hip")
    g = torch.randn(30, 50, device="cuda").bfloat16().t()              # dense, column-major
    cube = torch.randn(4, 6, 8, device="cuda").permute(2, 0, 1)
    want = true_norm([g, cube])
    assert abs(float(be.grad_norm([g, cube])) - want) <= 1.01 * U * want
    out = [torch.empty_like(g, dtype=torch.float32), torch.empty_like(cube)]
    be.clip_grad_norm([g, cube], 1.0, out=out)
    for t, o in ((g, out[0]), (cube, out[1])):
        exact = t.double() / (want + 1e-6)
        assert bool(((o.double() - exact).abs() <= 2.02 * U * exact.abs()).all())


@on_gpu
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_norm_that_is_no_number(bad):
    """The factor that the formula gives: 0 for an infinite norm, not a number for that."""
    be = get_backend("hip")
    grads = make([1000, -1000])
    grads[0][17] = bad
    norm = be.clip_grad_norm(grads, 1.0)
    assert str(float(norm)) == str(bad)
    if bad == float("inf"):
        assert bool((grads[1] == 0).all()) and bool(torch.isnan(grads[0][17])) and int(torch.isnan(grads[0]).sum()) == 1
    else:
        assert all(bool(torch.isnan(g).all()) for g in grads)


@on_gpu
def test_zeros_and_nothing():
    be = get_backend("hip")
    assert float(be.grad_norm([])) == 0.0 and float(be.clip_grad_norm([], 1.0)) == 0.0
    grads = [torch.zeros(100, device="cuda")]
    assert float(be.clip_grad_norm(grads, 1.0)) == 0.0 and bool((grads[0] == 0).all())
    assert float(be.clip_grad_norm(make([0, 0]), 1.0)) == 0.0
    grads = make([100])
    be.clip_grad_norm(grads, 0.0)
    assert bool((grads[0] == 0).all())


@on_gpu
def test_the_sum_is_reproducible():
    be = get_backend("hip")
    grads = make([1 << 22, -(1 << 20), 999])
    first = be.grad_norm(grads)
    assert all(torch.equal(be.grad_norm(grads), first) for _ in range(5))


@on_gpu
def test_more_than_2_to_32_elements_of_bytes():
    """Offsets past 32 bits: 2^31 + 5000 elements."""
    be = get_backend("hip")
    g = torch.zeros((1 << 31) + 5000, device="cuda", dtype=torch.bfloat16)
    g[-1], g[0], g[1 << 31] = 3.0, 4.0, 12.0
    assert float(be.clip_grad_norm([g], 6.5, eps=0.0)) == 13.0
    assert [float(g[i]) for i in (-1, 0, 1 << 31)] == [1.5, 2.0, 6.0]
    del g
    torch.cuda.empty_cache()


@on_gpu
def test_captured_with_other_work_between_replays():
    be = get_backend("hip")
    grads = make([5000, -3000])
    out = [torch.empty(g.shape, device="cuda") for g in grads]
    be.clip_grad_norm(grads, 1.0, out=out)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    norms = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            norms.append(be.clip_grad_norm(grads, 1.0, out=out))
    for seed in (1, 2, 3):
        for g, src in zip(grads, make([5000, -3000], seed=seed)):
            g.copy_(src)
        for graph, norm in zip(graphs, norms):
            graph.replay()
            torch.cuda.synchronize()
            got, scaled = norm.clone(), [o.clone() for o in out]
            assert torch.equal(be.clip_grad_norm(grads, 1.0, out=out), got) and all(torch.equal(a, b) for a, b in zip(scaled, out))


def refusals(be, device):
    a, b = make([100, 100], device=device)
    f = torch.zeros(100, device=device)
    return (lambda: be.grad_norm([a, a]), lambda: be.grad_norm([a, a[50:]]), lambda: be.grad_norm([a.half()]),
            lambda: be.grad_norm([a[::2]]), lambda: be.grad_norm([a.expand(3, 100)]), lambda: be.clip_grad_norm([a], -1.0),
            lambda: be.clip_grad_norm([a], float("nan")), lambda: be.clip_grad_norm([a], 1.0, eps=-1.0),
            lambda: be.clip_grad_norm([a, b], 1.0, out=[f]), lambda: be.clip_grad_norm([a, b], 1.0, out=[f, f]),
            lambda: be.clip_grad_norm([a], 1.0, out=[b]), lambda: be.clip_grad_norm([a], 1.0, out=[f[:50]]),
            lambda: be.clip_grad_norm([f], 1.0, out=[f]), lambda: be.clip_grad_norm([], 1.0, out=[f]),
            lambda: be.clip_grad_norm([f.view(10, 10)], 1.0, out=[torch.zeros(10, 10, device=device).t()]))


def test_refusals():
    for bad in refusals(get_backend("eager"), "cpu"):
        with pytest.raises(RuntimeError):
            bad()


@on_gpu
def test_refusals_on_the_device():
    for bad in refusals(get_backend("hip"), "cuda"):
        with pytest.raises(RuntimeError):
            bad()
    with pytest.raises(RuntimeError):
        get_backend("hip").grad_norm(make([10], device="cpu"))


def test_refusals_of_the_library():
    import ctypes

    lib = hip.load_library()
    ptrs = lambda *p: (ctypes.c_void_p * len(p))(*p)  # noqa: E731
    counts = lambda *n: (ctypes.c_int64 * len(n))(*n)  # noqa: E731
    types = lambda *n: (ctypes.c_int * len(n))(*n)  # noqa: E731
    norm = lambda p, n, t, to=16, ws=16, size=1 << 20: lib.kr_grad_norm(1, p, n, t, to, ws, size, None)  # noqa: E731
    assert lib.kr_grad_norm(0, ptrs(16), counts(1), types(0), 16, 16, 1 << 20, None) == -1
    assert norm(ptrs(17), counts(1), types(0)) == -1 and norm(ptrs(18), counts(1), types(1)) == -1 and norm(ptrs(None), counts(1), types(0)) == -1
    assert norm(ptrs(16), counts(-1), types(0)) == -1 and norm(ptrs(16), counts(1 << 37), types(0)) == -2
    assert norm(ptrs(16), counts(1), types(0), ws=None) == -1 and norm(ptrs(16), counts(1), types(0), ws=24) == -1
    assert norm(ptrs(16), counts(1), types(0), size=16) == -1 and norm(ptrs(16), counts(1), types(0), to=None) == -1
    clip = lambda out, m=1.0, e=0.0: lib.kr_grad_clip(1, ptrs(16), counts(1), types(0), out, m, e, 16, 16, 1 << 20, None)  # noqa: E731
    assert clip(None, -1.0) == -1 and clip(None, float("nan")) == -1 and clip(None, 1.0, -1.0) == -1 and clip(ptrs(None)) == -1
    assert clip(ptrs(18)) == -1
    assert lib.kr_grad_norm_workspace_bytes(128) == 16 + 4096 * 8 and lib.kr_grad_norm_workspace_bytes(129) == 16 + 2 * 4096 * 8
    assert lib.kr_grad_norm_workspace_bytes(0) == 0


def test_parameters():
    """One gradient for each parameter object, the main_grad where it keeps one."""
    a, b, c = (torch.nn.Parameter(torch.zeros(4)) for _ in range(3))
    a.grad, b.main_grad = torch.full((4,), 3.0), torch.full((4,), 4.0)
    c.main_grad = None
    assert float(grad_norm([a, b, c, a], backend="eager")) == 10.0
    out = [torch.zeros(4), torch.zeros(4)]
    assert float(clip_grad_norm([a, b, c], 5.0, eps=0.0, backend="eager", out=out)) == 10.0
    assert out[0].tolist() == [1.5] * 4 and out[1].tolist() == [2.0] * 4 and a.grad.tolist() == [3.0] * 4
    clip_grad_norm([a, b, c], 5.0, eps=0.0, backend="eager")
    assert a.grad.tolist() == [1.5] * 4 and b.main_grad.tolist() == [2.0] * 4
    b.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="main_grad and a grad"):
        grad_norm([b], backend="eager")
    assert float(grad_norm([c], backend="eager")) == 0.0


def test_one_parameter_and_gradients_with_a_history():
    """A parameter by itself is one, not its rows; gradients of a graph that is kept are scaled in place all the same."""
    p = torch.nn.Parameter(torch.full((2, 3), 2.0))
    (p.grad,) = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
    want = float(p.grad.detach().double().norm())
    assert float(grad_norm(p, backend="eager")) == pytest.approx(want, rel=1e-6)
    assert float(clip_grad_norm(p, 0.5 * want, eps=0.0, backend="eager")) == pytest.approx(want, rel=1e-6)
    assert p.grad.detach().flatten().tolist() == [6.0] * 6
    p.grad = None


def test_the_chunks_of_a_launch_are_counted_in_32_bits():
    """128 tensors to a launch, chunks of 4096 elements: the largest that is taken, 128 times, stays below 2^32 of them."""
    import ctypes

    lib = hip.load_library()
    # (without a place for the norm a count that is taken is refused for that, before anything is launched)
    norm = lambda n: lib.kr_grad_norm(1, (ctypes.c_void_p * 1)(16), (ctypes.c_int64 * 1)(n), (ctypes.c_int * 1)(0), None, 16, 1 << 20, None)  # noqa: E731
    most = (1 << 37) - 4096
    assert 128 * -(-most // 4096) < 1 << 32 <= 128 * -(-(most + 1) // 4096)
    assert norm(most) == -1 and norm(most + 1) == norm((1 << 37) - 1) == -2
