"""Layer norm forward and backward against the formulas in 64 bits.

Bounds.  Results are rounded once, half a step of bf16: 2^-8 of the value.  In front of that stand fp32 operations: a row's sums have at
most 8 elements a lane eight times over and 9 steps across lanes and waves, below 100 additions, so that a sum is 100 * 2^-24 of
the sum of its terms' sizes off, and so is what is formed from it, with a handful of operations more: F = 128 * 2^-24 of the sizes of
the terms below.  Column sums add at most `rows` terms of fp32: (rows + 64) * 2^-24 of their sizes."""

import pytest
import torch

from kareus_amd.backend import get_backend, hip

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]
HALF, F = 2.0 ** -8, 128 * 2.0 ** -24


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def make(rows, cols, seed=0, offset=0.3, device="cuda", dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x = (r(rows, cols) * torch.exp(0.5 * r(rows, 1)) + offset).to(device, dtype)
    dy = (r(rows, cols) * torch.exp(r(rows, 1))).to(device, dtype)
    res = r(rows, cols).to(device, dtype)
    return x, dy, res, (1 + 0.1 * r(cols)).to(device, dtype), (0.1 * r(cols)).to(device, dtype)


def reference(x, dy, w, b, eps, res=None):
    """Results in 64 bits and the sizes that the bounds go by."""
    x, dy, w, b = (t.double() for t in (x, dy, w, b))
    n = x.shape[1]
    mean = x.mean(1, keepdim=True)
    rs = (x.var(1, unbiased=False, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * rs
    size_xh = (x.abs() + x.abs().mean(1, keepdim=True)) * rs * (1 + xh.abs())
    g = dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    a1, a2 = g.abs().mean(1, keepdim=True), (g.abs() * (xh.abs() + size_xh)).mean(1, keepdim=True)
    out = {"y": xh * w + b, "dx": rs * (g - c1 - xh * c2), "dw": (dy * xh).sum(0), "db": dy.sum(0), "mean": mean[:, 0], "rstd": rs[:, 0]}
    tol = {"y": HALF * out["y"].abs() + F * (size_xh * w.abs() + b.abs()),
           "dx": F * rs * (g.abs() + a1 + (xh.abs() + size_xh) * a2 * 2),
           "mean": F * x.abs().mean(1) + 1e-30, "rstd": 4 * F * rs[:, 0] * (1 + (x.abs().mean(1, keepdim=True) * rs)[:, 0])}
    if res is not None:
        out["dx"] = out["dx"] + res.double()
        tol["dx"] = tol["dx"] + F * res.double().abs()
    tol["dx"] = tol["dx"] + HALF * out["dx"].abs()
    rows = x.shape[0]
    tol["dw"] = HALF * out["dw"].abs() + ((rows + 64) * 2.0 ** -24 * dy.abs() * xh.abs() + F * dy.abs() * size_xh).sum(0)
    tol["db"] = HALF * out["db"].abs() + (rows + 64) * 2.0 ** -24 * dy.abs().sum(0)
    return out, tol


def close(name, got, want, tol):
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= tol + 1e-30).all()), (name, float((off / (tol + 1e-30)).max()))


def check(x, dy, w, b, eps=1e-5, res=None, **kw):
    be = get_backend("hip")
    y, mean, rstd = be.layernorm_fwd(x, w, b, eps)
    dx, dw, db = be.layernorm_bwd(dy, x, mean, rstd, w, residual_grad=res, **kw)
    rows = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    want, tol = reference(rows(x), rows(dy), w, b, eps, None if res is None else rows(res))
    for name, t in (("y", y), ("mean", mean), ("rstd", rstd), ("dx", rows(dx)), ("dw", dw), ("db", db)):
        close(name, t, want[name], tol[name])
    return y, dx, dw, db


# widths of every number of lanes and vectors a lane: a row of one vector, of several rows to a wave, up to eight waves a row
@on_gpu
@pytest.mark.parametrize("cols", [8, 64, 72, 128, 136, 256, 264, 512, 520, 1024, 1032, 1544, 2048, 2056, 3584, 4096, 4104, 6152, 8192, 8200, 16384])
@pytest.mark.parametrize("rows", [1, 2, 7, 65])
def test_widths(rows, cols):
    x, dy, res, w, b = make(rows, cols, seed=rows + cols)
    check(x, dy, w, b)
    check(x, dy, w, b, res=res)


@on_gpu
@pytest.mark.parametrize("rows,cols", [(6023, 3584), (4099, 200), (33000, 64), (2100, 4096), (1030, 16384), (1030, 8192), (1100, 5640),
                                       (1281, 6152), (1537, 12288), (5000, 520), (2051, 1024)])
def test_more_rows_than_workgroups(rows, cols):
    x, dy, res, w, b = make(rows, cols)
    first = check(x, dy, w, b, res=res)
    again = check(x, dy, w, b, res=res)
    assert all(torch.equal(p, q) for p, q in zip(first, again))       # in a fixed order


@on_gpu
def test_a_large_mean_leaves_the_variance():
    """x = 1000 + noise: of sum x^2 - n mean^2 an fp32 sum keeps nothing."""
    x, dy, res, w, b = make(64, 4096, offset=1000.0)
    check(x, dy, w, b)


@on_gpu
def test_rows_of_one_value():
    x = torch.full((9, 512), 3.0, device="cuda").bfloat16()
    _, dy, _, w, b = make(9, 512)
    y, mean, rstd = get_backend("hip").layernorm_fwd(x, w, b, 1e-5)
    assert torch.equal(y, b.expand(9, -1)) and bool((mean == 3).all())
    check(x, dy, w, b)


@on_gpu
def test_infinite_and_nan_rows_stay_their_own():
    x, dy, res, w, b = make(12, 1024)
    x[3, 5], x[7, 9] = float("inf"), float("nan")
    be = get_backend("hip")
    y, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    bad = ~torch.isfinite(y).all(1)
    assert bad.tolist() == [i in (3, 7) for i in range(12)]
    dx = be.layernorm_bwd(dy, x, mean, rstd, w)[0]
    assert bool(torch.isfinite(dx[~bad]).all())


@on_gpu
@pytest.mark.parametrize("r", [1, 2, 4, 3])
def test_nanobatch_slices_and_strides(r):
    """Slices of some sequences are read and written where they lie (three of them are copied), other rows stay as they were."""
    s, b, h = 33, 6, 520
    x, dy, res, w, bias = make(s * b, h)
    x3, r3 = x.view(s, b, h)[:, 1:1 + r], res.view(s, b, h)[:, 2:2 + r]
    dy2 = dy.view(s, b, h)[:, :r].reshape(-1, h).contiguous()
    out = torch.full((s, b, h), 7.0, device="cuda").bfloat16()
    if r != 3:
        check(x3, dy2, w, bias, res=r3, out=out[:, 2:2 + r])
        assert bool((out[:, :2] == 7).all()) and bool((out[:, 2 + r:] == 7).all())
    check(x3, dy2, w, bias, res=r3)
    wide = torch.empty(s, h + 24, device="cuda").bfloat16()
    wide[:, 8:8 + h] = x[:s]
    check(wide[:, 8:8 + h], dy[:s], w, bias)
    check(wide.t().contiguous().t()[:, 8:8 + h], dy[:s], w, bias)      # column-major: copied
    off = torch.empty(s * h + 1, device="cuda").bfloat16()[1:].view(s, h).copy_(x[:s])
    check(off, dy[:s], w, bias)                                         # not 16-byte aligned: copied


@on_gpu
def test_partial_rows_of_several_calls_are_one_sum():
    be = get_backend("hip")
    x, dy, res, w, b = make(300, 1024)
    _, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    per = be.layernorm_partial_rows(100, 1024)
    buf = torch.full((3 * per, 2048), float("nan"), device="cuda")
    parts = []
    for i in range(3):
        at = slice(100 * i, 100 * i + 100)
        dx, no, none = be.layernorm_bwd(dy[at], x[at], mean[at], rstd[at], w, partials_out=buf[i * per:(i + 1) * per])
        assert no is None and none is None
        parts.append(dx)
    dw, db = be.layernorm_dparams(buf, w)
    want, tol = reference(x, dy, w, b, 1e-5)
    close("dx", torch.cat(parts), want["dx"], tol["dx"])
    close("dw", dw, want["dw"], tol["dw"])
    close("db", db, want["db"], tol["db"])


@on_gpu
def test_no_rows():
    be = get_backend("hip")
    _, _, _, w, b = make(1, 64)
    x = torch.empty(0, 64, device="cuda").bfloat16()
    y, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    dx, dw, db = be.layernorm_bwd(x, x, mean, rstd, w)
    assert y.shape == dx.shape == (0, 64) and mean.shape == (0,) and bool((dw == 0).all()) and bool((db == 0).all())


@on_gpu
def test_gradients_against_differences():
    """The sum of y dy along a direction against a difference in 64 bits: the reference's own formula is checked, and the kernel by it."""
    x, dy, res, w, b = make(5, 136)
    want, _ = reference(x, dy, w, b, 1e-5)
    d = torch.randn(x.shape, dtype=torch.float64, device="cuda")
    value = lambda t: (torch.nn.functional.layer_norm(t, (136,), w.double(), b.double(), 1e-5) * dy.double()).sum()  # noqa: E731
    h = 1e-6
    slope = (value(x.double() + h * d) - value(x.double() - h * d)) / (2 * h)
    assert abs(float(slope - (want["dx"] * d).sum())) <= 1e-6 * float((want["dx"] * d).abs().sum())
    check(x, dy, w, b)


@on_gpu
def test_more_than_2_to_31_elements():
    """The last rows of 4.6 GB tensors have the bits that they have by themselves."""
    be = get_backend("hip")
    x, dy, _, w, b = make(2000, 16384)
    big_x, big_dy = x.repeat(70, 1), dy.repeat(70, 1)
    y, mean, rstd = be.layernorm_fwd(big_x, w, b, 1e-5)
    dx, _, _ = be.layernorm_bwd(big_dy, big_x, mean, rstd, w)
    y1, mean1, rstd1 = be.layernorm_fwd(x, w, b, 1e-5)
    dx1, _, _ = be.layernorm_bwd(dy, x, mean1, rstd1, w)
    for big, one in ((y, y1), (mean, mean1), (rstd, rstd1), (dx, dx1)):
        assert torch.equal(big[-2000:], one) and torch.equal(big[:2000], one)
    del big_x, big_dy, y, dx
    torch.cuda.empty_cache()


@on_gpu
def test_captured_and_on_another_stream():
    be = get_backend("hip")
    x, dy, res, w, b = make(257, 512)
    eager = check(x, dy, w, b, res=res)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = check(x, dy, w, b, res=res)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, beside))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
        dx, dw, db = be.layernorm_bwd(dy, x, mean, rstd, w, residual_grad=res)
    for seed in (1, 2, 3):
        x2, dy2, res2, w2, b2 = make(257, 512, seed=seed)
        for to, src in ((x, x2), (dy, dy2), (res, res2)):
            to.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        want = check(x, dy, w, b, res=res)
        assert all(torch.equal(p, q) for p, q in zip((y, dx, dw, db), want))


@on_gpu
def test_refusals():
    be = get_backend("hip")
    x, dy, res, w, b = make(4, 64)
    _, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    for bad in (lambda: be.layernorm_fwd(x.float(), w, b, 1e-5), lambda: be.layernorm_fwd(x, w[:56], b, 1e-5),
                lambda: be.layernorm_fwd(x[:, :60], w[:60], b[:60], 1e-5), lambda: be.layernorm_fwd(x.cpu(), w, b, 1e-5),
                lambda: be.layernorm_fwd(x[0], w, b, 1e-5),
                lambda: be.layernorm_bwd(dy[:3], x, mean, rstd, w), lambda: be.layernorm_bwd(dy, x, mean[:3], rstd, w),
                lambda: be.layernorm_bwd(dy, x, mean, rstd, w, residual_grad=res[:, :56]),
                lambda: be.layernorm_bwd(dy, x, mean, rstd, w, out=torch.empty(64, 4, device="cuda").bfloat16().t()),
                lambda: be.layernorm_bwd(dy, x, mean, rstd, w, partials_out=torch.empty(1, 64, device="cuda")),
                lambda: be.layernorm_fwd(*[t.new_zeros(2, 16392) if t.dim() == 2 else t.new_zeros(16392) for t in (x, w, b)], 1e-5)):
        with pytest.raises(RuntimeError):
            bad()


@on_gpu
def test_the_residual_gradient_s_own_place_and_no_other():
    """With few rows the parameters' gradients are summed beside the rows: dx must not be where x or dy is; dres is read before it is
    written.  A gradient of a broadcast value is copied."""
    be = get_backend("hip")
    x, dy, res, w, b = make(37, 200)
    want = check(x, dy, w, b, res=res)
    _, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    for out in (x, dy):
        with pytest.raises(RuntimeError):
            be.layernorm_bwd(dy, x, mean, rstd, w, out=out)
    dx, _, _ = be.layernorm_bwd(dy, x, mean, rstd, w, residual_grad=res, out=res)
    assert dx.data_ptr() == res.data_ptr() and torch.equal(dx, want[1])
    check(x, dy[:1].expand(37, 200), w, b)


def test_an_output_that_is_an_input_of_the_eager_backend():
    be = get_backend("eager")
    x, dy, _, w, b = make(7, 40, device="cpu", dtype=torch.float32)
    _, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    for out in (x, dy):
        with pytest.raises(RuntimeError):
            be.layernorm_bwd(dy, x, mean, rstd, w, out=out)


def test_refusals_of_the_library():
    lib = hip.load_library()
    fwd = lambda *a: lib.kr_layernorm_fwd(*a, None)  # noqa: E731
    assert fwd(16, 16, 16, 16, 16, 16, 4, 16392, 16392, 1, 0, 1e-5) == -2       # wider than 16384
    assert fwd(16, 16, 16, 16, 16, 16, 4, 60, 64, 1, 0, 1e-5) == -2             # width not x8
    assert fwd(16, 16, 16, 16, 16, 16, 4, 64, 60, 1, 0, 1e-5) == -1             # row stride < width
    assert fwd(16, 16, 24, 16, 16, 16, 4, 64, 64, 1, 0, 1e-5) == -1             # bias not 16-byte aligned
    assert fwd(16, 16, None, 16, 16, 16, 4, 64, 64, 1, 0, 1e-5) == -1
    assert fwd(16, 16, 16, 16, 16, 16, 4, 64, 64, 3, 512, 1e-5) == -1           # runs are powers of two
    assert fwd(16, 16, 16, 16, 16, 16, 4, 64, 64, 8, 512, 1e-5) == -2           # ... that divide the rows
    bwd = lambda dg, db, ws, rows=4, ld=64: lib.kr_layernorm_bwd(  # noqa: E731
        16, 16, 16, 16, 16, None, 16, dg, db, ws, rows, 64, ld, 64, 1, 0, 0, 1, 0, 64, 1, 0, None)
    assert bwd(16, None, 16) == -1 and bwd(16, 16, None, rows=1025) == -1 and bwd(None, None, None) == -1 and bwd(16, 16, 24) == -1 and bwd(16, 16, 16, rows=0) == -1
    assert bwd(16, 16, 16, ld=68) == -2
    assert bwd(16, 16, 16) == -1                                                # dx where x and dy are
    assert lib.kr_layernorm_dparams(16, 0, 64, 16, 16, None) == -1 and lib.kr_layernorm_dparams(16, 1, 64, 16, None, None) == -1
    assert lib.kr_layernorm_bwd_partial_rows(257, 512) == 65 and lib.kr_layernorm_bwd_workspace_bytes(257, 512) == 65 * 2 * 512 * 4
    assert lib.kr_layernorm_bwd_partial_rows(4, 60) == 0 and lib.kr_layernorm_bwd_workspace_bytes(4, 16392) == 0


@pytest.mark.parametrize("res", [False, True])
def test_the_eager_backend(res):
    x, dy, r, w, b = make(7, 40, device="cpu", dtype=torch.float32)
    be = get_backend("eager")
    y, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    dx, dw, db = be.layernorm_bwd(dy, x, mean, rstd, w, residual_grad=r if res else None)
    want, _ = reference(x, dy, w, b, 1e-5, r if res else None)
    for name, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        assert torch.allclose(t.double(), want[name], rtol=1e-5, atol=1e-5)


@on_gpu
@pytest.mark.parametrize("rows,cols", [(3000, 64), (3000, 200), (2100, 512), (2500, 768), (1500, 1024), (1300, 2048), (1100, 4096), (1100, 5120),
                                       (1100, 8192), (1100, 12288), (1100, 16384), (1024, 8192), (700, 512), (5, 16384)])
def test_the_residual_gradient_s_own_place_in_every_form(rows, cols):
    """Rows of few lanes to eight waves, with the next row's loads ahead and without, few rows and many, a row stride: the same bits in
    the residual gradient's place as elsewhere."""
    be = get_backend("hip")
    x, dy, res, w, b = make(rows, cols)
    _, mean, rstd = be.layernorm_fwd(x, w, b, 1e-5)
    want = be.layernorm_bwd(dy, x, mean, rstd, w, residual_grad=res)
    wide = torch.full((rows, cols + 24), 7.0, device="cuda").bfloat16()
    wide[:, 8:8 + cols] = res
    for place in (res, wide[:, 8:8 + cols]):
        got = be.layernorm_bwd(dy, x, mean, rstd, w, residual_grad=place, out=place)
        assert got[0].data_ptr() == place.data_ptr() and all(torch.equal(p, q) for p, q in zip(got, want))
    assert bool((wide[:, :8] == 7.0).all()) and bool((wide[:, 8 + cols:] == 7.0).all())
