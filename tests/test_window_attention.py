"""Causal attention with a window and sinks, forward and backward, against the formulas in 64 bits.

Bounds, element by element, from what is rounded.  u = 2^-24, half a bf16 step 2^-8 of a value.
  scores       at most hd fp32 additions, the scale and the exponential's argument: es = (hd + 8) u scale sum |q k| + 8 u (1 + |x|);
               a probability is e = 2 max_j es + 2^-21 of itself off, the log-sum-exp max es + 8 u (1 + |lse|) + 2^-21
  o            probabilities rounded to bf16, then o: 2^-8 |o| + (2^-8 + e) sum p |v|
  dV           the same with P and dO: 2^-8 |dV| + sum (2^-8 + e) P |dO|
  delta        dO . o with the rounded o: D = sum |dO| (bound of o) + hd u sum |dO o|
               of a row's first 128 queries and windows up to 64, sum P dP over sum P: their errors weigh what dP is off delta by,
               D = sum P (e |dP - delta| + hd u sum |dO V|) + (s + 8) u sum P |dP|
  dS           rounded to bf16 behind P (dP - delta): ds = 2^-8 |dS| + P (e |dP - delta| + hd u sum |dO V| + D)
  dQ, dK       2^-8 of the result + scale sum ds |k|, scale sum ds |q|"""

import os
import re
import subprocess
import sys

import pytest
import torch

from kareus_amd.backend import get_backend, hip

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]
HALF, U = 2.0 ** -8, 2.0 ** -24


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def make(s, b, nq, nkv, hd, seed=0, device="cuda", dtype=torch.bfloat16):
    """Views of a fused projection, and a gradient."""
    gen = torch.Generator().manual_seed(seed)
    per = nq // nkv
    fused = torch.randn(s, b, nkv, per + 2, hd, generator=gen).to(device, dtype)
    do = torch.randn(s, b, nq * hd, generator=gen).to(device, dtype)
    return fused[:, :, :, :per], fused[:, :, :, per], fused[:, :, :, per + 1], do


def visible(s, window, sinks, device):
    i = torch.arange(s, device=device)
    back = i[:, None] - i
    return (back >= 0) & ((back < window) | (i < sinks))


def reference(q, k, v, do, scale, window, sinks, from_scores=False):
    s, b, nkv, per, hd = q.shape
    rows = lambda t: t.double().permute(1, 2, 3, 0, 4)                    # noqa: E731  [b, nkv, per, s, hd]
    q, g = rows(q), rows(do.view(s, b, nkv, per, hd))
    k, v = (t.double().permute(1, 2, 0, 3).unsqueeze(2) for t in (k, v))   # [b, nkv, 1, s, hd]
    seen = visible(s, window, sinks, q.device)
    t = lambda m: m.transpose(-1, -2)                                      # noqa: E731
    x = (q @ t(k) * scale).masked_fill(~seen, -torch.inf)
    size = (q.abs() @ t(k).abs() * scale).masked_fill(~seen, 0.0)
    es = ((hd + 8) * U * size + 8 * U * (1 + x.abs())).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    e = 2 * es + 2.0 ** -21
    lse = torch.logsumexp(x, -1)
    p = torch.softmax(x, -1)
    o = p @ v
    out = {"o": o, "lse": lse}
    tol = {"o": HALF * o.abs() + (HALF + e) * (p @ v.abs()), "lse": es[..., 0] + 8 * U * (1 + lse.abs()) + 2.0 ** -21}
    dp = g @ t(v)
    delta = (g * o).sum(-1, keepdim=True)
    d_off = (g.abs() * tol["o"]).sum(-1, keepdim=True) + hd * U * (g * o).abs().sum(-1, keepdim=True)
    ds = p * (dp - delta)
    if from_scores:
        d_off = (p * (e * (dp - delta).abs() + hd * U * (g.abs() @ t(v).abs()) + (s + 8) * U * dp.abs())).sum(-1, keepdim=True)
    ds_off = HALF * ds.abs() + p * (e * (dp - delta).abs() + hd * U * (g.abs() @ t(v).abs()) + d_off)
    group = lambda m: m.sum(2, keepdim=True)                               # noqa: E731
    out["dv"], out["dq"], out["dk"] = group(t(p) @ g), scale * (ds @ k), scale * group(t(ds) @ q)
    tol["dv"] = HALF * out["dv"].abs() + group(t(p * (HALF + e)) @ g.abs())
    tol["dq"] = HALF * out["dq"].abs() + scale * (ds_off @ k.abs())
    tol["dk"] = HALF * out["dk"].abs() + scale * group(t(ds_off) @ q.abs())
    back = {"o": lambda m: m.permute(3, 0, 1, 2, 4).reshape(s, b, nkv * per, hd), "dq": lambda m: m.permute(3, 0, 1, 2, 4),
            "dk": lambda m: m.permute(3, 0, 1, 2, 4).squeeze(3), "lse": lambda m: m.reshape(b, nkv * per, s)}
    back["dv"] = back["dk"]
    return {n: back[n](m) for n, m in out.items()}, {n: back[n](m) for n, m in tol.items()}


def close(name, got, want, tol):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    off = (got.double() - want).abs()
    assert bool((off <= tol + 1e-30).all()), (name, float((off / (tol + 1e-30)).max()))


def check(q, k, v, do, window, sinks, scale=None, beside=False, from_scores=False):
    be = get_backend("hip")
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    band = dict(window=window, sinks=sinks, beside_other_streams=beside)
    o, lse = be.attn_fwd(q, k, v, scale, **band)
    dq, dk, dv = be.attn_bwd(do, q, k, v, o, lse, scale, **band)
    want, tol = reference(q, k, v, do, scale, window, sinks, from_scores)
    for name, t in (("lse", lse), ("o", o), ("dv", dv), ("dk", dk), ("dq", dq)):
        close(name, t, want[name], tol[name])
    return o, lse, dq, dk, dv


# lengths around tiles of 64 and 128 and their ends, windows within a tile, of a tile, over several; sinks inside the window's reach or far from it
@on_gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("s,window,sinks", [
    (1, 1, 0), (2, 1, 0), (2, 1, 1), (3, 1, 1), (17, 4, 2), (64, 16, 0), (64, 1, 0), (64, 63, 0), (65, 64, 0), (65, 1, 4), (127, 50, 3), (128, 64, 0),
    (128, 1, 0), (128, 127, 0), (129, 128, 0), (129, 100, 4), (192, 64, 64), (192, 65, 63), (200, 7, 130), (255, 128, 1), (256, 128, 0),
    (256, 64, 4), (257, 64, 4), (257, 129, 33), (300, 1, 1), (384, 128, 32), (384, 200, 4), (385, 31, 65), (512, 256, 4), (640, 128, 200),
    (640, 300, 129), (700, 65, 1), (1000, 333, 40), (1000, 999, 0), (1024, 512, 16), (1100, 20, 1000)])
def test_lengths_windows_and_sinks(s, window, sinks, hd):
    check(*make(s, 1, 2, 1, hd, seed=s + window), window, sinks)


@on_gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("b,nq,nkv", [(1, 1, 1), (2, 3, 3), (3, 8, 2), (1, 7, 1), (2, 12, 3), (5, 16, 16)])
@pytest.mark.parametrize("s,window,sinks", [(333, 100, 5), (256, 96, 0)])
def test_heads(b, nq, nkv, hd, s, window, sinks):
    check(*make(s, b, nq, nkv, hd), window, sinks)


# rows with few keys: of a window, of a short sequence, all but one of them with next to no probability
@on_gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [None, 1.0])
@pytest.mark.parametrize("s,b,nq,nkv,window,sinks", [(2, 1, 2, 1, 1, 1), (2, 2, 1, 1, 2, 0), (3, 1, 4, 2, 1, 40), (24, 1, 2, 1, 19, 1), (31, 1, 2, 2, 12, 40),
                                                     (100, 2, 3, 1, 100, 0), (128, 1, 4, 4, 70, 9), (300, 1, 2, 2, 64, 4), (515, 1, 4, 2, 33, 130),
                                                     (700, 2, 2, 1, 1, 1), (1300, 8, 16, 4, 20, 0), (1300, 8, 16, 4, 64, 66)])
def test_rows_with_few_keys(s, b, nq, nkv, window, sinks, scale, hd):
    check(*make(s, b, nq, nkv, hd, seed=s), window, sinks, scale=scale, from_scores=True)


# rows that leave the sinks' keys to a kernel of their own, and those around the shortest that do
@on_gpu
@pytest.mark.parametrize("hd,nq,nkv", [(64, 2, 2), (64, 6, 2), (128, 3, 3), (128, 4, 1)])
@pytest.mark.parametrize("s,window,sinks", [(896, 127, 3), (896, 128, 3), (897, 128, 130), (512, 127, 4), (512, 128, 4), (513, 129, 33), (1153, 1, 33),
                                            (1280, 100, 200), (1300, 30, 1), (1408, 65, 65), (1536, 128, 32), (1111, 63, 129)])
def test_sinks_of_long_rows(s, window, sinks, hd, nq, nkv):
    check(*make(s, 2, nq, nkv, hd, seed=s), window, sinks)


@on_gpu
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("beside", [False, True])
def test_many_workgroups(hd, beside):
    """More tiles than units: several heads of a group to a workgroup, one half's dQ."""
    check(*make(1300, 8, 16, 4, hd), 200, 6, beside=beside)


@on_gpu
@pytest.mark.parametrize("s,b,nq,hd,window,sinks", [(2304, 8, 4, 64, 2048, 5), (2816, 4, 6, 64, 2200, 0), (4352, 4, 4, 128, 4096, 70), (4864, 7, 2, 128, 4200, 0),
                                                    (4864, 7, 2, 128, 4111, 130)])
def test_long_windows(s, b, nq, hd, window, sinks):
    """dQ over 256-query tiles, one wave per SIMD.  (The reference goes head by head: 64-bit scores of thousands of tokens.)"""
    be = get_backend("hip")
    q, k, v, do = make(s, b, nq, 1, hd)
    q, k, v, do = (t.contiguous() for t in (q, k, v, do))
    band = dict(window=window, sinks=sinks)
    o, lse = be.attn_fwd(q, k, v, hd ** -0.5, **band)
    dq, dk, dv = be.attn_bwd(do, q, k, v, o, lse, hd ** -0.5, **band)
    for bi in (0, b - 1):
        part = slice(bi, bi + 1)
        want, tol = reference(q[:, part], k[:, part], v[:, part], do[:, part].contiguous(), hd ** -0.5, window, sinks)
        for name, t in (("lse", lse[part]), ("o", o[:, part]), ("dv", dv[:, part]), ("dk", dk[:, part]), ("dq", dq[:, part])):
            close(name, t, want[name], tol[name])
    torch.cuda.empty_cache()


@on_gpu
@pytest.mark.parametrize("hd", [8, 40, 80, 96, 120])
def test_other_head_dimensions(hd):
    check(*make(210, 2, 4, 2, hd), 50, 3)


@on_gpu
def test_scores_over_a_wide_range():
    """The running maximum moves in every tile; a sink that takes nearly all of a row."""
    q, k, v, do = make(500, 1, 2, 1, 128)
    k *= torch.linspace(0.2, 8, 500, device="cuda").view(-1, 1, 1, 1).bfloat16()
    check(q, k, v, do, 130, 4)
    k[:4] = 3 * q[-1:, :, :, 0]
    check(q, k, v, do, 130, 4)
    check(q, k.flip(0), v, do, 130, 4, scale=0.5)


@on_gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_a_window_that_hides_nothing_is_plain_attention(hd):
    be = get_backend("hip")
    for window, sinks in ((300, 0), (1 << 40, 0), (299, 1), (100, 200), (1, 1 << 40)):    # (short rows keep to the window's kernels)
        check(*make(300, 2, 4, 2, hd), window, sinks)
    q, k, v, do = make(520, 2, 4, 2, hd)
    plain = be.attn_fwd(q, k, v, 0.1)
    grads = be.attn_bwd(do, q, k, v, *plain, 0.1)
    for window, sinks in ((520, 0), (1 << 40, 0), (519, 1), (320, 200), (1, 1 << 40)):
        got = be.attn_fwd(q, k, v, 0.1, window=window, sinks=sinks)
        assert all(torch.equal(a, b) for a, b in zip(plain, got))
        assert all(torch.equal(a, b) for a, b in zip(grads, be.attn_bwd(do, q, k, v, *got, 0.1, window=window, sinks=sinks)))


@on_gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_layouts(hd):
    """Dense query heads, batch-major tensors, slices of a wider batch, rows that no kernel can read where they lie."""
    be = get_backend("hip")
    s, b, nq, nkv = 290, 4, 6, 2
    q, k, v, do = make(s, b, nq, nkv, hd)
    o, lse, dq, dk, dv = check(q, k, v, do, 77, 5)
    band = dict(window=77, sinks=5)
    scale = hd ** -0.5
    major = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    odd = lambda t: torch.empty(*t.shape[:-1], hd + 1, device="cuda").bfloat16()[..., 1:].copy_(t)  # noqa: E731
    dense = q.reshape(s, b, nq, hd).contiguous()
    for x, y, z in ((dense, k.contiguous(), v.contiguous()), (major(dense), major(k), major(v)), (odd(dense), odd(k), odd(v))):
        o2, lse2 = be.attn_fwd(x, y, z, scale, **band)
        assert torch.equal(o2, o) and torch.equal(lse2, lse)
        for g in (do, do.view(s, b, nq, hd), major(do.view(s, b, nq, hd)), odd(do.view(s, b, nq, hd))):
            got = be.attn_bwd(g, x, y, z, o, lse, scale, **band)
            assert all(torch.equal(p.reshape(r.shape), r) for p, r in zip(got, (dq, dk, dv)))
    part = slice(1, 3)
    o2, lse2 = be.attn_fwd(q[:, part], k[:, part], v[:, part], scale, **band)
    assert torch.equal(o2, o[:, part]) and torch.equal(lse2, lse[part])
    got = be.attn_bwd(do[:, part].contiguous(), q[:, part], k[:, part], v[:, part], o2, lse2, scale, **band)
    assert torch.equal(got[0], dq[:, part])


@on_gpu
def test_offsets_past_32_bits():
    """The last sequence of a buffer of more than 4 GB, alone and where it lies."""
    be = get_backend("hip")
    s, b, nkv, per, hd = 9000, 40, 8, 4, 128
    fused = torch.zeros(s, b, nkv, per + 2, hd, device="cuda", dtype=torch.bfloat16)
    assert fused.numel() * 2 > 1 << 32
    one = torch.randn(s, 1, nkv, per + 2, hd, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    fused[:, -1:] = one
    do = torch.zeros(s, b, nkv * per * hd, device="cuda", dtype=torch.bfloat16)
    do[:, -1:] = torch.randn(s, 1, nkv * per * hd, device="cuda").bfloat16()
    cut = lambda t: (t[:, :, :, :per], t[:, :, :, per], t[:, :, :, per + 1])  # noqa: E731
    o, lse = be.attn_fwd(*cut(fused), 0.09, window=600, sinks=4)
    grads = be.attn_bwd(do, *cut(fused), o, lse, 0.09, window=600, sinks=4)
    alone = do[:, -1:].contiguous()
    o1, lse1 = be.attn_fwd(*cut(one), 0.09, window=600, sinks=4)
    grads1 = be.attn_bwd(alone, *cut(one), o1, lse1, 0.09, window=600, sinks=4)
    assert torch.equal(o[:, -1:], o1) and torch.equal(lse[-1:], lse1) and torch.equal(grads[0][:, -1:], grads1[0])
    for a, c in zip(grads[1:], grads1[1:]):       # (heads are added in another order: fp32, rounded once)
        assert bool(((a[:, -1:].double() - c.double()).abs() <= 2.02 * HALF * c.double().abs() + 1e-3).all())
    del fused, do, o, grads
    torch.cuda.empty_cache()


@on_gpu
def test_gradients_against_differences():
    q, k, v, do = make(40, 1, 2, 1, 64)
    want, _ = reference(q, k, v, do, 0.125, 9, 2)
    seen = visible(40, 9, 2, "cuda")

    def value(q, k, v):
        rows = lambda t: t.permute(1, 2, 3, 0, 4)  # noqa: E731
        k, v = (t.permute(1, 2, 0, 3).unsqueeze(2) for t in (k, v))
        p = (rows(q) @ k.transpose(-1, -2) * 0.125).masked_fill(~seen, -torch.inf).softmax(-1)
        return ((p @ v) * rows(do.double().view(q.shape))).sum()

    at = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn_like(at[i])
        step = [t + 1e-6 * d if j == i else t for j, t in enumerate(at)], [t - 1e-6 * d if j == i else t for j, t in enumerate(at)]
        slope = (value(*step[0]) - value(*step[1])) / 2e-6
        assert abs(float(slope - (want[name] * d).sum())) <= 1e-6 * float((want[name] * d).abs().sum())


@on_gpu
def test_captured_and_on_other_streams():
    be = get_backend("hip")
    band = dict(window=64, sinks=4)
    q, k, v, do = make(257, 1, 8, 8, 64)
    first = check(q, k, v, do, **band)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            o, lse = be.attn_fwd(q, k, v, 0.125, **band)
            results.append((o, lse, *be.attn_bwd(do, q, k, v, o, lse, 0.125, **band)))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for r in results for a, b in zip(r, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = be.attn_fwd(q, k, v, 0.125, **band)
        got = (o, lse, *be.attn_bwd(do, q, k, v, o, lse, 0.125, **band))
    fused = q._base
    for seed in (1, 2, 3):
        q2, _, _, do2 = make(257, 1, 8, 8, 64, seed=seed)
        fused.copy_(q2._base)
        do.copy_(do2)
        graph.replay()
        torch.cuda.synchronize()
        want = check(q, k, v, do, **band)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@on_gpu
def test_no_tokens():
    be = get_backend("hip")
    q, k, v, do = make(0, 2, 4, 2, 64)
    o, lse = be.attn_fwd(q, k, v, 0.125, window=4, sinks=1)
    dq, dk, dv = be.attn_bwd(do, q, k, v, o, lse, 0.125, window=4, sinks=1)
    assert o.shape == (0, 2, 4, 64) and lse.shape == (2, 4, 0) and dq.shape == q.shape and dk.shape == k.shape


def refusals(be, device):
    q, k, v, do = make(20, 1, 4, 2, 64, device=device, dtype=torch.bfloat16)
    return (lambda: be.attn_fwd(q, k, v, 0.1, window=-1), lambda: be.attn_fwd(q, k, v, 0.1, window=4, sinks=-1),
            lambda: be.attn_fwd(q, k, v, 0.1, sinks=4), lambda: be.attn_fwd(q, k, v, 0.1, causal=False, window=4))


def test_refusals():
    for bad in refusals(get_backend("eager"), "cpu"):
        with pytest.raises(RuntimeError):
            bad()


@on_gpu
def test_refusals_on_the_device():
    be = get_backend("hip")
    q, k, v, do = make(20, 1, 4, 2, 64)
    o, lse = be.attn_fwd(q, k, v, 0.1, window=4)
    wide = torch.zeros(20, 1, 1, 136, device="cuda").bfloat16()
    bwd = lambda **c: be.attn_bwd(*[c.get(n, t) for n, t in zip(("do", "q", "k", "v", "o", "lse"), (do, q, k, v, o, lse))], 0.1, window=4)  # noqa: E731
    for bad in (*refusals(be, "cuda"), lambda: be.attn_fwd(q, k, v, 0.0, window=4), lambda: be.attn_fwd(q, k, v, -0.1, window=4),
                lambda: be.attn_fwd(q, k, v, 0.1, general_kernels=True, window=4), lambda: be.attn_fwd(wide, wide, wide, 0.1, window=4),
                lambda: be.attn_fwd(q, k[:10], v[:10], 0.1, window=4), lambda: be.attn_fwd(q.float(), k, v, 0.1, window=4),
                lambda: be.attn_fwd(q.cpu(), k, v, 0.1, window=4), lambda: bwd(do=do[:10]), lambda: bwd(o=o[:, :, :2]),
                lambda: bwd(lse=lse[:, :2]), lambda: bwd(lse=lse.double()), lambda: bwd(k=k[:, :, :1])):
        with pytest.raises(RuntimeError):
            bad()


def test_refusals_of_the_library():
    lib = hip.load_library()

    def fwd(s=250, hd=64, nq=4, scale=0.1, window=10, sinks=2, flags=0, q=16, stride=64, lse=16):
        return lib.kr_attn_window_fwd(q, 16, 16, 16, lse, s, 1, nq, 2, hd, scale, *([stride] * 14), window, sinks, flags, None)

    assert fwd(window=0) == -1 and fwd(window=-3) == -1 and fwd(sinks=-1) == -1 and fwd(scale=0.0) == -1 and fwd(scale=float("nan")) == -1
    assert fwd(flags=0x200) == -1 and fwd(q=24) == -1 and fwd(q=None) == -1 and fwd(lse=None) == -1 and fwd(stride=68) == -1
    assert fwd(hd=80) == -2 and fwd(hd=136) == -2 and fwd(nq=3) == -2 and fwd(stride=1 << 25) == -2 and fwd(stride=0) == -2 and fwd(s=0) == -1

    def bwd(ws=16, window=10, s=250, hd=64):
        return lib.kr_attn_window_bwd(*([16] * 9), ws, s, 1, 4, 2, hd, 0.1, *([64] * 28), window, 2, 0, None)

    assert bwd(ws=None) == -1 and bwd(ws=24) == -1 and bwd(window=0) == -1 and bwd(s=0) == -1 and bwd(hd=72) == -2
    size = lambda *a: lib.kr_attn_window_bwd_workspace_bytes(*a)  # noqa: E731
    stats, parts = 2 * 4 * 384 * 4, 2 * 4 * 384 * 64 * 4
    assert size(300, 1, 4, 2, 64, 50, 0) == stats + parts
    assert size(300, 1, 4, 4, 64, 50, 0) == size(300, 1, 4, 4, 64, 50, 20) == stats
    # four heads' 32 sinks, the queries from 50 on in eleven stretches of 128: 2 x 2048 sums each, and the first key tile's own
    assert size(1300, 1, 4, 4, 64, 50, 20) == 2 * 4 * 1408 * 4 + 4 * 11 * 2 * 2048 * 4 + 2 * 4 * 128 * 64 * 4
    assert size(600, 1, 4, 2, 64, 600, 0) == size(600, 1, 4, 2, 64, 400, 200) == lib.kr_attn_bwd_workspace_bytes_strided(600, 1, 4, 2, 64, 64)
    assert size(300, 1, 4, 2, 64, 300, 0) == size(300, 1, 4, 2, 64, 200, 100) == stats + parts
    assert size(300, 1, 4, 2, 80, 50, 0) == 0 and size(300, 1, 4, 2, 64, 0, 0) == 0


def test_the_eager_backend():
    be = get_backend("eager")
    q, k, v, do = make(30, 2, 4, 2, 16, device="cpu", dtype=torch.float32)
    o, lse = be.attn_fwd(q, k, v, 0.25, window=6, sinks=2)
    dq, dk, dv = be.attn_bwd(do, q, k, v, o, lse, 0.25, window=6, sinks=2)
    want, _ = reference(q, k, v, do, 0.25, 6, 2)
    for name, t in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert torch.allclose(t.double().reshape(want[name].shape), want[name], rtol=1e-5, atol=1e-5), name


def band_tiles(tmp_path):
    """The kernels' lists of key and query tiles and their order of workgroups, compiled for the host from their source."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    source = open(os.path.join(root, "kareus_amd", "csrc", "kr_attention.hip")).read()
    plain = lambda text: text.replace("__device__ __forceinline__", "inline")  # noqa: E731
    begin = source.index("struct Band {")
    band = plain(source[begin:source.index("// Output staging.", begin)])
    begin = source.index("template <int TQ>\n__device__ __forceinline__ int band_query_tiles(")
    queries = plain(source[begin:source.index("\n}\n", begin) + 3])
    xcds = re.search(r"^constexpr int kXcds = \d+;$", source, re.M).group(0)
    (tmp_path / "band.cpp").write_text(f"""#include <cstdint>
{xcds}
{band}
{queries}
extern "C" int keys(int tk, int window, int sinks, int q0, int rows, int* list) {{
  if (tk == 64) {{ BandTiles<64> t(Band{{window, sinks}}, q0, rows); for (int n = 0; n < t.total + 1; ++n) list[n] = t.of(n); return t.total; }}
  BandTiles<128> t(Band{{window, sinks}}, q0, rows); for (int n = 0; n < t.total + 1; ++n) list[n] = t.of(n); return t.total;
}}
extern "C" int queries(int tq, int window, int sinks, int key0, int sp) {{
  return tq == 64 ? band_query_tiles<64>(Band{{window, sinks}}, key0, sp) : band_query_tiles<128>(Band{{window, sinks}}, key0, sp);
}}
extern "C" void order(int grouped, int nblocks, int ntiles, int nheads, int per, int* tile, int* pair) {{
  for (int i = 0; i < nblocks; ++i)
    grouped ? band_order<true>(i, nblocks, ntiles, nheads, per, tile[i], pair[i])
            : band_order<false>(i, nblocks, ntiles, nheads, per, tile[i], pair[i]);
}}
extern "C" int hides(int window, int sinks, int key0, int n, int q) {{ return band_hides(Band{{window, sinks}}, key0, n, q); }}
extern "C" int hides_all(int window, int sinks, int key0, int n, int q) {{ return band_hides_all(Band{{window, sinks}}, key0, n, q); }}
""")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "band.cpp", "-o", "band.so"], cwd=tmp_path, check=True)
    import ctypes

    return ctypes.CDLL(str(tmp_path / "band.so"))


def test_tiles_that_the_kernels_walk(tmp_path):
    """Every visible pair's tile once, no tile beyond the sequence's last, what lies behind the list marked as such."""
    import ctypes

    lib = band_tiles(tmp_path)
    sp = 768
    for tk in (64, 128):
        for window in (1, 2, 63, 64, 65, 128, 200, 500):
            for sinks in (0, 1, 64, 65, 130, 400):
                seen = visible(sp, window, sinks, "cpu")
                for q0 in range(0, sp, 128):
                    tiles = (ctypes.c_int * 64)()
                    n = lib.keys(tk, window, sinks, q0, 128, tiles)
                    walked = list(tiles[:n])
                    assert walked == sorted(set(walked)) and walked[-1] * tk < q0 + 128 <= sp and tiles[n] * tk >= q0 + 128
                    for t in range(sp // tk):
                        block = seen[q0:q0 + 128, t * tk:(t + 1) * tk]
                        assert t in walked or not bool(block.any())
                        for r in range(0, 128, 32):
                            part = block[r:r + 32]
                            past = torch.arange(t * tk, (t + 1) * tk) > torch.arange(q0 + r, q0 + r + 32)[:, None]
                            if bool((~part & ~past).any()):
                                assert lib.hides(window, sinks, t * tk, tk, q0 + r + 31)
                            if lib.hides_all(window, sinks, t * tk, tk, q0 + r):
                                assert not bool(part.any())
                for some in (0, sinks):
                    near = visible(sp, window, some, "cpu")
                    for key0 in range(0, sp, 128):
                        end = lib.queries(tk, window, some, key0, sp)
                        assert key0 // tk < end <= sp // tk and not bool(near[end * tk:, key0:key0 + 128].any())


def test_the_order_of_workgroups_is_a_permutation(tmp_path):
    import ctypes

    lib = band_tiles(tmp_path)
    for ntiles, heads, per in ((1, 1, 1), (3, 8, 4), (16, 6, 3), (33, 5, 1), (130, 2, 2)):
        n = ntiles * heads
        for grouped in (0, 1):
            tile, pair = (ctypes.c_int * n)(), (ctypes.c_int * n)()
            lib.order(grouped, n, ntiles, heads, per, tile, pair)
            assert sorted(zip(tile, pair)) == [(t, p) for t in range(ntiles) for p in range(heads)]


def test_the_window_kernels_keep_their_reads_in_front_of_barriers(tmp_path):
    """What tests/test_attention_asm.py reads in the plain dK/dV and dQ kernels, in those with a window."""
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    from test_attention_asm import CSRC, HIPCC, _kernel_body, early_readers

    if not os.path.exists(HIPCC):
        pytest.skip("hipcc is not installed")
    out = tmp_path / "kr_attention_window.s"
    subprocess.run(["make", "-C", CSRC, f"HIPCC={HIPCC}", f"ASMDIR={tmp_path}", str(out)], check=True, stdout=subprocess.DEVNULL,
                   stderr=subprocess.DEVNULL, timeout=600)
    text = out.read_text()
    names = set(re.findall(r"^_Z\w*(attn_bwd_dkdv_kernel\w*):", text, re.M))
    assert len(names) == 4
    for name in names:
        blocks = []
        for piece in re.split(r"^\s+s_barrier\b", "\n".join(_kernel_body(text, name)), flags=re.M):
            mfmas, hand_over, fragments = (len(re.findall(rf"^\s+{op}", piece, re.M)) for op in ("v_mfma", "ds_read_b128", "ds_read_b64_tr"))
            if mfmas == 16 and hand_over == 4:
                blocks.append(fragments)
        assert len(blocks) >= 2 and set(blocks) == {32}, (name, blocks)
    names = set(re.findall(r"^(_Z\w*attn_bwd_dq_w64_kernel\w*):", text, re.M))
    assert len(names) == 4
    for name in names:   # the hand-placed MFMAs: 128 of the plain kernel's, and the two steps of the loop over hidden keys
        body = text[text.index("\n" + name + ":"):]
        n_asm, bad = early_readers(body[:body.index(".Lfunc_end")].split("\n"))
        assert n_asm == 192 and not bad, (name, n_asm, bad[:5])
    spills = [int(n) for n in re.findall(r"\.vgpr_spill_count:\s*(\d+)", text)]
    assert spills and not any(spills)


def long_window(s, b, nq, hd, window, sinks):
    be = get_backend("hip")
    q, k, v, do = (t.contiguous() for t in make(s, b, nq, 1, hd))
    o, lse = be.attn_fwd(q, k, v, hd ** -0.5, window=window, sinks=sinks)
    return (q, k, v, do), o, lse, *be.attn_bwd(do, q, k, v, o, lse, hd ** -0.5, window=window, sinks=sinks)


@on_gpu
@pytest.mark.parametrize("s,b,nq,hd,window,sinks", [(2300, 8, 4, 64, 2048, 5), (2177, 8, 4, 64, 2050, 0), (4340, 4, 4, 128, 4096, 70),
                                                    (4737, 7, 2, 128, 4111, 130)])
def test_long_windows_of_ragged_rows(s, b, nq, hd, window, sinks):
    """dQ over 256-query tiles, the last of which rows leave: its second half with one token and with nearly all of them."""
    (q, k, v, do), o, lse, dq, dk, dv = long_window(s, b, nq, hd, window, sinks)
    for bi in (0, b - 1):
        part = slice(bi, bi + 1)
        want, tol = reference(q[:, part], k[:, part], v[:, part], do[:, part].contiguous(), hd ** -0.5, window, sinks)
        for name, t in (("lse", lse[part]), ("o", o[:, part]), ("dv", dv[:, part]), ("dk", dk[:, part]), ("dq", dq[:, part])):
            close(name, t, want[name], tol[name])
    torch.cuda.empty_cache()


@on_gpu
@pytest.mark.parametrize("s,b,nq,hd,window,sinks", [(2304, 8, 4, 64, 2048, 5), (2300, 8, 4, 64, 2048, 0), (4352, 4, 4, 128, 4096, 70),
                                                    (4340, 4, 4, 128, 4096, 0)])
def test_first_tokens_under_a_long_window(s, b, nq, hd, window, sinks):
    """The first 128 queries form delta from the scores in every form of dQ.  (They see one another alone; the reference's 256 tokens
    leave room in sum P |dP| for delta's own way through the matrix unit's sums, hd u |delta|, beside the 66 additions of a lane.)"""
    (q, k, v, do), _, _, dq, _, _ = long_window(s, b, nq, hd, window, sinks)
    for bi in (0, b - 1):
        part = [t[:256, bi:bi + 1].contiguous() for t in (q, k, v, do)]
        want, tol = reference(*part, hd ** -0.5, 256, 0, from_scores=True)
        close("dq", dq[:128, bi:bi + 1], want["dq"][:128], tol["dq"][:128])


@on_gpu
@pytest.mark.parametrize("s,nq,nkv,hd,window,sinks", [(384, 8, 2, 64, 100, 3), (512, 8, 2, 128, 100, 3), (700, 4, 4, 128, 65, 0), (512, 4, 2, 64, 600, 0),
                                                      (2304, 4, 1, 64, 2048, 5), (4340, 2, 1, 128, 4096, 0)])
def test_beside_other_streams(s, nq, nkv, hd, window, sinks):
    """Whole rows to a workgroup whatever their number: the same bits for a sequence in a batch of any size."""
    be = get_backend("hip")
    big = 40 if s < 1024 else 10
    q, k, v, do = make(s, 1, nq, nkv, hd)
    band = dict(window=window, sinks=sinks, beside_other_streams=True)
    o, lse = be.attn_fwd(q, k, v, hd ** -0.5, **band)
    dq, dk, dv = be.attn_bwd(do, q, k, v, o, lse, hd ** -0.5, **band)
    q, k, v, do = (t.repeat_interleave(big, dim=1) for t in (q, k, v, do))
    o2, lse2 = be.attn_fwd(q, k, v, hd ** -0.5, **band)
    assert torch.equal(o2[:, 7:8], o) and torch.equal(lse2[7:8], lse)
    assert torch.equal(be.attn_bwd(do, q, k, v, o2, lse2, hd ** -0.5, **band)[0][:, 7:8], dq)
