"""Rotary positions on several axes against complex rotations in 64 bits.

Bounds.  One rounding, half a step of bf16: 2^-8 of the value.  The angle in turns is formed in 64 bits and its fraction rounded to
32: half a turn times 2^-25, which is pi * 2^-24 of a radian; sine and cosine are a few units off, the products and the sum three
roundings: together below 16 * 2^-24 of |a| + |b|."""

import pytest
import torch

from kareus_amd import RotaryAxes, rotary_axes
from kareus_amd.backend import get_backend, hip
from kareus_amd.operators import rotary_frequencies
from kareus_amd.rotary_axes import axis_of_frequency, inverse_frequencies

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]
HALF, F = 2.0 ** -8, 16 * 2.0 ** -24


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def sections_of(hd, axes):
    half = hd // 2
    each = half // (axes + 1)
    return (half - each * (axes - 1),) + (each,) * (axes - 1)


def make(s, b, heads, hd, axes, far=100000, device="cuda", dtype=torch.bfloat16, interleaved=False, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randn(s, b, heads, hd, generator=gen).to(device, dtype)
    p = torch.randint(0, far, (axes, b, s), generator=gen).to(device)
    return t, rotary_axes(p, hd, sections_of(hd, axes), 500000.0, interleaved)


def reference(t, at, backward=False):
    half = t.shape[-1] // 2
    axis = axis_of_frequency(at.sections, at.interleaved).tolist()
    angle = (at.positions.double()[axis] * at.inv_freq[:, None, None]).permute(2, 1, 0)
    angle = (-angle if backward else angle).view(angle.shape[:2] + (1,) * (t.dim() - 3) + (half,))
    x = t.double()
    a, b = x[..., :half], x[..., half:]
    out = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
    size = (a.abs() + b.abs()).repeat((1,) * (t.dim() - 1) + (2,))
    return out, HALF * out.abs() + F * size


def close(got, want, tol):
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= tol).all()), float((off / (tol + 1e-30)).max())


@on_gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("hd", [16, 64, 80, 96, 128, 256])
def test_heads(hd, axes, interleaved):
    be = get_backend("hip")
    t, at = make(37, 2, 5, hd, axes, interleaved=interleaved)
    close(be.rope_axes_fwd(t, at), *reference(t, at))
    close(be.rope_axes_bwd(t, at), *reference(t, at, True))


@on_gpu
@pytest.mark.parametrize("s,b,ng,per,hd", [(1, 1, 1, 1, 64), (389, 1, 2, 4, 128), (200, 3, 8, 4, 128), (33, 2, 3, 1, 64), (3001, 4, 1, 7, 128)])
def test_fused_buffers(s, b, ng, per, hd):
    be = get_backend("hip")
    t, at = make(s, b, ng * (per + 2), hd, 3, far=1 << 24)
    fused = t.view(s, b, ng, per + 2, hd)
    before = fused.clone()
    for backward in (False, True):
        out = be.rope_axes_fused(fused, per, at, backward=backward)
        want, tol = reference(fused, at, backward)
        close(out[:, :, :, :per + 1], want[:, :, :, :per + 1], tol[:, :, :, :per + 1])
        assert torch.equal(out[:, :, :, per + 1], fused[:, :, :, per + 1]) and torch.equal(fused, before)
        place = fused.clone()
        assert be.rope_axes_fused(place, per, at, backward=backward, out=place) is place and torch.equal(place, out)
        to = torch.empty_like(fused)
        assert be.rope_axes_fused(fused, per, at, backward, to) is to and torch.equal(to, out)


@on_gpu
@pytest.mark.parametrize("far", [1 << 20, 1 << 31, 1 << 40])
def test_far_positions(far):
    """Where a 32-bit angle has lost its fraction.  (64-bit turns at 2^40 are 2^-13 of a turn off: the bound's second part.)"""
    be = get_backend("hip")
    t, at = make(64, 2, 4, 128, 3, far=far)
    p = at.positions
    p[:, :, -1] = far
    want, tol = reference(t, at)
    half = t.shape[-1] // 2
    size = (t.double()[..., :half].abs() + t.double()[..., half:].abs()).repeat(1, 1, 1, 2)
    close(be.rope_axes_fwd(t, at), want, tol + far * 2.0 ** -51 * 8 * size)


@on_gpu
def test_equal_positions_are_the_plain_rotation():
    be = get_backend("hip")
    t, _ = make(128, 2, 6, 128, 3)
    p = torch.arange(128, device="cuda").expand(3, 2, 128).contiguous()
    at = rotary_axes(p, 128, (16, 24, 24), 500000.0)
    plain = be.rope_fwd(t, rotary_frequencies(128, 128, 500000.0, device="cuda")).double()
    size = t.double().abs().amax() * 2
    # (the plain one's fp32 table: an angle of 127 radians is 127 * 3 * 2^-24 off)
    assert bool(((be.rope_axes_fwd(t, at).double() - plain).abs() <= 2 * HALF * plain.abs() + (F + 384 * 2.0 ** -24) * size).all())


@on_gpu
def test_negative_positions_views_and_strides():
    be = get_backend("hip")
    t, at = make(50, 4, 6, 64, 3)
    at.positions.neg_()
    close(be.rope_axes_fwd(t, at), *reference(t, at))
    part = at.sequences(1, 3)
    close(be.rope_axes_fwd(t[:, 1:3], part), *reference(t[:, 1:3], part))
    by_token = RotaryAxes(at.positions.permute(2, 1, 0).contiguous().permute(2, 1, 0), at.inv_freq, at.sections)
    assert torch.equal(be.rope_axes_fwd(t, by_token), be.rope_axes_fwd(t, at))
    grouped = t.view(50, 4, 2, 3, 64)
    assert torch.equal(be.rope_axes_fwd(grouped, at), be.rope_axes_fwd(t, at))
    odd = torch.empty(50, 4, 6, 65, device="cuda").bfloat16()[..., 1:].copy_(t)      # strides of 65: copied
    assert torch.equal(be.rope_axes_fwd(odd, at), be.rope_axes_fwd(t, at))


@on_gpu
def test_back_and_forth_is_the_input():
    be = get_backend("hip")
    t, at = make(100, 2, 6, 128, 3, far=1 << 20)
    back = be.rope_axes_bwd(be.rope_axes_fwd(t, at), at).double()
    half = t.shape[-1] // 2
    size = (t.double()[..., :half].abs() + t.double()[..., half:].abs()).repeat(1, 1, 1, 2)
    assert bool(((back - t.double()).abs() <= 3 * HALF * size).all())


@on_gpu
def test_more_than_2_to_31_elements():
    be = get_backend("hip")
    s, b, heads, hd = 420000, 1, 40, 128
    t = torch.randn(1000, b, heads, hd, device="cuda").bfloat16().repeat(s // 1000, 1, 1, 1)
    at = rotary_axes(torch.arange(s, device="cuda").expand(3, b, s), hd, (24, 20, 20))
    turned = be.rope_axes_fwd(t, at)
    part = be.rope_axes_fwd(t[-1000:].contiguous(), at._replace(positions=at.positions[:, :, -1000:]))
    assert t.numel() > 1 << 31 and torch.equal(turned[-1000:], part)
    del t, turned
    torch.cuda.empty_cache()


@on_gpu
def test_captured():
    be = get_backend("hip")
    t, at = make(389, 1, 10, 128, 3)
    fused = t.view(389, 1, 2, 5, 128)
    be.rope_axes_fused(fused, 3, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = be.rope_axes_fused(fused, 3, at)
    for seed in (1, 2, 3):
        t2, at2 = make(389, 1, 10, 128, 3, seed=seed)
        fused.copy_(t2.view(fused.shape))
        at.positions.copy_(at2.positions)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, be.rope_axes_fused(fused, 3, at))


@on_gpu
def test_refusals():
    be = get_backend("hip")
    t, at = make(8, 2, 5, 64, 3)
    fused = t.view(8, 2, 1, 5, 64)
    for bad in (lambda: be.rope_axes_fwd(t, at._replace(positions=at.positions[:, :1])),
                lambda: be.rope_axes_fwd(t, at._replace(positions=at.positions.int())),
                lambda: be.rope_axes_fwd(t, at._replace(positions=at.positions[:2])),
                lambda: be.rope_axes_fwd(t, at._replace(inv_freq=at.inv_freq.float())),
                lambda: be.rope_axes_fwd(t, at._replace(inv_freq=at.inv_freq[:16])),
                lambda: be.rope_axes_fwd(t, at._replace(sections=(8, 8, 8))),
                lambda: be.rope_axes_fwd(t, at._replace(sections=(40, -4, -4))),
                lambda: be.rope_axes_fwd(t, at._replace(inv_freq=at.inv_freq.cpu())),
                lambda: be.rope_axes_fwd(t.float(), at), lambda: be.rope_axes_fwd(t.cpu(), at),
                lambda: be.rope_axes_fwd(t[..., :24], at), lambda: be.rope_axes_fused(fused, 4, at),
                lambda: be.rope_axes_fused(fused[:, :1], 3, at.sequences(0, 1)),
                lambda: be.rope_axes_fused(fused, 3, at, out=fused.flatten()[:0].expand(0))):
        with pytest.raises(RuntimeError):
            bad()
    buf = torch.zeros(fused.numel() + 64, device="cuda").bfloat16()
    with pytest.raises(RuntimeError, match="overlaps"):
        be.rope_axes_fused(buf[:fused.numel()].view(fused.shape), 3, at, out=buf[64:].view(fused.shape))


@on_gpu
def test_no_tokens():
    be = get_backend("hip")
    t, at = make(0, 2, 4, 64, 3)
    assert be.rope_axes_fwd(t, at).shape == (0, 2, 4, 64)
    assert be.rope_axes_fused(t.view(0, 2, 1, 4, 64), 2, at).shape == (0, 2, 1, 4, 64)


def test_refusals_of_the_library():
    import ctypes

    lib = hip.load_library()

    def call(sections=(8, 8, 16), axes=None, hd=64, heads=5, group=5, rotate=4, t=16, stride=64, inv=16):
        c = (ctypes.c_int * len(sections))(*sections)
        return lib.kr_rope_axes(t, 16, 16, 8, 8, 1, len(sections) if axes is None else axes, inv, c, 0, 4, 2, heads, hd, stride, 64, 64, 64,
                                64, 64, 0, group, rotate, None)

    assert call(axes=0) == -1 and call(sections=(8, 8, 8)) == -1 and call(sections=(40, -8)) == -1
    assert call(sections=(8, 8, 8, 4, 4)) == -2 and call(hd=72, sections=(36,)) == -2 and call(hd=272, sections=(136,)) == -2
    assert call(group=4) == -1 and call(rotate=6) == -1 and call(t=24) == -1 and call(stride=68) == -1 and call(stride=0) == -2
    assert call(inv=12) == -1


def test_axes_of_frequencies():
    assert axis_of_frequency((2, 3, 3), False).tolist() == [0, 0, 1, 1, 1, 2, 2, 2]
    assert axis_of_frequency((4, 2, 2), True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert axis_of_frequency((8,), True).tolist() == [0] * 8
    with pytest.raises(RuntimeError):
        rotary_axes(torch.zeros(2, 1, 4, dtype=torch.int64), 32, (8, 4))
    assert torch.allclose(inverse_frequencies(8, 10000.0), torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15, atol=0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_eager_backend(interleaved):
    be = get_backend("eager")
    t, at = make(9, 2, 5, 32, 3, device="cpu", dtype=torch.float32, interleaved=interleaved)
    for backward, got in ((False, be.rope_axes_fwd(t, at)), (True, be.rope_axes_bwd(t, at))):
        assert torch.allclose(got.double(), reference(t, at, backward)[0], rtol=0, atol=1e-5)
    fused = t.view(9, 2, 1, 5, 32)
    out = be.rope_axes_fused(fused, 3, at)
    assert torch.equal(out[:, :, :, 4], fused[:, :, :, 4])
    assert torch.allclose(out[:, :, :, :4].double(), reference(fused, at)[0][:, :, :, :4], rtol=0, atol=1e-5)
    place = fused.clone()
    assert torch.equal(be.rope_axes_fused(place, 3, at, out=place), out)
