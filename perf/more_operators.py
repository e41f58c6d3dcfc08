"""Operators of decoder layers with layer norms, windowed attention and rotary positions of several axes, and of a training
step's end, in their plain form and through the framework.

A case is a flat dict:
  kind   "norm"       layer norm of x [t, h] forward, and backward from dy: y, dx, and the gradients of weight and bias;
                      residual: dx has the gradient of the residual branch added to it
         "attention"  causal attention of q [s, b, nq, hd] over k and v [s, b, nkv, hd] in which token i sees the last `window`
                      tokens, itself among them, and the first `sinks`: o and the log-sum-exp; backward: dq, dk and dv too
         "rotary"     query and key heads of a fused projection [s, b, nkv, nq / nkv + 2, hd] and of its gradient rotated by
                      the positions of `axes` axes: frequency i belongs to one axis, by sections one behind the other or interleaved
         "grads"      the 2-norm of all gradients of `layers` layers (bf16) and of a table of `vocab` rows (fp32, 0: none);
                      clip: and the gradients, scaled by min(1, 1 / (norm + 1e-6)), one behind the other in fp32
  t, h / s, b, nq, nkv, hd, window, sinks, backward / far (the largest position) / layers, h, nq, nkv, hd, ffn, vocab, clip
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5


def listed():
    return [
        # a unit-test sized layer, an odd number of tokens
        dict(name="norm_small", kind="norm", t=257, h=512, residual=False),
        # three packed sequences of a length that no tile divides
        dict(name="norm_ragged", kind="norm", t=6023, h=3584, residual=True),
        # a microbatch of eight sequences, 8B width
        dict(name="norm_large", kind="norm", t=32768, h=4096, residual=True),
        # a unit-test sized layer with a short window
        dict(name="attention_small", kind="attention", s=257, b=1, nq=8, nkv=8, hd=64, window=64, sinks=4, backward=True),
        # sequences that end inside a tile, four-way shard
        dict(name="attention_ragged", kind="attention", s=2007, b=3, nq=8, nkv=2, hd=128, window=500, sinks=5, backward=True),
        # scoring long texts: forward only, no sinks
        dict(name="attention_score", kind="attention", s=8192, b=2, nq=16, nkv=4, hd=64, window=1024, sinks=0, backward=False),
        # training on long texts, four-way shard
        dict(name="attention_long", kind="attention", s=16384, b=1, nq=8, nkv=2, hd=128, window=4096, sinks=64, backward=True),
        # a prompt with a small image, interleaved axes
        dict(name="rotary_prompt", kind="rotary", s=389, b=1, nq=8, nkv=2, hd=128, axes=3, interleaved=True, far=4096),
        # a microbatch of long videos, far into them
        dict(name="rotary_video", kind="rotary", s=8191, b=4, nq=32, nkv=8, hd=128, axes=3, interleaved=False, far=1 << 20),
        # one small layer: the norm alone, as it is logged
        dict(name="grads_small", kind="grads", layers=1, h=512, nq=4, nkv=2, hd=128, ffn=1024, vocab=0, clip=False),
        # a four-way shard of four layers and the table's fp32 gradient, clipped for the optimizer
        dict(name="grads_stack", kind="grads", layers=4, h=4096, nq=8, nkv=2, hd=128, ffn=3584, vocab=32064, clip=True),
        # a thin eight-way shard of many layers
        dict(name="grads_many", kind="grads", layers=28, h=2048, nq=2, nkv=1, hd=128, ffn=768, vocab=0, clip=True),
    ]


def _spread(rng, lo, hi, unit=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / unit)) * unit)


def _cost(c):
    w = work(c)
    return w["flops"] / 1e15 + w["bytes"] / 4e12


def draw(rng):
    """One more case: any kind; tokens from one to 32768, widths 64 to 16384 (multiples of 8), sequences up to 16384 with windows
    from one token to more than the sequence; at most the largest listed case's work."""
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("norm", "norm", "attention", "attention", "attention", "rotary", "grads"))
        nkv = rng.choice((1, 2, 3, 8))
        heads = dict(nq=nkv * rng.choice((1, 2, 4)), nkv=nkv, hd=rng.choice((64, 128)))
        if kind == "norm":
            c = dict(kind=kind, t=_spread(rng, 1, 32768), h=_spread(rng, 64, 16384, 8), residual=rng.random() < 0.5)
        elif kind == "attention":
            s = _spread(rng, 1, 16384)
            c = dict(kind=kind, s=s, b=rng.choice((1, 2, 3)), **heads, window=_spread(rng, 1, max(2, s + s // 4)),
                     sinks=rng.choice((0, 1, 4, 40, 130)), backward=rng.random() < 0.7)
            if c["b"] * c["nq"] * s * s > 1 << 31:
                continue
        elif kind == "rotary":
            c = dict(kind=kind, s=_spread(rng, 1, 8192), b=rng.choice((1, 2, 3, 4)), **heads, axes=rng.choice((1, 2, 3, 4)),
                     interleaved=rng.random() < 0.5, far=_spread(rng, 8192, 1 << 24))
        else:
            c = dict(kind=kind, layers=_spread(rng, 1, 32), h=_spread(rng, 256, 4096, 8), **heads, ffn=_spread(rng, 256, 4096, 8),
                     vocab=rng.choice((0, 0, 1000, 32064)), clip=rng.random() < 0.7)
        if _cost(c) <= most:
            return c


# ---- states ---------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _gradients(gen, t, n):
    """Small, and over three orders of magnitude from token to token."""
    return (_normal(gen, t, n) * (1e-4 * torch.exp(1.5 * _normal(gen, t, 1)))).bfloat16()


def _sections(c):
    """Frequencies of each axis: the first (time) a share of its own, the others alike, as many as there are in all."""
    half, n = c["hd"] // 2, c["axes"]
    each = half // (n + 1) if n > 1 else 0
    rest = (half - each) // (n - 1) if n > 1 else 0
    return (half - rest * (n - 1),) + (rest,) * (n - 1)


def _positions(c, gen):
    """Texts with images among them: [axes, b, s].  A text's tokens have one position on all axes; an image's, a row of w after
    another, the image's own on the first and their place in it on the others; every sequence starts anywhere up to `far`."""
    s, b, n = c["s"], c["b"], c["axes"]
    i = torch.arange(s, device="cuda").expand(b, s)
    start = torch.randint(0, c["far"] - s + 1 if c["far"] > s else 1, (b, 1), generator=gen, device="cuda")
    w = torch.randint(5, 40, (b, 1), generator=gen, device="cuda")
    block, at = i // (w * w), i % (w * w)
    image = block % 2 == 1
    base = start + torch.where(image, block * w * w, i)
    place = torch.stack([torch.zeros_like(at), at // w, at % w, at % 7])[:n]
    return (base + torch.where(image, place, torch.zeros_like(place))).contiguous()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "norm":
        t, h = c["t"], c["h"]
        x = _normal(gen, t, h) * torch.exp(0.5 * _normal(gen, t, 1)) + 0.3
        x[:, ::97] *= 12.0
        return dict(c, x=x.bfloat16(), dy=_gradients(gen, t, h), dres=_gradients(gen, t, h) if c["residual"] else None,
                    weight=(1.0 + 0.1 * _normal(gen, h)).bfloat16(), bias=(0.1 * _normal(gen, h)).bfloat16())
    if c["kind"] == "attention":
        s, b, nkv, hd, per = c["s"], c["b"], c["nkv"], c["hd"], c["nq"] // c["nkv"]
        fused = _normal(gen, s, b, nkv, per + 2, hd)
        if c["sinks"]:
            fused[:c["sinks"], :, :, per] += 0.5 * fused[-1:, :, :, 0]     # keys that later queries look for
        fused = fused.bfloat16()
        do = _gradients(gen, s * b, c["nq"] * hd).view(s, b, c["nq"] * hd) if c["backward"] else None
        return dict(c, q=fused[:, :, :, :per], k=fused[:, :, :, per], v=fused[:, :, :, per + 1], do=do, scale=hd ** -0.5)
    if c["kind"] == "rotary":
        shape = (c["s"], c["b"], c["nkv"], c["nq"] // c["nkv"] + 2, c["hd"])
        at = torch.arange(0, c["hd"], 2, dtype=torch.float64, device="cuda") / c["hd"]
        return dict(c, fused=_normal(gen, *shape).bfloat16(), grad=_normal(gen, *shape).bfloat16(), positions=_positions(c, gen),
                    inv_freq=1.0 / 500000.0 ** at, sections=_sections(c))
    size = lambda i: 10.0 ** (-2.0 - 0.2 * (i % 9))  # noqa: E731
    grads = [(_normal(gen, *shape) * size(i)).bfloat16() for i, shape in enumerate(_shapes(c))]
    if c["vocab"]:
        grads.append(_normal(gen, c["vocab"], c["h"]) * 1e-2)
    if not c["clip"]:
        return dict(c, grads=grads)
    flat = torch.empty(sum(g.numel() for g in grads), device="cuda")       # as an optimizer holds them
    return dict(c, grads=grads, flat=flat, out=[p.view(g.shape) for p, g in zip(flat.split([g.numel() for g in grads]), grads)])


def _shapes(c):
    """The parameters of a layer, in order: a norm's weight and bias, the projections, another norm's."""
    h, q = c["h"], c["nq"] * c["hd"]
    layer = [(h,), (h,), (q + 2 * c["nkv"] * c["hd"], h), (h, q), (h,), (h,), (2 * c["ffn"], h), (h, c["ffn"])]
    return layer * c["layers"]


# ---- one pass -------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from kareus_amd import RotaryAxes
    from kareus_amd.backend import get_backend

    be = get_backend("hip")
    if st["kind"] == "norm":
        y, mean, rstd = be.layernorm_fwd(st["x"], st["weight"], st["bias"], EPS)
        dx, dweight, dbias = be.layernorm_bwd(st["dy"], st["x"], mean, rstd, st["weight"], residual_grad=st["dres"])
        return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
    if st["kind"] == "attention":
        band = dict(window=st["window"], sinks=st["sinks"])
        o, lse = be.attn_fwd(st["q"], st["k"], st["v"], st["scale"], **band)
        if not st["backward"]:
            return {"o": o, "lse": lse}
        dq, dk, dv = be.attn_bwd(st["do"], st["q"], st["k"], st["v"], o, lse, st["scale"], **band)
        return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    if st["kind"] == "rotary":
        at = RotaryAxes(st["positions"], st["inv_freq"], st["sections"], st["interleaved"])
        per = st["fused"].shape[3] - 2
        return {"fused": be.rope_axes_fused(st["fused"], per, at), "grad": be.rope_axes_fused(st["grad"], per, at, backward=True)}
    if not st["clip"]:
        return {"norm": be.grad_norm(st["grads"])}
    return {"norm": be.clip_grad_norm(st["grads"], 1.0, out=st["out"]), "grads": st["flat"]}


def _heads(t, per):
    """[s, b, nkv, per, hd] -> fp32 [b, nkv, per s, hd]."""
    s, b, nkv, _, hd = t.shape
    return t.float().permute(1, 2, 3, 0, 4).reshape(b, nkv, per * s, hd)


def _rows(t, s, per):
    """[b, nkv, per s, hd] -> bf16 [s, b, nkv, per, hd]."""
    b, nkv, _, hd = t.shape
    return t.view(b, nkv, per, s, hd).permute(3, 0, 1, 2, 4).bfloat16().contiguous()


def _axis_of(sections, interleaved, device):
    """The axis of each frequency: one section behind the other, or in turn while an axis has any left, the first behind that."""
    n = len(sections)
    i = torch.arange(sum(sections), device=device)
    edges = torch.tensor(sections, device=device)
    if not interleaved:
        return (i[:, None] >= edges.cumsum(0)).sum(1)
    return torch.where(i // n < edges[i % n], i % n, torch.zeros_like(i))


def _turn(t, cos, sin):
    """Query and key heads of [s, b, nkv, per + 2, hd] rotated, halves layout; value heads as they are."""
    a, b = t[..., :-1, :].float().chunk(2, -1)
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).bfloat16()
    return torch.cat([turned, t[..., -1:, :]], 3)


def _run_plain(st):
    if st["kind"] == "norm":
        x, dy, w = st["x"].float(), st["dy"].float(), st["weight"].float()
        d = x - x.mean(1, keepdim=True)
        r = torch.rsqrt(d.square().mean(1, keepdim=True) + EPS)
        xh = d * r
        y = xh * w + st["bias"].float()
        g = dy * w
        dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        if st["residual"]:
            dx += st["dres"].float()
        return {"y": y.bfloat16(), "dx": dx.bfloat16(), "dweight": (dy * xh).sum(0).bfloat16(), "dbias": dy.sum(0).bfloat16()}
    if st["kind"] == "attention":
        s, b, nkv, per, hd = st["q"].shape
        q, k, v = _heads(st["q"], per), _heads(st["k"].unsqueeze(3), 1), _heads(st["v"].unsqueeze(3), 1)
        i = torch.arange(s, device=q.device)
        back = i[:, None] - i
        seen = (back >= 0) & ((back < st["window"]) | (i < st["sinks"]))
        x = (q @ k.transpose(2, 3) * st["scale"]).view(b, nkv, per, s, s).masked_fill_(~seen, -math.inf).view(b, nkv, per * s, s)
        top = x.amax(3, keepdim=True)
        p = x.sub_(top).exp_()
        total = p.sum(3, keepdim=True)
        p /= total
        o = p @ v
        lse = (top + total.log()).view(b, nkv * per, s)
        out = {"o": _rows(o, s, per).view(s, b, nkv * per, hd), "lse": lse}
        if not st["backward"]:
            return out
        do = _heads(st["do"].view(s, b, nkv, per, hd), per)
        dv = p.transpose(2, 3) @ do
        dp = do @ v.transpose(2, 3)
        ds = dp.sub_((do * o).sum(3, keepdim=True)).mul_(p).mul_(st["scale"])
        return dict(out, dq=_rows(ds @ k, s, per), dk=_rows(ds.transpose(2, 3) @ q, s, 1).squeeze(3), dv=_rows(dv, s, 1).squeeze(3))
    if st["kind"] == "rotary":
        at = st["positions"][_axis_of(st["sections"], st["interleaved"], st["positions"].device)]    # [hd / 2, b, s]
        angle = (at.double() * st["inv_freq"][:, None, None]).permute(2, 1, 0)[:, :, None, None]
        cos, sin = angle.cos().float(), angle.sin().float()
        return {"fused": _turn(st["fused"], cos, sin), "grad": _turn(st["grad"], cos, -sin)}
    norm = torch.stack([g.double().square().sum() for g in st["grads"]]).sum().sqrt()
    if not st["clip"]:
        return {"norm": norm.float()}
    factor = (1.0 / (norm + 1e-6)).clamp(max=1.0).float()
    return {"norm": norm.float(), "grads": torch.cat([g.flatten().float() for g in st["grads"]]).mul_(factor)}


# ---- what a pass cannot do without ---------------------------------------------------------------
def _pairs(s, window, sinks):
    """Visible (token, earlier or same token) pairs of a sequence."""
    w = min(window, s)
    near = w * (w + 1) // 2 + (s - w) * w
    n = s - w                                # tokens whose window has left the first tokens: 1 .. n of them out of sight
    far = n * (n + 1) // 2 if n <= sinks else sinks * (sinks + 1) // 2 + (n - sinks) * sinks
    return near + far


def work(case):
    c = case
    if c["kind"] == "norm":
        n = c["t"] * c["h"]
        return {"bytes": 2 * n * (5 if c["residual"] else 4) + 8 * c["h"], "flops": 20 * n}
    if c["kind"] == "attention":
        tokens = c["s"] * c["b"]
        q, kv = 2 * tokens * c["nq"] * c["hd"], 2 * tokens * c["nkv"] * c["hd"]
        pairs = c["b"] * c["nq"] * _pairs(c["s"], c["window"], c["sinks"])
        lse = 4 * tokens * c["nq"]
        if not c["backward"]:
            return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * pairs * c["hd"]}
        return {"bytes": 4 * q + 4 * kv + lse, "flops": 14 * pairs * c["hd"]}
    if c["kind"] == "rotary":
        tokens = c["s"] * c["b"]
        n = tokens * (c["nq"] + 2 * c["nkv"]) * c["hd"]
        return {"bytes": 2 * 2 * 2 * n + 8 * c["axes"] * tokens, "flops": 2 * 3 * n}
    n = sum(math.prod(shape) for shape in _shapes(c))
    table = c["vocab"] * c["h"]
    read = 2 * n + 4 * table
    return {"bytes": read + (4 * (n + table) if c["clip"] else 0), "flops": (3 if c["clip"] else 2) * (n + table)}


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_attention(st):
    """A stretch of queries at a time over the keys that any of them sees."""
    s, b, nkv, per, hd = st["q"].shape
    q = st["q"].double().permute(1, 2, 3, 0, 4).contiguous()
    k, v = (st[n].double().permute(1, 2, 0, 3).unsqueeze(2).contiguous() for n in ("k", "v"))
    o, lse = torch.zeros_like(q), torch.zeros_like(q[..., 0])
    both = st["backward"]
    if both:
        do = st["do"].double().view(s, b, nkv, per, hd).permute(1, 2, 3, 0, 4).contiguous()
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    step = max(1, (1 << 27) // (b * nkv * per * s))
    for lo in range(0, s, step):
        hi = min(s, lo + step)
        keys = torch.arange(hi, device=q.device)
        keys = keys[(keys < st["sinks"]) | (keys > lo - st["window"])]
        rows = torch.arange(lo, hi, device=q.device).unsqueeze(1)
        hidden = (keys > rows) | ((rows - keys >= st["window"]) & (keys >= st["sinks"]))
        ks, vs = k[:, :, :, keys], v[:, :, :, keys]
        z = torch.einsum("bgpid,bgpjd->bgpij", q[..., lo:hi, :], ks.expand(-1, -1, per, -1, -1)) * st["scale"]
        z = z.masked_fill(hidden, -math.inf)
        lse[..., lo:hi] = torch.logsumexp(z, -1)
        p = torch.softmax(z, -1)
        o[..., lo:hi, :] = p @ vs
        if both:
            g = do[..., lo:hi, :]
            dv.index_add_(3, keys, (p.transpose(3, 4) @ g).sum(2, keepdim=True))
            dz = p * (g @ vs.transpose(3, 4) - (g * o[..., lo:hi, :]).sum(-1, keepdim=True)) * st["scale"]
            dq[..., lo:hi, :] = dz @ ks
            dk.index_add_(3, keys, (dz.transpose(3, 4) @ q[..., lo:hi, :]).sum(2, keepdim=True))
    first = lambda t: t.permute(3, 0, 1, 2, 4).contiguous()  # noqa: E731
    out = {"o": first(o).view(s, b, nkv * per, hd), "lse": lse.view(b, nkv * per, s)}
    return dict(out, dq=first(dq), dk=first(dk).squeeze(3), dv=first(dv).squeeze(3)) if both else out


def _exact_norm(st):
    x = st["x"].double().requires_grad_(True)
    w, b = (st[n].double().requires_grad_(True) for n in ("weight", "bias"))
    y = torch.nn.functional.layer_norm(x, x.shape[1:], w, b, EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), st["dy"].double())
    return {"y": y.detach(), "dx": dx + st["dres"].double() if st["residual"] else dx, "dweight": dw, "dbias": db}


def _exact_rotary(st):
    """Pairs of channels as complex numbers times e^(i angle)."""
    sections, n = st["sections"], len(st["sections"])
    axis = []
    if st["interleaved"]:
        for i in range(sum(sections)):
            axis.append(i % n if i // n < sections[i % n] else 0)
    else:
        for a, size in enumerate(sections):
            axis += [a] * size
    half = len(axis)
    place = st["positions"].double().permute(2, 1, 0)[:, :, axis] * st["inv_freq"]
    found = {}
    for name, sign in (("fused", 1.0), ("grad", -1.0)):
        t = st[name].double()
        z = torch.complex(t[..., :half], t[..., half:]) * torch.polar(torch.ones_like(place), sign * place)[:, :, None, None]
        z = torch.cat([z.real, z.imag], -1)
        z[..., -1, :] = t[..., -1, :]
        found[name] = z
    return found


def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "norm":
        return _exact_norm(st)
    if st["kind"] == "attention":
        return _exact_attention(st)
    if st["kind"] == "rotary":
        return _exact_rotary(st)
    norm = sum(torch.linalg.vector_norm(g.double()) ** 2 for g in st["grads"]) ** 0.5
    if not st["clip"]:
        return {"norm": norm}
    factor = min(1.0, 1.0 / (float(norm) + 1e-6))
    return {"norm": norm, "grads": torch.cat([g.double().flatten() for g in st["grads"]]) * factor}
