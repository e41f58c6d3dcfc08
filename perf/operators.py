"""Operators of a shard's training step in their plain form and through the framework: products of 8-bit blocks, linear layers
in 8-bit blocks with both gradients, the scaled token embedding, and its gradient by sorted tokens.

8-bit blocks.  A matrix with rows contiguous along the contraction is held as e4m3 values ``q [rows, pitch]`` (zero from the
contraction's end to the next multiple of 128) and one byte ``s [ceil(k / 128), >= rows]`` per row and block of 128:
value = q * 2^(s - 127).  A block's exponent is the smallest that brings its largest magnitude to 448 or below.  Weights have
one exponent per 128 x 128 tile, so that both orientations hold the same values.

A case is a flat dict:
  kind   "product"     quantised operands in hand: out [m, n] = A . B^T over k
         "step"        bf16 x [t, k], w [n, k], dy [t, n] -> y = x w^T, dx = dy w, dw = dy^T x, quantising what each product takes
         "lookup"      ids [b, s] -> scale * table rows, [s, b, h]
         "gradient"    the table's gradient from ids and d(out): whole, in bf16
         "main_grad"   the same over `micro` microbatches, summed in an fp32 gradient of the table
  m, n, k / t, n, k / b, s, h, vocab, scale, skew (the share of tokens that are one id), micro
"""

from __future__ import annotations

import math

import torch

own = False

LARGEST = 448.0   # of e4m3


def listed():
    return [
        # one token against a kept 8-bit weight: scoring token by token
        dict(name="product_one_token", kind="product", m=1, n=4096, k=4096),
        # a prompt of an odd length through the small configuration's up projection
        dict(name="product_prompt", kind="product", m=389, n=2752, k=512),
        # a weight gradient: few outputs, a contraction over an odd number of tokens
        dict(name="product_weight_gradient", kind="product", m=1536, n=4096, k=6023),
        # the full-width 8B layer's first MLP projection at 16384 tokens
        dict(name="product_large", kind="product", m=16384, n=28672, k=4096),
        # a unit-test sized layer, an odd number of tokens
        dict(name="step_small", kind="step", t=257, n=1376, k=512),
        # three packed sequences of a length that no tile divides, four-way shard
        dict(name="step_ragged", kind="step", t=6023, n=4096, k=3584),
        # eight-way thin shard
        dict(name="step_thin", kind="step", t=32768, n=1536, k=2048),
        # the four-way shard's first MLP projection at 16384 tokens
        dict(name="step_wide", kind="step", t=16384, n=7168, k=4096),
        # a short prompt
        dict(name="lookup_short", kind="lookup", b=1, s=37, h=4096, vocab=32064, scale=64.0),
        # a microbatch of long sequences
        dict(name="lookup_long", kind="lookup", b=8, s=4096, h=2048, vocab=128256, scale=2048.0 ** 0.5),
        # packed sequences with a padding id, the whole gradient written
        dict(name="gradient_padded", kind="gradient", b=8, s=2007, h=4096, vocab=32064, scale=64.0, skew=0.3),
        # gradient accumulation over four microbatches of a large vocabulary
        dict(name="main_grad_4", kind="main_grad", b=2, s=4096, h=2048, vocab=128256, scale=1.0, skew=0.0, micro=4),
    ]


def _spread(rng, lo, hi, unit=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / unit)) * unit)


def draw(rng):
    """One more case: any kind; tokens from one to 32768, features 64 to 28672 (multiples of 8), contractions of any length;
    tables of 1000 to 151936 rows; at most the largest listed case's work."""
    cost = lambda c: work(c)["flops"] / 1e15 + work(c)["bytes"] / 4e12  # noqa: E731
    most = max(cost(c) for c in listed())
    while True:
        kind = rng.choice(("product", "product", "step", "step", "lookup", "gradient", "main_grad"))
        if kind == "product":
            c = dict(kind=kind, m=_spread(rng, 1, 32768), n=_spread(rng, 64, 28672, 8), k=_spread(rng, 64, 16384))
        elif kind == "step":
            c = dict(kind=kind, t=_spread(rng, 1, 32768), n=_spread(rng, 64, 14336, 8), k=_spread(rng, 64, 14336, 8))
        else:
            b = rng.choice((1, 2, 3, 4, 8))
            c = dict(kind=kind, b=b, s=_spread(rng, 1, 32768 // b), h=_spread(rng, 256, 8192, 8),
                     vocab=_spread(rng, 1000, 151936), scale=rng.choice((1.0, 8.0, 45.25)))
            if kind != "lookup":
                c["skew"] = rng.choice((0.0, 0.1, 0.9))
            if kind == "main_grad":
                c["micro"] = rng.choice((1, 2, 4))
        if cost(c) <= most and c.get("h", 1) * c.get("vocab", 1) <= 1 << 29:
            return c


# ---- the plain form of the 8-bit blocks ---------------------------------------------------------
def _block_exponent(amax):
    """Smallest e with amax 2^-e <= 448 = 0.875 2^9 (frexp: amax = f 2^p, f in [0.5, 1))."""
    f, p = torch.frexp(amax)
    e = torch.where(f > 0.875, p - 8, p - 9)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(-127, 127)


def _pow2(e):
    """2^e in fp32, exactly, for whole e of -126 and more (-127: 0, which no block but a zero one asks for)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _padded(x, rows, cols):
    out = x.new_zeros(rows, cols)
    out[:x.shape[0], :x.shape[1]] = x
    return out


def _quantise(x, tiles=False):
    """fp32 [r, c], blocks along c -> e4m3 values [r, cp] (fp32), exponents [r, c / 128]."""
    r, c = x.shape
    rb, cb = -(-r // 128), -(-c // 128)
    if tiles:
        p = _padded(x, rb * 128, cb * 128).view(rb, 128, cb, 128)
        e = _block_exponent(p.abs().amax((1, 3)))
        e = e.view(rb, 1, cb).expand(rb, 128, cb).reshape(rb * 128, cb)[:r]
        p = p.view(rb * 128, cb, 128)[:r]
    else:
        p = _padded(x, r, cb * 128).view(r, cb, 128)
        e = _block_exponent(p.abs().amax(2))
    q = (p * _pow2(-e).unsqueeze(2)).to(torch.float8_e4m3fn).float()
    return q.view(r, cb * 128), e


def _values(x, tiles=False):
    """What the blocks of x stand for, fp32 [r, c]."""
    q, e = _quantise(x, tiles)
    return (q.view(q.shape[0], -1, 128) * _pow2(e).unsqueeze(2)).view(q.shape)[:, :x.shape[1]]


def _held(x):
    """x in the documented format: (q [r, cp] e4m3, s [c / 128, r up to a multiple of 4] bytes)."""
    q, e = _quantise(x)
    s = torch.full((e.shape[1], (x.shape[0] + 3) // 4 * 4), 127, dtype=torch.uint8, device=x.device)
    s[:, :x.shape[0]] = (e.t() + 127).to(torch.uint8)
    return q.to(torch.float8_e4m3fn), s


def _stand_for(q, s, k):
    r = q.shape[0]
    e = s[:, :r].t().to(torch.int32) - 127
    return (q.float().view(r, -1, 128) * _pow2(e).unsqueeze(2)).view(r, -1)[:, :k]


# ---- states ---------------------------------------------------------------------------------------
def _activations(t, k, gen):
    """Tokens of different sizes, a few channels far larger than the rest."""
    x = torch.randn(t, k, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(t, 1, generator=gen, device="cuda"))
    x[:, ::97] *= 12.0
    return x


def _gradients(t, n, gen):
    """Small, and over three orders of magnitude from token to token."""
    return torch.randn(t, n, generator=gen, device="cuda") * (1e-4 * torch.exp(1.5 * torch.randn(t, 1, generator=gen, device="cuda")))


def _ids(c, gen):
    """Frequent and rare ids as in text (the cube of a uniform number), and a share of one id."""
    u = torch.rand(c["b"], c["s"], generator=gen, device="cuda")
    ids = (u * u * u * c["vocab"]).long().clamp_(max=c["vocab"] - 1)
    if c.get("skew"):
        one = torch.rand(c["b"], c["s"], generator=gen, device="cuda") < c["skew"]
        ids = torch.where(one, torch.full_like(ids, c["vocab"] // 2), ids)
    return ids


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if c["kind"] == "product":
        a, b = _held(_activations(c["m"], c["k"], gen)), _held(0.02 * torch.randn(c["n"], c["k"], generator=gen, device="cuda"))
        return dict(c, a=a, b=b)
    if c["kind"] == "step":
        return dict(c, x=_activations(c["t"], c["k"], gen).bfloat16(), dy=_gradients(c["t"], c["n"], gen).bfloat16(),
                    w=(0.02 * torch.randn(c["n"], c["k"], generator=gen, device="cuda")).bfloat16())
    if c["kind"] == "lookup":
        return dict(c, ids=_ids(c, gen), table=(0.02 * torch.randn(c["vocab"], c["h"], generator=gen, device="cuda")).bfloat16())
    n = c.get("micro", 1)
    return dict(c, ids=[_ids(c, gen) for _ in range(n)],
                dout=[_gradients(c["s"] * c["b"], c["h"], gen).view(c["s"], c["b"], c["h"]).bfloat16() for _ in range(n)])


# ---- one pass -------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(st):
    from kareus_amd import BlockOperand
    from kareus_amd.backend import get_backend

    be = get_backend("hip")
    kind = st["kind"]
    if kind == "product":
        return be.block_matmul(BlockOperand(*st["a"], st["k"]), BlockOperand(*st["b"], st["k"]))
    if kind == "step":
        x = be.quantize_blocks(st["x"], by_row=True, by_col=True)
        w = be.quantize_blocks(st["w"], by_row=True, by_col=True, tiles=True)
        y = be.block_matmul(x.by_row, w.by_row)
        dy = be.quantize_blocks(st["dy"], by_row=True, by_col=True)
        return {"y": y, "dx": be.block_matmul(dy.by_row, w.by_col), "dw": be.block_matmul(dy.by_col, x.by_col)}
    if kind == "lookup":
        return be.embedding_fwd(st["ids"], st["table"], scale=st["scale"])
    if kind == "gradient":
        return be.embedding_bwd_sorted(st["ids"][0], st["dout"][0], st["vocab"], scale=st["scale"])
    out = torch.empty(st["vocab"], st["h"], dtype=torch.float32, device=st["dout"][0].device)
    for i, (ids, dout) in enumerate(zip(st["ids"], st["dout"])):
        be.embedding_bwd_sorted(ids, dout, st["vocab"], scale=st["scale"], out=out, accumulate=i > 0)
    return out


def _run_plain(st):
    kind = st["kind"]
    if kind == "product":
        return (_stand_for(*st["a"], st["k"]) @ _stand_for(*st["b"], st["k"]).t()).bfloat16()
    if kind == "step":
        x, w, dy = st["x"].float(), _values(st["w"].float(), tiles=True), st["dy"].float()
        y = _values(x) @ w.t()
        dx = _values(dy) @ w
        dw = _values(dy.t().contiguous()) @ _values(x.t().contiguous()).t()
        return {"y": y.bfloat16(), "dx": dx.bfloat16(), "dw": dw.bfloat16()}
    if kind == "lookup":
        return (st["table"][st["ids"].t()].float() * st["scale"]).bfloat16()
    ids, dout = torch.stack(st["ids"]), torch.stack(st["dout"])
    total = dout.new_zeros(st["vocab"], st["h"], dtype=torch.float32)
    total.index_add_(0, ids.transpose(1, 2).reshape(-1), dout.view(-1, st["h"]).float())
    total *= st["scale"]
    return total if kind == "main_grad" else total.bfloat16()


# ---- what a pass cannot do without ---------------------------------------------------------------
def _blocks(r, c):
    return r * c + r * -(-c // 128)


def _distinct(c):
    """Rows of the table that a microbatch is expected to touch: ids are the cube of a uniform number times the vocabulary."""
    t, v = c["b"] * c["s"], c["vocab"]
    edges = [i / 256 for i in range(257)]
    rows = 0.0
    for lo, hi in zip(edges, edges[1:]):
        n = v * (hi - lo)
        share = (1 - c.get("skew", 0.0)) * (hi ** (1 / 3) - lo ** (1 / 3))
        rows += n * -math.expm1(-t * share / n)
    return min(rows + 1, t, v)


def work(case):
    c = case
    if c["kind"] == "product":
        return {"bytes": _blocks(c["m"], c["k"]) + _blocks(c["n"], c["k"]) + 2 * c["m"] * c["n"], "flops": 2 * c["m"] * c["n"] * c["k"]}
    if c["kind"] == "step":
        x, w, y = c["t"] * c["k"], c["n"] * c["k"], c["t"] * c["n"]
        return {"bytes": 2 * (2 * x + 2 * w + 2 * y), "flops": 6 * c["t"] * c["n"] * c["k"]}
    t = c["b"] * c["s"]
    if c["kind"] == "lookup":
        return {"bytes": 8 * t + 2 * _distinct(c) * c["h"] + 2 * t * c["h"], "flops": t * c["h"]}
    micro = c.get("micro", 1)
    return {"bytes": micro * (8 * t + 2 * t * c["h"]) + (4 if c["kind"] == "main_grad" else 2) * c["vocab"] * c["h"],
            "flops": micro * t * c["h"]}


# ---- the definition in 64 bits -------------------------------------------------------------------
def _power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_blocks(x, axis, tiles=False):
    """x in 64 bits, each block of 128 along `axis` (and along both for tiles) rounded to the multiples that e4m3 holds at its exponent."""
    x = x.double()
    size = x.abs()
    for d in ((0, 1) if tiles else (axis,)):
        size = torch.cat([p.amax(d, keepdim=True).expand_as(p) for p in size.split(128, d)], d)
    size = size.clamp(min=2.0 ** -140)
    e = torch.ceil(torch.log2(size / LARGEST))
    e = torch.where(size > LARGEST * _power(e), e + 1, e)
    e = torch.where(size <= LARGEST * _power(e - 1), e - 1, e).clamp(-127, 127)
    v = x / _power(e)
    binade = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    binade = torch.where(v.abs() < _power(binade), binade - 1, binade).clamp(min=-6)
    unit = _power(binade - 3)
    return torch.round(v / unit) * unit * _power(e)


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    if c["kind"] == "product":
        both = []
        for q, s in (st["a"], st["b"]):
            scale = _power(s[:, :q.shape[0]].double() - 127).t()
            both.append((q.double() * scale.repeat_interleave(128, 1))[:, :c["k"]].contiguous())
        return both[0] @ both[1].t()
    if c["kind"] == "step":
        w = _exact_blocks(st["w"], 1, tiles=True)
        y = _exact_blocks(st["x"], 1) @ w.t()
        dx = _exact_blocks(st["dy"], 1) @ w
        return {"y": y, "dx": dx, "dw": _exact_blocks(st["dy"], 0).t() @ _exact_blocks(st["x"], 0)}
    if c["kind"] == "lookup":
        return torch.nn.functional.embedding(st["ids"], st["table"]).double().transpose(0, 1) * c["scale"]
    total = torch.zeros(c["vocab"], c["h"], dtype=torch.float64, device="cuda")
    for ids, dout in zip(st["ids"], st["dout"]):
        total.index_put_((ids.reshape(-1),), dout.double().transpose(0, 1).reshape(-1, c["h"]) * c["scale"], accumulate=True)
    return total
