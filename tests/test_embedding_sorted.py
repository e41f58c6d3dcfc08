"""The scaled token embedding and its gradient by sorted tokens against the definition in 64 bits: ids of other shards, ids that fill
the batch, rows without a token, whole and accumulated gradients; refusals."""

import pytest
import torch

from kareus_amd.backend import get_backend

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]


def on_gpu(f):
    for m in gpu:
        f = m(f)
    return f


def ids_of(kind, b, s, rows, start, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        ids = torch.randint(start, start + rows, (b, s), generator=g)
    elif kind == "text":
        u = torch.rand(b, s, generator=g)
        ids = start + (u ** 3 * rows).long().clamp_(max=rows - 1)
    elif kind == "one":
        ids = torch.full((b, s), start + rows - 1)
    elif kind == "padded":
        ids = torch.randint(start, start + rows, (b, s), generator=g)
        ids[torch.rand(b, s, generator=g) < 0.7] = start
    else:                                                   # "shards": most ids belong to others, negative ones among them
        ids = torch.randint(start - 2 * rows, start + 3 * rows, (b, s), generator=g)
    return ids


def data(b, s, h, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(s, b, h, generator=g).bfloat16()


def definition(ids, dout, rows, start, scale):
    """(gradient in 64 bits, sum of magnitudes and number of tokens of each row)."""
    rel = (ids - start).t().reshape(-1)
    keep = (rel >= 0) & (rel < rows)
    flat = dout.reshape(-1, dout.shape[-1]).double()[keep]
    z = lambda *n: torch.zeros(*n, dtype=torch.float64, device=dout.device)  # noqa: E731
    total = z(rows, dout.shape[-1]).index_add_(0, rel[keep], flat) * scale
    mags = z(rows, dout.shape[-1]).index_add_(0, rel[keep], flat.abs()) * abs(scale)
    return total, mags, torch.bincount(rel[keep], minlength=rows)


def check(be, device, kind, b, s, h, rows, start, scale, out=None, accumulate=False):
    ids, dout = ids_of(kind, b, s, rows, start).to(device), data(b, s, h).to(device)
    want, mags, count = definition(ids, dout, rows, start, scale)
    before = None if out is None else out.double().clone()
    old = None if out is None else out.clone()
    got = be.embedding_bwd_sorted(ids, dout, rows, vocab_start=start, scale=scale, out=out, accumulate=accumulate)
    assert got.shape == (rows, h) and (out is None or got is out)
    if accumulate:
        assert torch.equal(got[count == 0], old[count == 0])     # rows without a token are left alone
        want = want + before
        mags = mags + before.abs()
    else:
        assert not got[count == 0].any()
    # fp32 sums of n terms, the product with the factor and the sum with what is there: (n + 2) roundings of half a step each, at most
    # of all the magnitudes; then the store's
    bound = mags * ((count + 2)[:, None] * 2.0 ** -24)
    if got.dtype == torch.bfloat16:
        bound = bound + want.abs() * 2.0 ** -8
    err = (got.double() - want).abs()
    assert (err <= bound * 1.001 + 1e-300).all(), (err / bound.clamp_min(1e-300)).max().item()
    return got


CASES = [("uniform", 1, 1, 8, 1, 0), ("uniform", 2, 3, 64, 7, 5), ("text", 2, 100, 520, 1000, 0), ("one", 3, 57, 72, 9, 100),
         ("padded", 4, 700, 1032, 4096, 0), ("shards", 2, 1000, 256, 300, 700), ("uniform", 1, 2048, 64, 511, 0),
         ("uniform", 1, 2049, 64, 512, 0), ("text", 2, 4099, 640, 32064, 32064), ("one", 8, 2500, 264, 3, 1), ("shards", 1, 4097, 128, 300000, 7),
         ("padded", 8, 2007, 512, 128256, 0)]


@pytest.mark.parametrize("kind,b,s,h,rows,start", CASES)
def test_eager_gradient(kind, b, s, h, rows, start):
    if b * s * h > 1 << 21:
        pytest.skip("on the device only")
    check(get_backend("eager"), "cpu", kind, b, s, h, rows, start, 8.0)


@pytest.mark.parametrize("kind,b,s,h,rows,start", CASES)
@on_gpu
def test_gradient(kind, b, s, h, rows, start):
    be = get_backend("hip")
    first = check(be, "cuda", kind, b, s, h, rows, start, 8.0)
    assert torch.equal(first, check(be, "cuda", kind, b, s, h, rows, start, 8.0))       # the same bits every time
    check(be, "cuda", kind, b, s, h, rows, start, 0.3, out=torch.full((rows, h), float("nan"), device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,b,s,h,rows,start", CASES)
@on_gpu
def test_gradient_added_to_what_is_there(kind, b, s, h, rows, start, dtype):
    g = torch.Generator().manual_seed(4)
    out = (10 * torch.randn(rows, h, generator=g)).to("cuda", dtype)
    check(get_backend("hip"), "cuda", kind, b, s, h, rows, start, 1.5, out=out, accumulate=True)


@on_gpu
def test_gradient_of_many_tokens():
    check(get_backend("hip"), "cuda", "text", 8, 16384, 64, 151936, 0, 1.0)
    check(get_backend("hip"), "cuda", "one", 8, 16384, 64, 1000, 0, 1.0)


@on_gpu
def test_gradient_of_a_strided_upstream_gradient_and_ids():
    be = get_backend("hip")
    b, s, h, rows = 3, 100, 72, 50
    ids, dout = ids_of("uniform", b, s, rows, 0).cuda(), data(b, s, h).cuda()
    plain = be.embedding_bwd_sorted(ids, dout, rows)
    wide = torch.zeros(s, b, 2 * h, dtype=torch.bfloat16, device="cuda")
    wide[..., :h] = dout
    assert torch.equal(be.embedding_bwd_sorted(ids.t().contiguous().t(), wide[..., :h], rows), plain)


@on_gpu
def test_the_same_bits_beside_other_work_and_in_a_graph():
    be = get_backend("hip")
    b, s, h, rows = 2, 3000, 512, 5000
    sets = [(ids_of(k, b, s, rows, 0, i).cuda(), data(b, s, h, i).cuda()) for i, k in enumerate(("text", "padded", "uniform"))]
    want = [be.embedding_bwd_sorted(*x, rows, scale=2.0) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st, x in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(be.embedding_bwd_sorted(*x, rows, scale=2.0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    held = [(i.clone(), d.clone()) for i, d in sets[:2]]
    main = torch.zeros(rows, h, device="cuda")
    graphs, outs = [], []
    for x in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(be.embedding_bwd_sorted(*x, rows, scale=2.0))
            be.embedding_bwd_sorted(*x, rows, scale=2.0, out=main, accumulate=True)
        graphs.append(graph)
    for r in range(4):
        for i in range(2):
            held[i][0].copy_(sets[(i + r) % 3][0])
            held[i][1].copy_(sets[(i + r) % 3][1])
        main.zero_()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        total = torch.zeros(rows, h, device="cuda")
        for i in range(2):
            assert torch.equal(outs[i], want[(i + r) % 3])
            be.embedding_bwd_sorted(*sets[(i + r) % 3], rows, scale=2.0, out=total, accumulate=True)
        assert torch.equal(main, total)


@pytest.mark.parametrize("b,s,h,rows,start", [(1, 1, 8, 1, 0), (3, 37, 520, 100, 50), (2, 4096, 1032, 32064, 0), (8, 64, 16384, 500, 0)])
@pytest.mark.parametrize("kind", ["uniform", "shards"])
@on_gpu
def test_scaled_lookup(kind, b, s, h, rows, start):
    be = get_backend("hip")
    ids, table = ids_of(kind, b, s, rows, start).cuda(), data(1, rows, h, 7)[:, 0].contiguous().cuda()
    got = be.embedding_fwd(ids, table, start, scale=45.25)
    rel = ids - start
    mine = (rel >= 0) & (rel < rows)
    want = torch.where(mine[..., None], table[rel.clamp(0, rows - 1)].double() * 45.25, 0.0).transpose(0, 1)
    assert torch.equal(got, want.to(torch.bfloat16))           # one rounding of an exact product
    assert torch.equal(be.embedding_fwd(ids, table, start, scale=1.0), be.embedding_fwd(ids, table, start))


@on_gpu
def test_lookup_of_a_row_that_is_not_finite():
    be = get_backend("hip")
    table = torch.zeros(4, 8, dtype=torch.bfloat16, device="cuda")
    table[0], table[1] = float("nan"), float("inf")
    got = be.embedding_fwd(torch.tensor([[0, 1, 2, -1, 4]], device="cuda"), table, scale=2.0)[:, 0]
    assert got[0].isnan().all() and (got[1] == float("inf")).all() and not got[2:].any()


def test_library_refuses_before_anything_is_launched():
    from kareus_amd.backend import hip

    lib = hip.load_library()
    ok = [16, 16, 16, 0, 4, 2, 64, 0, 100, 1.0, 0, 16, 1 << 20]
    for at, bad, rc in ((0, None, -1), (1, None, -1), (1, 8, -1), (2, None, -1), (2, 8, -1), (4, 0, -1), (5, 0, -1), (6, 0, -1), (6, 60, -2),
                        (8, 0, -1), (8, 1 << 27, -2), (4, 1 << 26, -2), (11, None, -1), (11, 8, -1), (12, 16, -1)):
        args = list(ok)
        args[at] = bad
        assert lib.kr_embedding_bwd_sorted(*args, None) == rc, (at, bad)
    assert lib.kr_embedding_bwd_sorted_workspace_bytes(0, 2, 64, 100) == 0
    assert lib.kr_embedding_bwd_sorted_workspace_bytes(1 << 26, 2, 64, 100) == 0
    assert lib.kr_embedding_bwd_sorted_workspace_bytes(4, 2, 64, 1 << 27) == 0
    ok = [16, 16, 16, 4, 2, 64, 0, 100, 2.0]
    for at, bad, rc in ((0, None, -1), (1, None, -1), (1, 8, -1), (2, 8, -1), (3, 0, -1), (5, 60, -2), (7, 0, -1)):
        args = list(ok)
        args[at] = bad
        assert lib.kr_embedding_fwd_scaled(*args, None) == rc, (at, bad)


def test_backend_refuses_host_tensors():
    be = get_backend("hip")
    ids, dout = torch.zeros(1, 2, dtype=torch.int64), torch.zeros(2, 1, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="HIP device"):
        be.embedding_bwd_sorted(ids, dout, 4)
    with pytest.raises(RuntimeError, match="HIP device"):
        be.embedding_fwd(ids, dout[:, 0], scale=2.0)


@on_gpu
def test_backend_refuses_on_the_device():
    be = get_backend("hip")
    ids, dout = torch.zeros(1, 2, dtype=torch.int64, device="cuda"), torch.zeros(2, 1, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="int64"):
        be.embedding_bwd_sorted(ids.int(), dout, 4)
    with pytest.raises(RuntimeError, match="bf16"):
        be.embedding_bwd_sorted(ids, dout.float(), 4)
    with pytest.raises(RuntimeError, match="must be"):
        be.embedding_bwd_sorted(ids, dout.transpose(0, 1), 4)
    with pytest.raises(RuntimeError, match="out must be"):
        be.embedding_bwd_sorted(ids, dout, 4, out=torch.zeros(5, 8, device="cuda"))
    with pytest.raises(RuntimeError, match="accumulate"):
        be.embedding_bwd_sorted(ids, dout, 4, accumulate=True)
    with pytest.raises(RuntimeError, match="kr_embedding_bwd_sorted"):
        be.embedding_bwd_sorted(ids, dout[..., :4].contiguous(), 4)
    with pytest.raises(RuntimeError, match="dense"):
        be.embedding_fwd(ids, torch.zeros(4, 16, dtype=torch.bfloat16, device="cuda")[:, :8], scale=2.0)
    # nothing to add: the gradient is zero, or what was there
    none = torch.zeros(1, 0, dtype=torch.int64, device="cuda")
    assert not be.embedding_bwd_sorted(none, dout[:0], 4).any()
    kept = torch.ones(4, 8, device="cuda")
    assert (be.embedding_bwd_sorted(none, dout[:0], 4, out=kept, accumulate=True) == 1).all()
