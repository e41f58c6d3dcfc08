"""Offsets that pass 32 bits: operands, results and gradients of more than 2^31 elements, looked at in rows on both sides."""

import pytest
import torch

from kareus_amd import BlockOperand
from kareus_amd.backend import get_backend

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]


@pytest.fixture(autouse=True)
def give_memory_back():
    """(Nothing that outlives a test is put into the large pieces that these leave in the allocator.)"""
    yield
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


def needs(gb):
    if torch.cuda.mem_get_info()[0] < gb << 30:
        pytest.skip(f"needs {gb} GB")


def test_quantises_more_than_2_31_elements():
    """36000 x 65536, both ways: the blocks of rows and columns at the ends are those of the same rows and columns alone."""
    needs(24)
    be = get_backend("hip")
    r, c = 36000, 65536
    x = torch.empty(r, c, dtype=torch.bfloat16, device="cuda")
    x.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    got = be.quantize_blocks(x, True, True)
    for lo, hi in ((0, 128), (32640, 32896), (35968, 36000)):
        part = be.quantize_blocks(x[lo:hi].contiguous()).by_row
        assert torch.equal(got.by_row.data[lo:hi].view(torch.uint8), part.data.view(torch.uint8))
        assert torch.equal(got.by_row.scales[:, lo:hi], part.scales[:, :hi - lo])
    for lo in (0, 32768, 65408):
        part = be.quantize_blocks(x[:, lo:lo + 128].contiguous(), False, True).by_col
        assert torch.equal(got.by_col.data[lo:lo + 128].view(torch.uint8), part.data.view(torch.uint8))
        assert torch.equal(got.by_col.scales[:, lo:lo + 128], part.scales[:, :128])


def whole(rows, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    data = torch.randint(0, 2, (rows, k), generator=g, device="cuda", dtype=torch.uint8).mul_(0x38).view(torch.float8_e4m3fn)   # 0 and 1
    return BlockOperand(data, torch.full((k // 128, (rows + 3) // 4 * 4), 127, dtype=torch.uint8, device="cuda"), k)


def values(t, lo, hi):
    return t.data[lo:hi].float()


@pytest.mark.parametrize("m,n,k", [(40000, 264, 65536), (264, 40000, 65536), (300000, 8192, 256), (8192, 300000, 256)])
def test_product_of_more_than_2_31_elements(m, n, k):
    """Zeros and ones: every sum is a whole number below 2^24."""
    needs(24)
    be = get_backend("hip")
    a, b = whole(m, k, 1), whole(n, k, 2)
    for got in (be.block_matmul(a, b), be.block_matmul_segments([BlockOperand(a.data[:, :128], a.scales[:1], 128), BlockOperand(a.data[:, 128:], a.scales[1:], k - 128)],
                                                                [BlockOperand(b.data[:, :128], b.scales[:1], 128), BlockOperand(b.data[:, 128:], b.scales[1:], k - 128)])):
        for rows in ((0, 8), (m // 2 - 3, m // 2 + 5), (m - 9, m)):
            for cols in ((0, 8), (n // 2 - 3, n // 2 + 5), (n - 9, n)):
                want = values(a, *rows) @ values(b, *cols).t()
                assert torch.equal(got[rows[0]:rows[1], cols[0]:cols[1]], want.bfloat16())
        del got


def test_embedding_of_more_than_2_31_elements():
    """600000 tokens of 4096: lookups and the gradient of rows whose tokens lie at both ends."""
    needs(32)
    be = get_backend("hip")
    b, s, h, rows = 4, 150000, 4096, 5000
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, rows, (b, s), generator=g, device="cuda")
    table = torch.empty(rows, h, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    out = be.embedding_fwd(ids, table, scale=8.0)
    for t in (0, 74999, 131072, 149999):
        assert torch.equal(out[t], (table[ids[:, t]].float() * 8).bfloat16())
    dw = be.embedding_bwd_sorted(ids, out, rows, scale=0.5, out=torch.empty(rows, h, device="cuda"))
    flat = out.view(-1, h)
    for r in (0, 2500, 4999):
        at = (ids.t().reshape(-1) == r).nonzero()[:, 0]
        want, mags = flat[at].double().sum(0) * 0.5, flat[at].double().abs().sum(0) * 0.5
        assert ((dw[r].double() - want).abs() <= mags * (len(at) + 2) * 2.0 ** -24).all()
