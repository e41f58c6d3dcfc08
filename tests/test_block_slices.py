"""Rows of a larger operand in 8-bit blocks as an operand: one block and several, scales that begin and end anywhere."""

import pytest
import torch

from kareus_amd import BlockOperand
from kareus_amd.backend import get_backend
from kareus_amd.block_scaled import blocks_of

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a HIP device")]


def operand(rows, k, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, blocks_of(k) * 128, generator=g)
    x[:, k:] = 0
    return get_backend("hip").quantize_blocks(x.to("cuda", torch.bfloat16)).by_row._replace(length=k)


@pytest.mark.parametrize("k", [1, 100, 128, 129, 200, 1000])
@pytest.mark.parametrize("start,rows", [(0, 130), (132, 130), (130, 130), (133, 1), (4, 3), (1, 9), (255, 7)])
def test_rows_of_a_larger_operand(k, start, rows):
    be = get_backend("hip")
    a, b = operand(262, k, 1), operand(272, k, 2)
    whole = be.block_matmul(a, b)
    part = BlockOperand(a.data[start:start + rows], a.scales[:, start:start + rows], k)
    few = be.block_matmul(part, b)
    # (fewer rows may be cut or added up otherwise: two sums of the same products, a bf16 step at most, and their fp32 orders)
    tol = 2.0 ** -7 * whole[start:start + rows].float().abs() + 1e-4 * k ** 0.5
    assert ((few.float() - whole[start:start + rows].float()).abs() <= tol).all()
    dense = BlockOperand(part.data.clone(), torch.nn.functional.pad(part.scales, (0, -rows % 4)).contiguous(), k)
    assert torch.equal(few, be.block_matmul(dense, b))
    cols = start // 8 * 8
    other = BlockOperand(b.data[cols:cols + 16], b.scales[:, cols:cols + 16], k)
    assert torch.equal(be.block_matmul(part, other), be.block_matmul(dense, BlockOperand(other.data.clone(), other.scales.contiguous(), k)))
    # over pairs, the same two twice
    assert torch.equal(be.block_matmul_segments([part, part], [other, other]),
                       be.block_matmul_segments([dense, dense], [other._replace(data=other.data.clone(), scales=other.scales.contiguous())] * 2))


@pytest.mark.parametrize("k", [128, 300])
def test_scales_that_end_with_their_storage(k):
    """130 rows' scales, 132 apart, in a storage that holds not a byte behind the last; scales 130 apart; one block's for all blocks."""
    be = get_backend("hip")
    a, b = operand(130, k, 1), operand(72, k, 2)
    want, nb = be.block_matmul(a, b), blocks_of(k)
    tight = torch.empty((nb - 1) * 132 + 130, dtype=torch.uint8, device="cuda").as_strided((nb, 130), (132, 1))
    tight.copy_(a.scales[:, :130])
    assert torch.equal(be.block_matmul(a._replace(scales=tight), b), want)
    assert torch.equal(be.block_matmul(a._replace(scales=a.scales[:, :130].contiguous()), b), want)
    first = a._replace(scales=a.scales[:1].expand(nb, -1))
    assert torch.equal(be.block_matmul(first, b), be.block_matmul(first._replace(scales=first.scales.contiguous()), b))


def test_a_single_row_of_any_stride():
    be = get_backend("hip")
    a, b = operand(5, 256, 1), operand(72, 256, 2)
    row = torch.empty(256 + 7, dtype=torch.float8_e4m3fn, device="cuda")[:256].as_strided((1, 256), (7, 1))
    row.copy_(a.data[3:4])
    assert torch.equal(be.block_matmul(BlockOperand(row, a.scales[:, 3:4], 256), b), be.block_matmul(a, b)[3:4])
