"""Matrices held in 8-bit blocks: e4m3 values with one power-of-two scale per block of 128 along the contraction.

What the reference's linear layers reach through TransformerEngine's quantizers (``quantizer`` / ``with_quantized_compute`` arguments,
kareus/transformer_engine/pytorch/ops/basic/basic_linear.py:391-604); the block layout here is this package's own."""

from __future__ import annotations

from typing import NamedTuple, Optional

from torch import Tensor

#: contraction elements that share a scale
BLOCK = 128
#: largest magnitude of e4m3: a block's scale brings its largest value to this or below
E4M3_MAX = 448.0


def blocks_of(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


class BlockOperand(NamedTuple):
    """One operand of a block product, ``rows`` vectors of ``length`` contraction elements.

    ``data`` ``[rows, pitch]`` float8_e4m3fn, contiguous along the contraction, ``pitch`` a multiple of 16 and at least ``length``
    rounded up to a multiple of 128; the values from ``length`` to that multiple are read and have to be zero.
    ``scales`` ``[blocks, >= rows]`` uint8, a row per block of 128 contraction elements; the value of an element is
    ``data * 2^(scale - 127)``.  Any rows of an operand are one, ``data[i:j]`` and ``scales[:, i:j]``; scales that do not begin at a
    multiple of 4 bytes, are not a multiple of 4 apart or end with their storage within one are copied for a product."""

    data: Tensor
    scales: Tensor
    length: int

    @property
    def rows(self) -> int:
        return self.data.shape[0]


class BlockScaled(NamedTuple):
    """A matrix ``[r, c]`` in 8-bit blocks, in the orientations that were asked for: ``by_row`` holds its rows (a contraction over the
    columns), ``by_col`` its columns (a contraction over the rows)."""

    by_row: Optional[BlockOperand]
    by_col: Optional[BlockOperand]
