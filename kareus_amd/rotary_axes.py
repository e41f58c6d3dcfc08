"""Rotary positions on several axes: a token has a place in time, height and width (text: the same on all), and each frequency of a head
turns by the place on one of them.

What Megatron's multimodal rotary embedding makes a table of angles for, ``[s, b, 1, hd]`` from ``position_ids [axes, b, s]`` and a
``mrope_section``; here the positions themselves go to the kernels."""

from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence, Tuple

import torch
from torch import Tensor

#: axes that the kernels take (KR_ROPE_MAX_AXES)
MAX_AXES = 4


class RotaryAxes(NamedTuple):
    """``positions`` ``[axes, b, s]`` int64; ``inv_freq`` ``[hd / 2]`` float64, in radians per position; ``sections``: how many of the
    frequencies each axis has, ``hd / 2`` in all.  They lie one axis behind the other, or ``interleaved``: in turn while an axis has any
    left, and the first axis has what is behind that, also where an axis gets fewer than its section for want of turns (layers refuse
    such sections).  Angles are formed in 64 bits."""

    positions: Tensor
    inv_freq: Tensor
    sections: Tuple[int, ...]
    interleaved: bool = False

    def sequences(self, lo: int, hi: int) -> "RotaryAxes":
        """The positions of sequences ``lo`` to ``hi`` of the batch (a view)."""
        return self._replace(positions=self.positions[:, lo:hi])

    def version(self) -> Optional[int]:
        """Counts the writes to the positions (None: such a tensor does not)."""
        return None if self.positions.is_inference() else self.positions._version

    def check(self, s: int, b: int, hd: int) -> None:
        """Raises unless these are the positions of ``[s, b]`` tokens with heads of ``hd`` channels."""
        p, f = self.positions, self.inv_freq
        if p.dim() != 3 or p.dtype != torch.int64 or tuple(p.shape[1:]) != (b, s) or not 1 <= p.shape[0] <= MAX_AXES:
            raise RuntimeError(f"rotary positions must be int64 [1 to {MAX_AXES} axes, {b}, {s}], got {p.dtype} {tuple(p.shape)}")
        if f.dtype != torch.float64 or tuple(f.shape) != (hd // 2,) or not f.is_contiguous():
            raise RuntimeError(f"inv_freq must be dense float64 [{hd // 2}], got {f.dtype} {tuple(f.shape)}")
        check_sections(self.sections, hd)
        if len(self.sections) != p.shape[0]:
            raise RuntimeError(f"{len(self.sections)} sections for positions on {p.shape[0]} axes")
        if p.device != f.device:
            raise RuntimeError(f"rotary positions on {p.device}, inv_freq on {f.device}")


def check_sections(sections: Sequence[int], hd: int) -> None:
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0 or sum(sections) != hd // 2:
        raise RuntimeError(f"sections {tuple(sections)} are not the {hd // 2} frequencies of {hd} channels on 1 to {MAX_AXES} axes")


def check_sections_in_turn(sections: Sequence[int]) -> None:
    """Raises unless frequencies dealt in turn give every axis as many as its section says: of 64, (4, 28, 32) would become 22, 21 and 21."""
    axes = _axes(sections, True)
    dealt = tuple(axes.count(a) for a in range(len(sections)))
    if dealt != tuple(sections):
        raise RuntimeError(f"sections {tuple(sections)} cannot be had in turn: the axes would get {dealt} frequencies")


def _axes(sections: Sequence[int], interleaved: bool) -> List[int]:
    n = len(sections)
    if interleaved:
        return [i % n if i // n < sections[i % n] else 0 for i in range(sum(sections))]
    return [a for a, size in enumerate(sections) for _ in range(size)]


def axis_of_frequency(sections: Sequence[int], interleaved: bool, device=None) -> Tensor:
    """The axis of each frequency, ``[hd / 2]`` int64."""
    return torch.tensor(_axes(sections, interleaved), dtype=torch.int64, device=device)


def rotary_axes(positions: Tensor, dim: int, sections: Sequence[int], base: float = 10000.0, interleaved: bool = False,
                inv_freq: Optional[Tensor] = None) -> RotaryAxes:
    """Positions ``[axes, b, s]`` with frequencies ``base^(-2i / dim)`` (or the given ones), in 64 bits."""
    check_sections(sections, dim)
    if inv_freq is None:
        inv_freq = inverse_frequencies(dim, base, positions.device)
    return RotaryAxes(positions, inv_freq, tuple(int(n) for n in sections), bool(interleaved))


def inverse_frequencies(dim: int, base: float, device=None) -> Tensor:
    return (base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).to(device)
