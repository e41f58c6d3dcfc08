"""The end of a training step: the 2-norm of the gradients that one process holds and clipping by it, the local part of
3rdparty/Megatron-LM/megatron/core/optimizer/clip_grads.py (``get_grad_norm_fp32``, ``clip_grad_by_total_norm_fp32``).

Nothing here is reduced over ranks.  Where a model's gradients are split over processes, ``clip_grad_norm`` on each would scale each by a
factor of its own: take ``grad_norm`` of each part (those that every rank holds counted once), add the squares over the ranks, and scale
by the factor of that sum."""

from __future__ import annotations

from typing import Iterable, List, Optional, Sequence, Union

import torch
from torch import Tensor


def gradients_of(parameters: Union[Tensor, Iterable[torch.nn.Parameter]]) -> List[Tensor]:
    """The gradients that there are, one for each parameter object: its ``main_grad``, or where it keeps none its ``grad``.  One that has
    both raises: which of them a step goes by is not for this function to say."""
    found, seen = [], set()
    for p in [parameters] if isinstance(parameters, Tensor) else parameters:    # (of a tensor alone the rows would be gone through)
        if id(p) in seen:
            continue
        seen.add(id(p))
        main = getattr(p, "main_grad", None)
        if main is not None and p.grad is not None:
            raise RuntimeError("a parameter has a main_grad and a grad")
        g = main if main is not None else p.grad
        if g is not None:
            found.append(g)
    return found


def grad_norm(parameters: Union[Tensor, Iterable[torch.nn.Parameter]], backend: str = "hip") -> Tensor:
    """The 2-norm of all these gradients as one vector, fp32 on their device; nothing waits for it.  Of this process alone: the squares of
    several shards' norms are the caller's to add."""
    from .backend import get_backend

    return get_backend(backend).grad_norm(gradients_of(parameters))


def clip_grad_norm(parameters: Union[Tensor, Iterable[torch.nn.Parameter]], max_norm: float, eps: float = 1e-6, backend: str = "hip",
                   out: Optional[Sequence[Tensor]] = None) -> Tensor:
    """Scales all these gradients by ``min(1, max_norm / (norm + eps))`` and returns their norm before that, fp32 on their device; nothing
    waits for it.  The norm is that of these gradients: nothing is reduced over ranks.  ``out``: fp32 tensors, one for each gradient in
    order, that receive the scaled gradients (an optimizer's own), and the gradients stay as they are."""
    from .backend import get_backend

    return get_backend(backend).clip_grad_norm(gradients_of(parameters), max_norm, eps=eps, out=out)


def _layout(t: Tensor):
    return [(n, st) for n, st in zip(t.shape, t.stride()) if n != 1]


def _dense(t: Tensor) -> bool:
    """Whether the elements lie one behind the other, in any order."""
    end = 1
    for n, st in sorted(_layout(t), key=lambda d: d[1]):
        if st != end:
            return False
        end *= n
    return True


def check_gradients(tensors: List[Tensor], max_norm: float = 0.0, eps: float = 0.0, out=None) -> None:
    """Raises unless these are gradients that a norm can be taken of: dense bf16 or fp32 tensors on one device, none of them
    overlapping another or an output."""
    if not max_norm >= 0.0 or not eps >= 0.0:
        raise RuntimeError(f"clip_grad_norm: max_norm {max_norm} and eps {eps} must not be negative")
    if out is not None and len(out) != len(tensors):
        raise RuntimeError(f"clip_grad_norm: {len(out)} outputs for {len(tensors)} gradients")
    places = []
    for t in tensors if out is None else [*tensors, *out]:
        if t.device != tensors[0].device:
            raise RuntimeError(f"gradients on {tensors[0].device} and {t.device}")
        if t.dtype not in (torch.bfloat16, torch.float32):
            raise RuntimeError(f"a gradient is bf16 or fp32, got {t.dtype}")
        if t.layout != torch.strided or not (t.numel() == 0 or _dense(t)):
            raise RuntimeError(f"a gradient has to be dense, got {tuple(t.shape)} with strides {tuple(t.stride()) if t.layout == torch.strided else t.layout}")
        if t.numel():
            places.append((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()))
    for t, to in zip(tensors, out or ()):
        if to.dtype != torch.float32 or to.shape != t.shape or (t.numel() and _layout(to) != _layout(t)):
            raise RuntimeError(f"clip_grad_norm: an output must be fp32 with the shape and strides of its gradient, {tuple(t.shape)} "
                               f"{tuple(t.stride())}, got {to.dtype} {tuple(to.shape)} {tuple(to.stride())}")
    places.sort()
    for a, b in zip(places, places[1:]):
        if a[1] > b[0]:
            raise RuntimeError("a gradient appears twice or overlaps another tensor of the call")
