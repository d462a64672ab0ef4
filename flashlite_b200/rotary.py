"""Rotary positions: the table of cosines and sines, and the autograd wrapper.

``rotary_table`` makes the fp32 table that ``flash_attn_wmma.rotary``,
``rotary_backward`` and ``rotary_append`` read, once per model;
``rotary_embedding(q, k, table, ...)`` is the differentiable form, to be put
before ``flashlite_b200.attention.flash_attention``. No reference counterpart:
the reference has no positions.
"""
from __future__ import annotations

import math

import torch

from .flash_attn_wmma import rotary, rotary_backward


def rotary_table(positions: int, rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 original: int = 0, fast: float = 32.0, slow: float = 1.0, device="cuda") -> torch.Tensor:
    """``[positions, rot_dim]`` fp32: ``rot_dim/2`` cosines, then as many sines.

    Pair ``j`` turns by ``position * base**(-2j/rot_dim)``. For contexts
    ``factor`` times longer than trained on, ``scaling``:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"ntk"``: ``base`` times ``factor**(rot_dim / (rot_dim - 2))``, which leaves
      the fastest pair as it is and divides the slowest by ``factor``;
    * ``"by_parts"``: pairs that turn more than ``fast`` times over the
      ``original`` context keep their frequency, those that turn less than
      ``slow`` times have it divided by ``factor``, a linear ramp lies between;
      cosines and sines are scaled by ``0.1 ln(factor) + 1``, which sharpens the
      softmax of the longer context.

    Angles, cosines and sines are computed in 64 bits and rounded once: at
    position 10**6 a 32-bit angle would be off by several hundredths.
    """
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError("rot_dim must be an even number, at least 2")
    if positions < 0:
        raise ValueError("positions must not be negative")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError("base must be above 1 and factor at least 1")
    scale = 1.0
    if scaling == "ntk":
        if rot_dim < 4:
            raise ValueError("ntk scaling needs rot_dim of at least 4")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = float(base) ** (torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / -rot_dim)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "by_parts":
        if original <= 0 or not fast > slow:
            raise ValueError("by_parts scaling needs the original context length, and fast above slow")
        turns = freq * (original / (2.0 * math.pi))
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        freq = keep * freq + (1.0 - keep) * (freq / factor)
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in ("none", "ntk"):
        raise ValueError("scaling must be 'none', 'linear', 'ntk' or 'by_parts'")
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), freq)
    return torch.cat((angle.cos(), angle.sin()), dim=1).mul_(scale).float()


class _Rotary(torch.autograd.Function):
    """Rotation, or with ``inverse`` its gradient. The rotation is linear, so that each is the other's gradient, and
    gradients of any order are the same two calls."""

    @staticmethod
    def forward(ctx, q, k, table, positions, interleaved, layout, inverse):
        ctx.save_for_backward(table, positions)
        ctx.interleaved, ctx.layout, ctx.inverse = interleaved, layout, inverse
        return (rotary_backward if inverse else rotary)(q, k, table, positions, interleaved, layout)

    @staticmethod
    def backward(ctx, dq, dk):
        table, positions = ctx.saved_tensors
        dq, dk = (d if d is None or d.stride(-1) == 1 else d.contiguous() for d in (dq, dk))
        dq, dk = _Rotary.apply(dq, dk, table, positions, ctx.interleaved, ctx.layout, not ctx.inverse)
        return dq, dk, None, None, None, None, None


def rotary_embedding(q: torch.Tensor, k: torch.Tensor | None, table: torch.Tensor, positions: torch.Tensor | None = None,
                     interleaved: bool = False, layout: str = "bhnd") -> tuple[torch.Tensor, torch.Tensor | None]:
    """Differentiable (any order) ``rotary(q, k, table, positions)``; ``layout`` defaults to that of
    ``flash_attention``. The table gets no gradient: one that asks for it is refused."""
    if table.requires_grad and torch.is_grad_enabled():
        raise ValueError("rotary_embedding has no gradient of the table: pass table.detach()")
    return _Rotary.apply(q, k, table, positions, interleaved, layout, False)
