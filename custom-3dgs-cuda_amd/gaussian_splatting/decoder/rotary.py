"""Rotary positions with several axes (view or time, row, column of a patch; x, y, z of a
point), for queries and keys of images, video and scenes."""

from __future__ import annotations

from typing import Sequence

import torch as t

from gaussian_splatting.decoder._ext import module


def axis_frequencies(sections: Sequence[int], base: float = 10000.0, device=None) -> t.Tensor:
    """inv_freq of ``rotary_axes`` with a ladder of its own for each axis: the i-th of an
    axis's n pairs turns by base^(-i / n) per unit of position (fp32, formed in 64 bits)."""
    ladders = [base ** (-t.arange(n, dtype=t.float64) / n) for n in sections if n > 0]
    inv = t.cat(ladders) if ladders else t.empty(0, dtype=t.float64)
    return inv.to(t.float32).to(device)


def rotary_axes(x: t.Tensor, positions: t.Tensor, inv_freq: t.Tensor, sections: Sequence[int], *,
                interleaved: bool = False) -> t.Tensor:
    """Turns pairs of channels by their token's position.

    Args:
        x: (B, L, H, D) fp32, bf16 or fp16, any strides (a slice of a packed projection
            is read in place)
        positions: (L, A) or (B, L, A), float32, int32 or int64
        inv_freq: (P,) fp32, radians per unit of position of each pair
        sections: how many of the P pairs each of the A axes turns, in order; 2 P <= D
        interleaved: pairs are channels (2i, 2i + 1) instead of (i, i + P)

    Returns:
        (B, L, H, D) contiguous; channels from 2 P on are x's.  Differentiable in x;
        positions and inv_freq are data, and raise where a gradient would be wanted.
    """
    if t.is_grad_enabled() and (positions.requires_grad or inv_freq.requires_grad):
        raise ValueError("rotary_axes forms no gradient for positions or inv_freq: detach them")
    return module().decoder_rotary(x, positions, inv_freq, list(sections), interleaved)
