"""Norm and rotation of heads in 64 bits: the oracle of the CUDA kernel.

Test infrastructure only, from the operator's definition.
"""

from __future__ import annotations

import torch


def rotate(x, positions, frequencies, *, weight=None, eps=1e-6, rotary_start=0, interleaved=False, amplitude=1.0):
    """(the heads normed and rotated, the magnitudes that each element is made of), float64."""
    y = x.double().clone()
    if weight is not None:
        n = weight.numel()
        y[..., :n] = y[..., :n] / torch.sqrt((y[..., :n] ** 2).mean(-1, keepdim=True) + eps) * weight.double()
    size = y.abs()
    pairs = frequencies.numel()
    i = torch.arange(pairs, device=x.device)
    a, b = (rotary_start + 2 * i, rotary_start + 2 * i + 1) if interleaved else (rotary_start + i, rotary_start + pairs + i)
    angle = (positions.double()[:, None] * frequencies.double())[:, None]
    ya, yb = y[..., a].clone(), y[..., b].clone()
    y[..., a] = amplitude * (ya * torch.cos(angle) - yb * torch.sin(angle))
    y[..., b] = amplitude * (yb * torch.cos(angle) + ya * torch.sin(angle))
    size[..., a] = size[..., b] = abs(amplitude) * (ya.abs() + yb.abs())
    return y, size
