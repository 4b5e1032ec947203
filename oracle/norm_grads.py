"""The gradients of LayerNorm and RMSNorm over the last axis, in 64 bits on CPU torch, with the
bounds their 32-bit evaluation is held to.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  The reference's norms are forward only: the
functions here follow the definition and are pinned by automatic differentiation and by
differences (tests/test_norm_bwd_api.py).
"""
from __future__ import annotations

import torch

from .rope import ULP, rounded  # noqa: F401  (rounded: for the callers)

# Roundings that one value of a row meets, and sums of a row: a lane adds up to 32 values one
# after the other, in each of up to 4 accesses, then come 6 steps in a wave and 16 waves.
STEPS = 64


def backward(dy, x, w, eps, layer_norm):
    """([dx, dw, db or None], their bounds) of [rows, cols] tensors of any type.

    With X = |x| + mean |x| a value x - mean is off by STEPS ULP X; so is u = (x - mean) r by that
    times r, and r itself, relatively, by STEPS ULP (1 + mean(X^2) r^2), as a sum of squares of
    values that are that far off.  Every term of dx is a product of such values; a sum over rows
    adds one rounding a row for the rows that one lane adds up (the 256th part of all, at least
    one), and the steps that join the lanes.
    """
    x, dy, w = x.double(), dy.double(), w.double()
    rows = x.shape[0]
    mean = x.mean(1, keepdim=True) if layer_norm else torch.zeros(rows, 1, dtype=torch.float64)
    d = x - mean
    r = 1.0 / (d.square().mean(1, keepdim=True) + eps).sqrt()
    u, g = d * r, dy * w
    dx = g - u * (g * u).mean(1, keepdim=True)
    size = x.abs() + (x.abs().mean(1, keepdim=True) if layer_norm else 0.0)
    big = size * r
    bound = g.abs() + big * (g.abs() * big).mean(1, keepdim=True)
    if layer_norm:
        dx = dx - g.mean(1, keepdim=True)
        bound = bound + g.abs().mean(1, keepdim=True)
    spread = 1.0 + big.square().mean(1, keepdim=True)
    bound = STEPS * ULP * r * bound * spread
    lane = STEPS + rows / 256
    out = [r * dx, (dy * u).sum(0), dy.sum(0) if layer_norm else None]
    bounds = [bound, lane * ULP * (dy.abs() * big * spread).sum(0),
              lane * ULP * dy.abs().sum(0) if layer_norm else None]
    return out, bounds
