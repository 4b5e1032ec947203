"""The rotation of queries and keys and the per-head RMSNorm ahead of it, in 64 bits on CPU
torch, with the bounds their 32-bit evaluation is held to.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  The reference has no such operator: the
functions here follow the definition (pair by pair, position by position), and are pinned
by complex multiplication, by automatic differentiation and by differences
(tests/test_rope_api.py).  Tensors are [batch, tokens, heads, head_dim].
"""
from __future__ import annotations

import math

import torch

ULP = 2.0 ** -24  # half a step of a 32-bit rounding, relative


def axis_of(sections, order):
    """The position axis of each frequency."""
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections[1:]), []
    for p in range(sum(sections)):
        a = p % len(sections)
        if a > 0 and left[a - 1] > 0:
            left[a - 1] -= 1
            out.append(a)
        else:
            out.append(0)
    return out


def angles(positions, inv_freq, lead, sections=None, order="blocks"):
    """[batch, tokens, n_freq] angles of positions as the operators take them."""
    n = inv_freq.shape[0]
    sections = (n,) if sections is None else tuple(sections)
    pos = positions.double()
    if len(sections) == 1:
        pos = pos[None]
    pos = (pos if pos.dim() == 3 else pos[:, None, :]).expand(len(sections), *lead)
    cols = [pos[a] * float(inv_freq[p]) for p, a in enumerate(axis_of(sections, order))]
    return torch.stack(cols, -1)


def pairs(n, pairing):
    """The two values of each of n pairs."""
    if pairing == "half":
        return list(range(n)), list(range(n, 2 * n))
    return list(range(0, 2 * n, 2)), list(range(1, 2 * n, 2))


def turn(x, theta, pairing, scale=1.0, back=False, size=False):
    """x turned by theta [batch, tokens, n] (`back`: by the transpose); with `size` the sums
    of the magnitudes that enter each value instead."""
    first, second = pairs(theta.shape[-1], pairing)
    c, s = torch.cos(theta)[:, :, None], torch.sin(theta)[:, :, None]
    if back:
        s = -s
    a, b = x[..., first], x[..., second]
    out = x.abs() if size else x.clone()
    if size:
        out[..., first] = out[..., second] = abs(scale) * (a.abs() + b.abs())
    else:
        out[..., first] = scale * (a * c - b * s)
        out[..., second] = scale * (b * c + a * s)
    return out


def rms(x, eps):
    return 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)


def subnormal(x, eps):
    """Relative error that 1 / sqrt(mean + eps) has beyond that: where the squares lie below
    2^-126, each of the D additions and the product with 1 / D round by up to 2^-150, which
    is 2^-149 of the mean of D squares; the root halves it."""
    return 2.0 ** -150 / ((x * x).mean(-1, keepdim=True) + eps)


def forward(x, theta, pairing, scale=1.0, weight=None, eps=None):
    """One side's output and the bound of a 32-bit evaluation's error.  `eps` None: no norm.

    Norm: the sum of D squares is a chain of at most 16 per lane and a tree of 6 (relative
    error 22 steps, halved by the root), 1 / sqrt 2 steps, the products with the weight and
    with cos and sin 2, and cos and sin themselves are within 3 steps of 1; the two
    products and their sum 2: 22 / 2 + 2 + 2 + 3 + 2 = 20 steps of the magnitudes.  Without
    the norm 8."""
    x = x.double()
    more = 0.0
    if eps is not None:
        more = subnormal(x, eps)
        x = x * rms(x, eps)
        if weight is not None:
            x = x * weight.double()
    steps = 8 if eps is None else 20
    return (turn(x, theta, pairing, scale),
            (steps * ULP + more) * turn(x, theta, pairing, scale, size=True))


def backward(dy, x, theta, pairing, scale, weight, eps):
    """(dx, dweight) of one side, and the bounds of their errors.

    dn is within 8 steps of its magnitudes G; dx = r (dn w - u m), u = x r, m =
    mean(dn w u): r within 13 steps, the sum of m 22 more, the products 2 each, so that
    80 steps of r (G |w| + |u| mean(G |w| |u|)) hold all.  The weight's gradient adds N
    terms of G |u|, each within 8 + 13 + 2 steps, in chains of fewer than 400 + N / 256
    additions: a lane adds N / 256 at most where both sides' passes together are no more
    than 5 times this side's heads (4096 waves, a side's in proportion to its passes + 2
    per share), the sums of its workgroup and of the rows fewer than 400."""
    dy, x = dy.double(), x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    dn = turn(dy, theta, pairing, scale, back=True)
    size = turn(dy, theta, pairing, scale, back=True, size=True)
    r = rms(x, eps)
    u = x * r
    dx = r * (dn * w - u * (dn * w * u).mean(-1, keepdim=True))
    reach = (size * w.abs() * u.abs()).mean(-1, keepdim=True)
    more = subnormal(x, eps)  # r enters three times
    dx_bound = (80 * ULP + 3 * more) * r * (size * w.abs() + u.abs() * reach)
    terms = (dn * u).flatten(0, 2)
    sizes = (size * u.abs() * (1 + more / ULP)).flatten(0, 2)
    steps = 423 + terms.shape[0] / 256
    return dx, terms.sum(0), dx_bound, steps * ULP * sizes.sum(0)


def rounded(bound, value, dtype):
    """`bound` and the rounding of the result to `dtype`: half a step, and half the smallest
    subnormal number."""
    if dtype == torch.float32:
        return bound + 2.0 ** -126
    f = torch.finfo(dtype)
    return bound * (1 + f.eps) + f.eps / 2 * value.abs() + f.tiny * f.eps / 2


def inv_freq(n, base=10000.0, dtype=torch.float32):
    return torch.tensor([math.pow(base, -i / n) for i in range(n)], dtype=torch.float64).to(dtype)
