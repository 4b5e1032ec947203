"""Softmax cross entropy of a projection onto a vocabulary, and its gradients, in 64 bits, with the
bounds their evaluation in 32 bits (and, backward, with the logits' gradients rounded to the
inputs' type) is held to.  On whatever device the tensors are.

TEST INFRASTRUCTURE ONLY (see oracle/__init__.py).  The reference has no such operator: its
cross_entropy takes logits.  Pinned by oracle/pytorch_impl.cross_entropy_fwd / _bwd, automatic
differentiation and differences (tests/test_linear_ce_api.py).
"""
from __future__ import annotations

import torch

from .rope import ULP, rounded  # noqa: F401  (rounded: for the callers)


def _product_steps(n, dtype):
    """Roundings in a sum of n products on the matrix cores: they add 16 products of 16-bit values
    (exact in fp32), or 2 of fp32, to a sum at a time, with up to 5 roundings inside; each of
    those may cut off rather than round, hence twice."""
    return 2 * (n / (2 if dtype == torch.float32 else 16) + 5)


def _logits(x, w, scale):
    """(scaled logits, how far fp32 may be off)."""
    xd, wd = x.double(), w.double()
    logits = scale * torch.matmul(xd, wd.T)
    size = abs(scale) * torch.matmul(xd.abs(), wd.abs().T)
    return logits, (_product_steps(x.shape[1], x.dtype) * size + logits.abs()) * ULP


def _parts(x, labels, ignored):
    keep = labels.long() != ignored
    return keep, torch.where(keep[:, None], x.double(), 0.0).to(x.dtype)


def _target(logits, labels, smoothing, total, start):
    """The smoothed label distribution on this slice of the classes, and whether it has the label."""
    local = labels.long() - start
    hit = (local >= 0) & (local < logits.shape[1])
    target = torch.full_like(logits, smoothing / total)
    rows = hit.nonzero()[:, 0]
    target[rows, local[rows]] += 1.0 - smoothing
    return target, hit


def forward(x, w, labels, smoothing=0.0, logit_scale=1.0, lse_square_scale=0.0, ignored_index=-100,
            total_classes=None, class_start_idx=0, split=False):
    """([loss, lse, z_loss], their bounds).

    A logsumexp is off by as much as its logits at most, by the roundings of its sum (a lane adds
    64 exponentials, 8 blocks, 2 halves and up to 4 waves join, then every 32nd tile, then 32 of
    those: relative errors of the sum are absolute ones of its log) and by those of the
    exponentials, whose arguments the logarithm of the classes' number bounds on average."""
    total = w.shape[0] if total_classes is None else total_classes
    keep, x = _parts(x, labels, ignored_index)
    logits, off = _logits(x, w, logit_scale)
    target, hit = _target(logits, labels, smoothing, total, class_start_idx)
    lse = torch.logsumexp(logits, 1)
    n = w.shape[0]
    off_lse = off.max(1).values + (200 + n / 4096 + 2 * lse.abs()) * ULP
    base = torch.zeros_like(lse) if split else lse
    z = torch.zeros_like(lse) if split else lse_square_scale * lse * lse
    off_z = 0.0 if split else abs(lse_square_scale) * 2 * lse.abs() * off_lse + 4 * z.abs() * ULP
    loss = torch.where(hit, base - (target * logits).sum(1),
                       smoothing * (base - logits.sum(1) / total))
    steps = 200 + n / 4096
    off_loss = (off_lse + (target * (off + steps * ULP * logits.abs())).sum(1) +
                8 * ULP * (lse.abs() + (target * logits).abs().sum(1)))
    out = [torch.where(keep, t, 0.0) for t in (loss + z, lse, z)]
    bounds = [torch.where(keep, t + torch.zeros_like(lse), 0.0)
              for t in (off_loss + off_z + 2 * ULP * loss.abs(), off_lse, off_z)]
    return out, bounds


def backward(dloss, x, w, lse, labels, smoothing=0.0, logit_scale=1.0, lse_square_scale=0.0,
             ignored_index=-100, total_classes=None, class_start_idx=0):
    """([dx, dw], their bounds), `lse` taken as it is.

    p = exp(L - lse) is off, relatively, by L's error and the exponential's (its argument's
    rounding and 4 of its own); dL then meets a rounding to the inputs' type, which for fp16 has
    a smallest step 2^-34 of the largest possible dL (for dx: of the token's own, whatever the
    others' losses weigh); the products add as in the logits."""
    total = w.shape[0] if total_classes is None else total_classes
    keep, x = _parts(x, labels, ignored_index)
    logits, off = _logits(x, w, logit_scale)
    target, _ = _target(logits, labels, smoothing, total, class_start_idx)
    lse = lse.double()[:, None]
    scale = torch.where(keep, dloss.double() * logit_scale, 0.0)[:, None]
    f = 1.0 + 2.0 * lse_square_scale * lse
    arg = logits - lse
    p = arg.exp() * f
    d = scale * (p - target)
    off_d = scale.abs() * (p.abs() * (off + (arg.abs() + 8) * ULP) + 4 * ULP * target)
    if x.dtype != torch.float32:
        off_d = off_d * 1.01 + torch.finfo(x.dtype).eps / 2 * d.abs()
    off_x = off_w = off_d
    if x.dtype == torch.float16:
        step = 2.0 ** -34 * scale.abs() * (abs(1 - smoothing) + abs(smoothing) / total + f.abs())
        off_x, off_w = off_d + step, off_d + step.max()
    off_x, off_w = (torch.where(keep[:, None], t, 0.0) for t in (off_x, off_w))
    xd, wd = x.double(), w.double()
    wide = _product_steps(w.shape[0], x.dtype) + w.shape[0] / 1024
    deep = _product_steps(x.shape[0], x.dtype)
    out = [torch.matmul(d, wd), torch.matmul(d.T, xd)]
    bounds = [torch.matmul(off_x + wide * ULP * (d.abs() + off_x), wd.abs()),
              torch.matmul((off_w + deep * ULP * (d.abs() + off_w)).T, xd.abs())]
    return out, bounds
