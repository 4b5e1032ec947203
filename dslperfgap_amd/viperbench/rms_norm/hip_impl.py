"""ViperBench/rms_norm - HIP backend.

Unified API of ViperBench/rms_norm/pytorch_impl.py:3-10:
``rms_norm(x, normalized_shape, weight, eps=1e-5) -> Tensor``, reducing over
the last ``len(normalized_shape)`` dims:
``((x.float() / sqrt(mean(x.float()**2) + eps)) * weight.float()).to(x.dtype)``.

One read of x and one write of y per call (libvbhip ``vbh_rms_norm_fwd``).

``rms_norm_bwd(dy, x, normalized_shape, weight, eps=1e-5) -> (dx, dweight)``, its gradients
from the forward's inputs and the gradient of its output: two reads and one write of the
rows (``vbh_rms_norm_bwd``).  No reference counterpart (its rms_norm is forward only).
"""
import os
import sys

_ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
if _ROOT not in sys.path:
    sys.path.insert(0, _ROOT)

import torch  # noqa: E402

from dslperfgap_amd import _bridge, _lib, _norm_bwd  # noqa: E402


def rms_norm(x, normalized_shape, weight, eps=1e-5):
    """RMS normalization: y = x / sqrt(mean(x^2) + eps) * weight."""
    # the common call: contiguous x and weight (of x's dtype or fp32) on the
    # current GPU, normalized over the last dim
    if type(normalized_shape) is tuple and len(normalized_shape) == 1:
        key = (x.shape, x.dtype, weight.shape, weight.dtype)
        p = _PLANS.get(key)
        if p is None:
            p = _PLANS.put(key, _plan(*key))
        if p:
            dev = x.get_device()
            if (dev >= 0 and dev == _raw_device() and weight.get_device() == dev and
                    x.is_contiguous() and weight.is_contiguous()):
                rows, cols, code, wcode, fn = p
                y = torch.empty_like(x)
                rc = fn(x.data_ptr(), weight.data_ptr(), y.data_ptr(), rows, cols, float(eps),
                        code, wcode, _raw_stream(dev))
                if rc != 0:
                    raise _lib.VbhError("vbh_rms_norm_fwd", rc, _lib.last_error())
                return y
    dev = _bridge.require_gpu("rms_norm", x, weight)
    k = len(tuple(normalized_shape))
    if k > x.dim():
        raise RuntimeError(f"rms_norm: normalized_shape {tuple(normalized_shape)} has more dims "
                           f"than input {list(x.shape)}")
    dt = _bridge.float_code(x, "rms_norm")
    cols = x.shape[-1] if k == 1 else _bridge.numel_prod(x.shape[x.dim() - k:])
    if weight.numel() != cols:
        raise RuntimeError(f"rms_norm: weight has {weight.numel()} elements, the normalized "
                           f"dims hold {cols}")
    # weight.float() in the golden: any float weight is exact in fp32; keep the
    # x dtype when it matches (no extra pass), else widen the small vector once
    w = weight.contiguous() if weight.dtype in (x.dtype, torch.float32) else weight.float()
    wdt = _bridge.FLOAT_CODES[w.dtype]
    x = x.contiguous()
    y = torch.empty_like(x)
    rows = x.numel() // cols if cols else 0
    _bridge.launch("vbh_rms_norm_fwd", dev, _bridge.ptr(x), _bridge.ptr(w), _bridge.ptr(y), rows,
                   cols, float(eps), dt, wdt)
    return y


# (x shape, dtype, weight shape, dtype) -> (rows, cols, dtype codes, entry point) of
# a last-dim RMSNorm, or False where a call needs the general path
_PLANS = _bridge.PlanCache()
_raw_device, _raw_stream = _bridge._raw_device, _bridge._raw_stream


def _plan(shape, dtype, wshape, wdtype):
    code = _bridge.FLOAT_CODES.get(dtype)
    if (code is None or len(shape) == 0 or wdtype not in (dtype, torch.float32) or
            _bridge.numel_prod(wshape) != shape[-1] or shape[-1] == 0):
        return False
    cols = int(shape[-1])
    return (_bridge.numel_prod(shape) // cols, cols, code, _bridge.FLOAT_CODES[wdtype],
            _lib.entry("vbh_rms_norm_fwd"))


def rms_norm_bwd(dy, x, normalized_shape, weight, eps=1e-5):
    """The gradients of rms_norm's x and weight from that of its output (x's shape and
    dtype).  The weight's gradient is summed in fp32 in a fixed order and has the weight's
    shape and dtype."""
    what = "rms_norm_bwd"
    if not 0.0 <= float(eps) <= _norm_bwd.MOST_EPS:
        raise ValueError(f"{what}: eps must be finite in 32 bits and not negative, got {eps}")
    if tuple(normalized_shape) == tuple(weight.shape):
        got = _norm_bwd.common(dy, x, weight, None, float(eps), False)
        if got is not None:
            return got[:2]
    k = len(tuple(normalized_shape))
    if k > x.dim():
        raise RuntimeError(f"{what}: normalized_shape {tuple(normalized_shape)} has more dims "
                           f"than input {list(x.shape)}")
    cols = _bridge.numel_prod(x.shape[x.dim() - k:])
    if weight.numel() != cols:
        raise RuntimeError(f"{what}: weight has {weight.numel()} elements, the normalized "
                           f"dims hold {cols}")
    wide = weight.dtype in (x.dtype, torch.float32)
    dev, dx, dw, args = _norm_bwd.prepare(what, dy, x, weight if wide else weight.float(), None,
                                          eps, False)
    dy, x, w, rest = args
    _bridge.launch("vbh_rms_norm_bwd", dev, dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                   dx.data_ptr(), dw.data_ptr(), *rest)
    return dx, dw if wide else dw.to(weight.dtype)
