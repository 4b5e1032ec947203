"""ViperBench/layer_norm - HIP backend.

Unified API of ViperBench/layer_norm/pytorch_impl.py:5-12:
``layer_norm(x, weight, bias, eps=1e-5) -> Tensor`` = F.layer_norm over the
trailing ``weight.shape`` dims, same shape and dtype as ``x``.

One read of x and one write of y per call (libvbhip ``vbh_layer_norm_fwd``);
launched on torch's current stream, no host synchronisation.

``layer_norm_bwd(dy, x, weight, bias, eps=1e-5) -> (dx, dweight, dbias)``, its gradients
from the forward's inputs and the gradient of its output: two reads and one write of the
rows (``vbh_layer_norm_bwd``).  No reference counterpart (its layer_norm is forward only).
"""
import os
import sys

_ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
if _ROOT not in sys.path:  # loadable by file path, as ViperBench's harness loads impls
    sys.path.insert(0, _ROOT)

import torch  # noqa: E402

from dslperfgap_amd import _bridge, _lib, _norm_bwd  # noqa: E402


def layer_norm(x, weight, bias, eps=1e-5):
    """Unified API: layer_norm(x, weight, bias, eps) -> Tensor.

    Like the reference golden, eps other than 1e-5 raises ValueError
    (ViperBench/layer_norm/pytorch_impl.py:9-11).
    """
    if eps != 1e-5:
        raise ValueError(f"Only eps=1e-5 is supported (got {eps}). "
                         "The Triton kernel hardcodes eps=1e-5.")
    # the common call: contiguous x, weight and bias of one dtype on the current
    # GPU, normalized over the last dim -- straight to the row kernel
    dt = x.dtype
    if bias is not None and weight.dtype is dt and bias.dtype is dt:
        key = (x.shape, weight.shape, bias.shape, dt)
        p = _PLANS.get(key)
        if p is None:
            p = _PLANS.put(key, _plan(x, weight, bias))
        if p:
            dev = x.get_device()
            if (dev >= 0 and dev == _raw_device() and weight.get_device() == dev and
                    bias.get_device() == dev and x.is_contiguous() and
                    weight.is_contiguous() and bias.is_contiguous()):
                rows, cols, code, fn = p
                y = torch.empty_like(x)
                rc = fn(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), y.data_ptr(), rows,
                        cols, 1e-5, code, code, _raw_stream(dev))
                if rc != 0:
                    raise _lib.VbhError("vbh_layer_norm_fwd", rc, _lib.last_error())
                return y
    dev = _bridge.require_gpu("layer_norm", x, weight, bias)
    norm_shape = tuple(weight.shape)
    k = len(norm_shape)
    if tuple(x.shape[x.dim() - k:]) != norm_shape or x.dim() < k:
        raise RuntimeError(f"layer_norm: normalized_shape {list(norm_shape)} does not match "
                           f"the trailing dims of input {list(x.shape)}")
    if bias is not None and tuple(bias.shape) != norm_shape:
        raise RuntimeError(f"layer_norm: bias shape {list(bias.shape)} != {list(norm_shape)}")
    dt = _bridge.float_code(x, "layer_norm")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"layer_norm: weight dtype {weight.dtype} must be {x.dtype} or float32")
    if bias is not None and bias.dtype != weight.dtype:
        raise TypeError("layer_norm: weight and bias dtypes differ")
    wdt = _bridge.FLOAT_CODES[weight.dtype]
    cols = _bridge.numel_prod(norm_shape)
    x = x.contiguous()
    w = weight.contiguous()
    b = bias.contiguous() if bias is not None else None
    y = torch.empty_like(x)
    rows = x.numel() // cols if cols else 0
    _bridge.launch("vbh_layer_norm_fwd", dev, _bridge.ptr(x), _bridge.ptr(w), _bridge.ptr(b),
                   _bridge.ptr(y), rows, cols, float(eps), dt, wdt)
    return y


# (x shape, weight shape, bias shape, dtype) -> (rows, cols, dtype code, entry
# point) of a last-dim LayerNorm with weight and bias of x's dtype, or False
_PLANS = _bridge.PlanCache()
_raw_device, _raw_stream = _bridge._raw_device, _bridge._raw_stream


def _plan(x, weight, bias):
    code = _bridge.FLOAT_CODES.get(x.dtype)
    if (code is None or x.dim() == 0 or weight.dim() != 1 or
            x.shape[-1] != weight.shape[0] or bias.shape != weight.shape):
        return False
    cols = weight.shape[0]
    return (x.numel() // cols if cols else 0, cols, code, _lib.entry("vbh_layer_norm_fwd"))


def layer_norm_bwd(dy, x, weight, bias, eps=1e-5):
    """The gradients of layer_norm's x, weight and bias from that of its output (x's shape
    and dtype).  ``bias`` is only asked whether there is one: its gradient is None without.
    The weights' gradients are summed in fp32 in a fixed order and have the weights' dtype.
    """
    if eps != 1e-5:
        raise ValueError(f"Only eps=1e-5 is supported (got {eps}). "
                         "The Triton kernel hardcodes eps=1e-5.")
    got = _norm_bwd.common(dy, x, weight, bias, 1e-5, True)
    if got is not None:
        return got
    what = "layer_norm_bwd"
    norm_shape = tuple(weight.shape)
    k = len(norm_shape)
    if x.dim() < k or tuple(x.shape[x.dim() - k:]) != norm_shape:
        raise RuntimeError(f"{what}: normalized_shape {list(norm_shape)} does not match "
                           f"the trailing dims of input {list(x.shape)}")
    if bias is not None:
        if bias.shape != weight.shape:
            raise RuntimeError(f"{what}: bias shape {list(bias.shape)} != {list(norm_shape)}")
        if bias.dtype != weight.dtype:
            raise TypeError(f"{what}: weight and bias dtypes differ")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"{what}: weight dtype {weight.dtype} must be {x.dtype} or float32")
    dev, dx, dw, args = _norm_bwd.prepare(what, dy, x, weight, bias, eps, True)
    db = None if bias is None else _bridge.empty(weight, weight.shape)
    dy, x, weight, rest = args
    _bridge.launch("vbh_layer_norm_bwd", dev, dy.data_ptr(), x.data_ptr(), weight.data_ptr(),
                   dx.data_ptr(), dw.data_ptr(), _bridge.ptr(db), *rest)
    return dx, dw, db
