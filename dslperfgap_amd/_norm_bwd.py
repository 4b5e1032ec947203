"""Host side of the norms' gradients (``viperbench/layer_norm``, ``viperbench/rms_norm``): what
both check and allocate."""
from __future__ import annotations

import functools

import torch

from . import _bridge, _lib


MOST_EPS = torch.finfo(torch.float32).max  # eps is taken in 32 bits


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, cols: int, dtype: int, layer_norm: bool) -> int:
    return _lib.lib().vbh_norm_bwd_workspace_bytes(rows, cols, dtype, int(layer_norm))


_raw_device, _raw_stream = _bridge._raw_device, _bridge._raw_stream
# (x shape, dtype, weight shape, dtype, LayerNorm) of a call over the trailing weight.shape dims of
# contiguous tensors -> (rows, cols, dtype codes, workspace bytes, entry point), or False
_PLANS = _bridge.PlanCache()


def _plan(xs, dtype, ws, wdtype, layer_norm):
    code = _bridge.FLOAT_CODES.get(dtype)
    k = len(ws)
    cols = _bridge.numel_prod(ws)
    if (code is None or wdtype not in (dtype, torch.float32) or len(xs) < k or cols == 0 or
            xs[len(xs) - k:] != ws or 0 in xs):
        return False
    rows = _bridge.numel_prod(xs) // cols
    nbytes = _workspace_bytes(rows, cols, code, layer_norm)
    name = "vbh_layer_norm_bwd" if layer_norm else "vbh_rms_norm_bwd"
    return (rows, cols, code, _bridge.FLOAT_CODES[wdtype], nbytes, name, _lib.entry(name))


def common(dy, x, weight, bias, eps, layer_norm):
    """(dx, dweight, dbias) of the common call, straight to the entry point: contiguous tensors on
    the current GPU, normalized over the trailing weight.shape dims; None where the call needs the
    general path, which raises the errors of invalid calls."""
    key = (x.shape, x.dtype, weight.shape, weight.dtype, layer_norm)
    p = _PLANS.get(key)
    if p is None:
        p = _PLANS.put(key, _plan(*key))
    if not p or dy.shape != x.shape or dy.dtype is not x.dtype:
        return None
    dev = x.get_device()
    if not (dev >= 0 and dev == _raw_device() and dy.get_device() == dev and
            weight.get_device() == dev and x.is_contiguous() and dy.is_contiguous() and
            weight.is_contiguous()):
        return None
    if bias is not None and (bias.shape != weight.shape or bias.dtype is not weight.dtype or
                             bias.get_device() != dev):
        return None
    rows, cols, code, wcode, nbytes, name, fn = p
    dx, dw = torch.empty_like(x), torch.empty_like(weight)
    ws = x.new_empty_strided((nbytes,), (1,), dtype=torch.uint8)
    if layer_norm:
        db = torch.empty_like(weight) if bias is not None else None
        rc = fn(dy.data_ptr(), x.data_ptr(), weight.data_ptr(), dx.data_ptr(), dw.data_ptr(),
                db.data_ptr() if bias is not None else None, rows, cols, eps, code, wcode,
                ws.data_ptr(), nbytes, _raw_stream(dev))
    else:
        db = None
        rc = fn(dy.data_ptr(), x.data_ptr(), weight.data_ptr(), dx.data_ptr(), dw.data_ptr(), rows,
                cols, eps, code, wcode, ws.data_ptr(), nbytes, _raw_stream(dev))
    if rc != 0:
        raise _lib.VbhError(name, rc, _lib.last_error())
    return dx, dw, db


def prepare(what, dy, x, weight, bias, eps, layer_norm):
    """(device, dx, dweight, (dy, x, weight, the entry point's arguments behind the outputs)) of
    a call whose x and weight fit each other; dy is checked against x here."""
    if dy.shape != x.shape:
        raise ValueError(f"{what}: dy must have shape {list(x.shape)}, got {list(dy.shape)}")
    if dy.dtype != x.dtype:
        raise TypeError(f"{what}: dy dtype {dy.dtype} must be {x.dtype}")
    code = _bridge.float_code(x, what)
    wcode = _bridge.float_code(weight, what)
    dev = _bridge.require_gpu(what, dy, x, weight, bias)
    dy, x, weight = dy.contiguous(), x.contiguous(), weight.contiguous()
    cols = weight.numel()
    rows = x.numel() // cols if cols else 0
    dx, dw = torch.empty_like(x), torch.empty_like(weight)
    nbytes = _workspace_bytes(rows, cols, code, layer_norm)
    ws = _bridge.empty(x, (nbytes,), torch.uint8)
    return dev, dx, dw, (dy, x, weight, (rows, cols, float(eps), code, wcode, ws.data_ptr(),
                                         nbytes))
