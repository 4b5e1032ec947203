"""Host side of the norms' gradients (``viperbench/layer_norm``, ``viperbench/rms_norm``): what
both check and allocate."""
from __future__ import annotations

import functools

import torch

from . import _bridge, _lib


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, cols: int, dtype: int, layer_norm: bool) -> int:
    return _lib.lib().vbh_norm_bwd_workspace_bytes(rows, cols, dtype, int(layer_norm))


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
