"""linear_cross_entropy - softmax cross entropy of a projection onto a vocabulary, without the
logits in memory, HIP backend.

``linear_cross_entropy_fwd(x, weight, labels, ...) -> (loss, lse, z_loss)``, three fp32
``[tokens]`` tensors: what ``cross_entropy_fwd`` (viperbench/cross_entropy) gives for
``logits = x @ weight.T`` in 32 bits, with ``x`` [tokens, hidden], ``weight`` [classes, hidden]
and one column block per row.  ``smoothing``, ``logit_scale``, ``lse_square_scale``,
``ignored_index``, ``total_classes`` (default: the rows of ``weight``), ``class_start_idx`` and
``SPLIT`` (``weight`` is a slice of the classes) are its options.  A token whose label is
``ignored_index`` takes no part: its loss, lse and z_loss are 0, whatever its ``x`` holds.

``linear_cross_entropy_bwd(dloss, x, weight, lse, labels, ...) -> (dx, dweight)``, the gradients
from the forward's inputs, its ``lse`` and the gradient of its ``loss`` (as in
``cross_entropy_bwd`` that of ``loss`` alone, z_loss included in it).  The logits are formed again
in pieces of the vocabulary; their gradients are rounded to ``x``'s dtype, summed in fp32 in a
fixed order and rounded once.  ``weight_grad=False`` leaves dweight out (None).

libvbhip ``vbh_linear_cross_entropy_fwd`` / ``_bwd``, on torch's current stream, no host
synchronisation.  No reference counterpart: the reference's nearest operator is
ViperBench/cross_entropy/pytorch_impl.py:4-141, which takes logits.
"""
import functools
import os
import sys

_ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
if _ROOT not in sys.path:
    sys.path.insert(0, _ROOT)

import torch  # noqa: E402

from dslperfgap_amd import _bridge, _lib  # noqa: E402


def _rows(t, what, name):
    """`t` as rows of contiguous values."""
    if t.dim() != 2:
        raise ValueError(f"{what}: {name} must be 2-D, got {list(t.shape)}")
    st = t.stride()
    if (st[1] != 1 and t.shape[1] > 1) or (st[0] < t.shape[1] and t.shape[0] > 1):
        return t.contiguous()
    return t


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _per_token(t, n, what, name):
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{what}: {name} must have shape [{n}], got {list(t.shape)}")
    return t


def _check(what, x, weight, labels, smoothing, logit_scale, lse_square_scale, ignored_index,
           total_classes, class_start_idx):
    """(x, weight, labels) as the entry points take them, and their arguments behind the pointers."""
    x, weight = _rows(x, what, "x"), _rows(weight, what, "weight")
    if x.shape[1] != weight.shape[1]:
        raise ValueError(f"{what}: x has {x.shape[1]} values per token, weight {weight.shape[1]}")
    if 0 in weight.shape:
        raise ValueError(f"{what}: weight is empty: {list(weight.shape)}")
    code = _bridge.float_code(x, what)
    if weight.dtype != x.dtype:
        raise TypeError(f"{what}: weight dtype {weight.dtype} must be {x.dtype}")
    _per_token(labels, x.shape[0], what, "labels")
    if labels.dtype not in _bridge.LABEL_CODES:
        if labels.dtype.is_floating_point or labels.dtype == torch.bool:
            raise TypeError(f"{what}: labels must be an integer tensor, got {labels.dtype}")
        labels = labels.to(torch.int64)
    total = weight.shape[0] if total_classes is None else int(total_classes)
    args = (x.shape[0], x.shape[1], weight.shape[0], _stride(x), _stride(weight), float(smoothing),
            float(logit_scale), float(lse_square_scale), int(ignored_index), total,
            int(class_start_idx), code, _bridge.LABEL_CODES[labels.dtype])
    return x, weight, labels.contiguous(), args


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(tokens, hidden, vocab, code, pad_weight, backward):
    return _lib.lib().vbh_linear_cross_entropy_workspace_bytes(tokens, hidden, vocab, code,
                                                               pad_weight, backward)


def _workspace(x, weight, code, backward):
    size = x.element_size()
    stride = _stride(weight) * size
    pad = (weight.data_ptr() % 16 != 0 or stride % 16 != 0 or weight.shape[1] * size % 16 != 0 or
           stride > 1 << 20)
    nbytes = _workspace_bytes(x.shape[0], x.shape[1], weight.shape[0], code, int(pad),
                              int(backward))
    return _bridge.empty(x, (nbytes,), torch.uint8), nbytes


_raw_device, _raw_stream = _bridge._raw_device, _bridge._raw_stream
# (shapes and dtypes of x, weight and labels, backward) of a call on contiguous tensors whose weight
# begins at a multiple of 16 bytes -> (tokens, hidden, classes, type codes, workspace bytes, entry
# point), or False where a call needs the general path (which raises the errors of invalid calls)
_PLANS = _bridge.PlanCache()


def _plan(xs, ws, dtype, wdtype, ls, ldtype, backward):
    code, lcode = _bridge.FLOAT_CODES.get(dtype), _bridge.LABEL_CODES.get(ldtype)
    if (code is None or lcode is None or wdtype is not dtype or len(xs) != 2 or len(ws) != 2 or
            len(ls) != 1 or xs[1] != ws[1] or ls[0] != xs[0] or 0 in xs or 0 in ws):
        return False
    pad = xs[1] * dtype.itemsize % 16 != 0
    nbytes = _workspace_bytes(xs[0], xs[1], ws[0], code, int(pad), int(backward))
    if not nbytes:
        return False
    return (xs[0], xs[1], ws[0], code, lcode, nbytes,
            _lib.entry("vbh_linear_cross_entropy_bwd" if backward else
                       "vbh_linear_cross_entropy_fwd"))


def _common(x, weight, labels, backward):
    """The plan of a common call and its device, or (None, -1)."""
    key = (x.shape, weight.shape, x.dtype, weight.dtype, labels.shape, labels.dtype, backward)
    p = _PLANS.get(key)
    if p is None:
        p = _PLANS.put(key, _plan(*key))
    if p:
        dev = x.get_device()
        if (dev >= 0 and dev == _raw_device() and weight.get_device() == dev and
                labels.get_device() == dev and x.is_contiguous() and weight.is_contiguous() and
                labels.is_contiguous() and weight.data_ptr() % 16 == 0):
            return p, dev
    return None, -1


def linear_cross_entropy_fwd(x, weight, labels, smoothing=0.0, logit_scale=1.0,
                             lse_square_scale=0.0, ignored_index=-100, total_classes=None,
                             class_start_idx=0, SPLIT=False):
    """Per-token loss, lse and z_loss of x @ weight.T against labels; see the module docstring."""
    p, dev = _common(x, weight, labels, False)
    if p is not None:
        tokens, hidden, vocab, code, lcode, nbytes, fn = p
        loss = x.new_empty_strided((tokens,), (1,), dtype=torch.float32)
        lse, z_loss = torch.empty_like(loss), torch.empty_like(loss)
        ws = x.new_empty_strided((nbytes,), (1,), dtype=torch.uint8)
        rc = fn(x.data_ptr(), weight.data_ptr(), labels.data_ptr(), loss.data_ptr(),
                lse.data_ptr(), z_loss.data_ptr(), tokens, hidden, vocab, hidden, hidden,
                float(smoothing), float(logit_scale), float(lse_square_scale),
                int(ignored_index), vocab if total_classes is None else int(total_classes),
                int(class_start_idx), code, lcode, int(bool(SPLIT)), ws.data_ptr(), nbytes,
                _raw_stream(dev))
        if rc != 0:
            raise _lib.VbhError("vbh_linear_cross_entropy_fwd", rc, _lib.last_error())
        return loss, lse, z_loss
    what = "linear_cross_entropy_fwd"
    x, weight, labels, args = _check(what, x, weight, labels, smoothing, logit_scale,
                                     lse_square_scale, ignored_index, total_classes,
                                     class_start_idx)
    dev = _bridge.require_gpu(what, x, weight, labels)
    loss, lse, z_loss = (_bridge.empty(x, (x.shape[0],), torch.float32) for _ in range(3))
    ws, nbytes = _workspace(x, weight, args[-2], False)
    _bridge.launch("vbh_linear_cross_entropy_fwd", dev, x.data_ptr(), weight.data_ptr(),
                   labels.data_ptr(), loss.data_ptr(), lse.data_ptr(), z_loss.data_ptr(), *args,
                   int(bool(SPLIT)), ws.data_ptr(), nbytes)
    return loss, lse, z_loss


def linear_cross_entropy_bwd(dloss, x, weight, lse, labels, smoothing=0.0, logit_scale=1.0,
                             lse_square_scale=0.0, ignored_index=-100, total_classes=None,
                             class_start_idx=0, weight_grad=True):
    """The gradients of linear_cross_entropy_fwd's x and weight from that of its loss."""
    f32 = torch.float32
    if (dloss.dtype is f32 and lse.dtype is f32 and dloss.shape == labels.shape and
            lse.shape == labels.shape):
        p, dev = _common(x, weight, labels, True)
        if (p is not None and dloss.get_device() == dev and lse.get_device() == dev and
                dloss.is_contiguous() and lse.is_contiguous()):
            tokens, hidden, vocab, code, lcode, nbytes, fn = p
            dx = torch.empty_like(x)
            dw = torch.empty_like(weight) if weight_grad else None
            ws = x.new_empty_strided((nbytes,), (1,), dtype=torch.uint8)
            rc = fn(dloss.data_ptr(), x.data_ptr(), weight.data_ptr(), lse.data_ptr(),
                    labels.data_ptr(), dx.data_ptr(), dw.data_ptr() if weight_grad else None,
                    tokens, hidden, vocab, hidden, hidden, float(smoothing), float(logit_scale),
                    float(lse_square_scale), int(ignored_index),
                    vocab if total_classes is None else int(total_classes), int(class_start_idx),
                    code, lcode, ws.data_ptr(), nbytes, _raw_stream(dev))
            if rc != 0:
                raise _lib.VbhError("vbh_linear_cross_entropy_bwd", rc, _lib.last_error())
            return dx, dw
    what = "linear_cross_entropy_bwd"
    x, weight, labels, args = _check(what, x, weight, labels, smoothing, logit_scale,
                                     lse_square_scale, ignored_index, total_classes,
                                     class_start_idx)
    for t, name in ((dloss, "dloss"), (lse, "lse")):
        _per_token(t, x.shape[0], what, name)
        if not t.dtype.is_floating_point:
            raise TypeError(f"{what}: {name} must be a float tensor, got {t.dtype}")
    dev = _bridge.require_gpu(what, dloss, x, weight, lse, labels)
    dloss, lse = (t.to(torch.float32).contiguous() for t in (dloss, lse))
    dx = _bridge.empty(x, x.shape)
    dw = _bridge.empty(weight, weight.shape) if weight_grad else None
    ws, nbytes = _workspace(x, weight, args[-2], True)
    _bridge.launch("vbh_linear_cross_entropy_bwd", dev, dloss.data_ptr(), x.data_ptr(),
                   weight.data_ptr(), lse.data_ptr(), labels.data_ptr(), dx.data_ptr(),
                   _bridge.ptr(dw), *args, ws.data_ptr(), nbytes)
    return dx, dw
