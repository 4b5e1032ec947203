"""Host side of the query / key operators (``viperbench/rope``, ``viperbench/qk_norm_rope``):
the checks of their arguments and the descriptors of their launches, cached by what
decides them.

Options are plain numbers when a plan is looked up by them (values that only equal such
are refused first); every other rule is checked where a plan is made, without a GPU, and a
call with tensors the plan knows goes straight to the entry point.
"""
from __future__ import annotations

import ctypes
import math
import numbers

import torch

from . import _bridge, _lib

POSITION_CODES = {torch.int32: _lib.I32, torch.int64: _lib.I64, torch.float32: _lib.F32}
ORDERS = {"blocks": _lib.ROPE_BLOCKS, "cycle": _lib.ROPE_CYCLE}
PAIRINGS = {"half": _lib.ROPE_HALF, "adjacent": _lib.ROPE_ADJACENT}

_raw_device, _raw_stream = _bridge._raw_device, _bridge._raw_stream
# what decides a call (shapes, strides, dtypes, options) -> its plan (make_plan)
_PLANS = _bridge.PlanCache()


def _strides(t):
    st = t.stride()
    return st[:3] if len(st) == 4 else (0, *st[:2])


def _check_pair(q, k, what, names, like=None):
    for t, name in zip((q, k), names):
        if t.dim() not in (3, 4):
            raise ValueError(f"{what}: {name} must be [tokens, heads, head_dim] or [batch, tokens, "
                             f"heads, head_dim], got {list(t.shape)}")
        _bridge.float_code(t, what)
        if t.dtype != q.dtype:
            raise TypeError(f"{what}: {names[0]} and {names[1]} dtypes differ")
    if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"{what}: {names[0]} {list(q.shape)} and {names[1]} {list(k.shape)} must "
                         "have the same tokens and head_dim")
    if like is not None:
        for t, x, name in zip((q, k), like, names):
            if t.shape != x.shape:
                raise ValueError(f"{what}: {name} must have shape {list(x.shape)}, got "
                                 f"{list(t.shape)}")
            if t.dtype != x.dtype:
                raise TypeError(f"{what}: {name} must be {x.dtype}, got {t.dtype}")


def _position_strides(positions, lead, axes, what):
    """(axis, batch, token) strides of the positions of [batch, tokens] = `lead`."""
    if positions.dtype not in POSITION_CODES:
        raise TypeError(f"{what}: positions must be int32, int64 or float32, got "
                        f"{positions.dtype}")
    shape, st = tuple(positions.shape), positions.stride()
    axis = 0
    if axes > 1:
        if not shape or shape[0] != axes:
            raise ValueError(f"{what}: positions of {axes} axes must have shape [{axes}, ...], "
                             f"got {list(shape)}")
        axis, shape, st = st[0], shape[1:], st[1:]
    if shape == lead:
        return (axis, 0, st[0]) if len(lead) == 1 else (axis, *st)
    if shape == lead[1:] and len(lead) == 2:  # one row for the whole batch
        return (axis, 0, st[0])
    front = f"{axes}, " if axes > 1 else ""
    want = " or ".join(f"[{front}{', '.join(map(str, s))}]" for s in {lead, lead[-1:]})
    raise ValueError(f"{what}: positions must have shape {want}, got {list(positions.shape)}")


def _number(what, value, name):
    """An option as a float."""
    if not isinstance(value, numbers.Real):
        raise TypeError(f"{what}: {name} must be a number, got {type(value).__name__}")
    return float(value)


def _sections(what, sections):
    """Sections as a tuple of ints."""
    if not (isinstance(sections, (tuple, list)) and
            all(isinstance(s, numbers.Integral) for s in sections)):
        raise TypeError(f"{what}: sections must be a tuple or list of integers, got {sections!r}")
    return tuple(map(int, sections))


def make_plan(what, q, k, positions, inv_freq, sections, section_order, pairing, scale, eps,
              weights, grads):
    """The plan of a call whose vectors and weights the kernels read as they are: (entry
    point, descriptor's address, shape and strides of the queries' output, of the keys',
    workspace bytes, descriptor), or the error its arguments deserve.  `sections`: None or a
    tuple of ints; `weights`: None (no norm) or (q_weight, k_weight); `grads`: None or
    (dq_out, dk_out)."""
    # the vectors that run through the rotation, under the name the caller knows
    names = ("dq_out", "dk_out") if what == "rope_bwd" else ("q", "k")
    _check_pair(q, k, what, names)
    if grads is not None:
        _check_pair(*grads, what, ("dq_out", "dk_out"), like=(q, k))
    lead, dim = tuple(q.shape[:-2]), q.shape[-1]
    if inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError(f"{what}: inv_freq must be a contiguous vector")
    if inv_freq.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"{what}: inv_freq must be float32 or float64, got {inv_freq.dtype}")
    n = inv_freq.shape[0]
    if not 1 <= dim <= _lib.ROPE_MAX_DIM:
        raise ValueError(f"{what}: head_dim must be 1..{_lib.ROPE_MAX_DIM}, got {dim}")
    heads, tokens = (q.shape[-2], k.shape[-2]), math.prod(lead)
    if max(heads) > _lib.ROPE_MAX_HEADS:
        raise ValueError(f"{what}: {names[0]} and {names[1]} may have at most "
                         f"{_lib.ROPE_MAX_HEADS} heads, got {heads[0]} and {heads[1]}")
    if tokens > _lib.ROPE_MAX_TOKENS:
        raise ValueError(f"{what}: fewer than 2^31 tokens are taken, got {tokens}")
    if tokens * sum(heads) * dim > _lib.ROPE_MAX_VALUES:
        raise ValueError(f"{what}: {names[0]} and {names[1]} may have at most 2^46 values, got "
                         f"{tokens * sum(heads) * dim}")
    if not 1 <= n <= dim // 2:
        raise ValueError(f"{what}: inv_freq of {n} does not fit a head_dim of {dim}")
    if section_order not in ORDERS:
        raise ValueError(f"{what}: section_order must be one of {sorted(ORDERS)}, got "
                         f"{section_order!r}")
    if pairing not in PAIRINGS:
        raise ValueError(f"{what}: pairing must be one of {sorted(PAIRINGS)}, got {pairing!r}")
    parts = (n,) if sections is None else sections
    if not 1 <= len(parts) <= _lib.ROPE_MAX_AXES:
        raise ValueError(f"{what}: sections must name 1..{_lib.ROPE_MAX_AXES} axes, got "
                         f"{list(parts)}")
    if min(parts) < 0 or sum(parts) != n:
        raise ValueError(f"{what}: sections {list(parts)} must add up to the {n} frequencies")
    if section_order == "cycle" and any(len(parts) * s > n for s in parts[1:]):
        raise ValueError(f"{what}: sections {list(parts)} do not fit {n} frequencies in turn")
    d = _lib.RopeDesc()
    d.batch, d.seq = lead if len(lead) == 2 else (1, lead[0])
    d.q_heads, d.k_heads, d.head_dim, d.n_freq = q.shape[-2], k.shape[-2], dim, n
    d.q_stride[:], d.k_stride[:] = _strides(q), _strides(k)
    if grads is not None:
        d.dq_stride[:], d.dk_stride[:] = (_strides(g) for g in grads)
    d.pos_stride[:] = _position_strides(positions, lead, len(parts), what)
    d.sections[:len(parts)] = parts
    d.axes, d.section_order, d.pairing = len(parts), ORDERS[section_order], PAIRINGS[pairing]
    d.dtype, d.w_dtype = _bridge.FLOAT_CODES[q.dtype], _lib.F32
    d.pos_dtype, d.f64_freq = POSITION_CODES[positions.dtype], inv_freq.dtype == torch.float64
    d.scale, d.eps = scale, eps  # rounded to 32 bits
    if not math.isfinite(d.scale):
        raise ValueError(f"{what}: scale must be finite in 32 bits, got {scale}")
    if not (math.isfinite(d.eps) and eps >= 0.0):
        raise ValueError(f"{what}: eps must be finite in 32 bits and not negative, got {eps}")
    if weights is not None:
        for w, name in zip(weights, ("q_weight", "k_weight")):
            if w is None:
                continue
            if tuple(w.shape) != (dim,):
                raise ValueError(f"{what}: {name} must have shape [{dim}], got {list(w.shape)}")
            d.w_dtype = _bridge.FLOAT_CODES[w.dtype]
    q_shape, k_shape = tuple(q.shape), tuple(k.shape)
    ws_bytes = (_lib.lib().vbh_qk_norm_rope_workspace_bytes(ctypes.byref(d))
                if grads is not None else 0)
    return (_lib.entry("vbh_" + what), ctypes.addressof(d), q_shape,
            _bridge.contiguous_strides(q_shape), k_shape, _bridge.contiguous_strides(k_shape),
            ws_bytes, d)


def _weight(w, dtype, what, name):
    """A weight the kernels read as it is: contiguous, of the vectors' dtype or fp32."""
    if w is None:
        return None
    if not w.dtype.is_floating_point:
        raise TypeError(f"{what}: {name} must be a floating tensor, got {w.dtype}")
    return w.contiguous() if w.dtype is dtype or w.dtype is torch.float32 else w.float()


def _weights(q_weight, k_weight, dtype, what):
    """Both weights as the kernels read them, of one dtype."""
    if (q_weight is not None and k_weight is not None and q_weight.dtype is k_weight.dtype and
            (q_weight.dtype is dtype or q_weight.dtype is torch.float32) and
            q_weight.is_contiguous() and k_weight.is_contiguous()):
        return q_weight, k_weight
    qw, kw = _weight(q_weight, dtype, what, "q_weight"), _weight(k_weight, dtype, what, "k_weight")
    if qw is not None and kw is not None and qw.dtype is not kw.dtype:
        return qw.float(), kw.float()
    return qw, kw


def _contiguous(t):
    """`t` with vectors that are contiguous."""
    st = t.stride()
    return t if not st or st[-1] == 1 else t.contiguous()


def _on(dev, what, *tensors):
    """The GPU all tensors lie on, `dev` or the error they deserve."""
    for t in tensors:
        if t is not None and (dev < 0 or t.get_device() != dev):
            return _bridge.require_gpu(what, *tensors)
    return dev


def _run(fn, what, dev, *args):
    if dev == _raw_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc != 0:
        raise _lib.VbhError("vbh_" + what, rc, _lib.last_error())


def rotate(what, q, k, positions, inv_freq, sections, section_order, pairing, scale):
    """rope_fwd, and rope_bwd with q and k the incoming gradients."""
    if sections is not None:
        sections = _sections(what, sections)
    if type(scale) is not float:
        scale = _number(what, scale, "scale")
    key = (what, q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, positions.shape,
           positions.stride(), positions.dtype, inv_freq.shape, inv_freq.stride(), inv_freq.dtype,
           sections, section_order, pairing, scale or str(scale))  # -0.0 == 0.0
    p = _PLANS.get(key)
    if p is None:
        qc, kc = _contiguous(q), _contiguous(k)
        if qc is not q or kc is not k:
            return rotate(what, qc, kc, positions, inv_freq, sections, section_order, pairing,
                          scale)
        p = _PLANS.put(key, make_plan(what, q, k, positions, inv_freq, sections, section_order,
                                      pairing, scale, 0.0, None, None))
    dev = q.get_device()
    if (dev < 0 or k.get_device() != dev or positions.get_device() != dev or
            inv_freq.get_device() != dev):
        dev = _bridge.require_gpu(what, q, k, positions, inv_freq)
    fn, desc, q_shape, q_strides, k_shape, k_strides, _, _ = p
    q_out = q.new_empty_strided(q_shape, q_strides)
    k_out = k.new_empty_strided(k_shape, k_strides)
    _run(fn, what, dev, desc, q.data_ptr(), k.data_ptr(), positions.data_ptr(),
         inv_freq.data_ptr(), q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


def norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, eps, sections, section_order,
                pairing, scale):
    what = "qk_norm_rope_fwd"
    if sections is not None:
        sections = _sections(what, sections)
    if type(scale) is not float:
        scale = _number(what, scale, "scale")
    if type(eps) is not float:
        eps = _number(what, eps, "eps")
    qw, kw = _weights(q_weight, k_weight, q.dtype, what)
    key = (what, q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, positions.shape,
           positions.stride(), positions.dtype, inv_freq.shape, inv_freq.stride(), inv_freq.dtype,
           sections, section_order, pairing, scale or str(scale), eps,
           None if qw is None else qw.shape, None if kw is None else kw.shape,
           (kw if qw is None else qw) is None or (kw if qw is None else qw).dtype)
    p = _PLANS.get(key)
    if p is None:
        qc, kc = _contiguous(q), _contiguous(k)
        if qc is not q or kc is not k:
            return norm_rotate(qc, kc, qw, kw, positions, inv_freq, eps, sections,
                               section_order, pairing, scale)
        p = _PLANS.put(key, make_plan(what, q, k, positions, inv_freq, sections, section_order,
                                      pairing, scale, eps, (qw, kw), None))
    dev = _on(q.get_device(), what, q, k, qw, kw, positions, inv_freq)
    fn, desc, q_shape, q_strides, k_shape, k_strides, _, _ = p
    q_out = q.new_empty_strided(q_shape, q_strides)
    k_out = k.new_empty_strided(k_shape, k_strides)
    _run(fn, what, dev, desc, q.data_ptr(), k.data_ptr(), None if qw is None else qw.data_ptr(),
         None if kw is None else kw.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
         q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


def norm_rotate_grads(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, eps,
                      sections, section_order, pairing, scale):
    what = "qk_norm_rope_bwd"
    if sections is not None:
        sections = _sections(what, sections)
    if type(scale) is not float:
        scale = _number(what, scale, "scale")
    if type(eps) is not float:
        eps = _number(what, eps, "eps")
    qw, kw = _weights(q_weight, k_weight, q.dtype, what)
    key = (what, q.shape, q.stride(), q.dtype, k.shape, k.stride(), k.dtype, positions.shape,
           positions.stride(), positions.dtype, inv_freq.shape, inv_freq.stride(), inv_freq.dtype,
           sections, section_order, pairing, scale or str(scale), eps,
           None if qw is None else qw.shape, None if kw is None else kw.shape,
           (kw if qw is None else qw) is None or (kw if qw is None else qw).dtype,
           dq_out.shape, dq_out.stride(), dq_out.dtype, dk_out.shape, dk_out.stride(),
           dk_out.dtype)
    p = _PLANS.get(key)
    if p is None:
        args = (dq_out, dk_out, q, k)
        dense = [_contiguous(t) for t in args]
        if any(a is not b for a, b in zip(args, dense)):
            return norm_rotate_grads(*dense, q_weight, k_weight, positions, inv_freq, eps,
                                     sections, section_order, pairing, scale)
        p = _PLANS.put(key, make_plan(what, q, k, positions, inv_freq, sections, section_order,
                                      pairing, scale, eps, (qw, kw),
                                      (dq_out, dk_out)))
    dev = _on(q.get_device(), what, q, k, dq_out, dk_out, qw, kw, positions, inv_freq)
    fn, desc, q_shape, q_strides, k_shape, k_strides, n, _ = p
    dq = q.new_empty_strided(q_shape, q_strides)
    dk = k.new_empty_strided(k_shape, k_strides)
    dqw = None if qw is None else torch.empty_like(qw)
    dkw = None if kw is None else torch.empty_like(kw)
    if qw is None and kw is None:
        n = 0
    ws = _bridge.empty(q, (n,), torch.uint8) if n else None
    _run(fn, what, dev, desc, dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(),
         _bridge.ptr(qw), _bridge.ptr(kw), positions.data_ptr(), inv_freq.data_ptr(),
         dq.data_ptr(), dk.data_ptr(), _bridge.ptr(dqw), _bridge.ptr(dkw), _bridge.ptr(ws), n)
    if dqw is not None and dqw.dtype is not q_weight.dtype:
        dqw = dqw.to(q_weight.dtype)
    if dkw is not None and dkw.dtype is not k_weight.dtype:
        dkw = dkw.to(k_weight.dtype)
    return dq, dk, dqw, dkw
