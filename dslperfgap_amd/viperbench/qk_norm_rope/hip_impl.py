"""qk_norm_rope - RMSNorm of every query and key head, then the rotation by position, in
one pass, HIP backend.

``qk_norm_rope_fwd(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, ...) ->
(q_out, k_out)``: each vector of ``head_dim`` values becomes ``x / sqrt(mean(x^2) + eps) *
weight`` (as ``rms_norm``) and is turned as by ``rope_fwd`` (viperbench/rope, which
describes ``positions``, ``inv_freq``, ``sections``, ``section_order``, ``pairing``,
``scale`` and the layouts); fp32 throughout, rounded once.  A vector of finite values whose
squares add up beyond the range of fp32 becomes zeros, as in ``rms_norm``, and so do its
gradients; with ``eps`` 0 one whose squares are all 0 in fp32 (values below 2^-75) has no
finite output.

``qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, ...) ->
(dq, dk, dq_weight, dk_weight)`` from the forward's inputs and the gradients of its
outputs (the same shapes and dtype, any strides).

The weights are ``[head_dim]``, or None for ones (whose gradient is then None).  Their
gradients are summed in fp32 in a fixed order and have the weights' dtype.

One read and one write of each vector per call (libvbhip ``vbh_qk_norm_rope_fwd``), two
reads and one write backward (``vbh_qk_norm_rope_bwd``).  No reference counterpart:
the reference's nearest operator is ViperBench/rms_norm/pytorch_impl.py:3-10.
"""
import os
import sys

_ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
if _ROOT not in sys.path:
    sys.path.insert(0, _ROOT)

from dslperfgap_amd import _rope  # noqa: E402


def qk_norm_rope_fwd(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, sections=None,
                     section_order="blocks", pairing="half", scale=1.0):
    """Per-head RMSNorm of queries and keys, then the rotation."""
    return _rope.norm_rotate(q, k, q_weight, k_weight, positions, inv_freq, eps, sections,
                             section_order, pairing, scale)


def qk_norm_rope_bwd(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6,
                     sections=None, section_order="blocks", pairing="half", scale=1.0):
    """The gradients of qk_norm_rope_fwd's q, k and weights from those of its outputs."""
    return _rope.norm_rotate_grads(dq_out, dk_out, q, k, q_weight, k_weight, positions, inv_freq,
                                   eps, sections, section_order, pairing, scale)
