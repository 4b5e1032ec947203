"""rope - rotation of queries and keys by position, HIP backend.

``rope_fwd(q, k, positions, inv_freq, ...) -> (q_out, k_out)`` and its gradient
``rope_bwd(dq_out, dk_out, positions, inv_freq, ...) -> (dq, dk)``.

* ``q`` is ``[tokens, q_heads, head_dim]`` or ``[batch, tokens, q_heads, head_dim]``,
  ``k`` the same with its own number of heads; float32, float16 or bfloat16, in any
  strides (a slice of a packed projection, a transposed ``[batch, heads, tokens,
  head_dim]``).  The outputs are new contiguous tensors of the same shape.  Limits:
  ``head_dim`` 1024, 65536 heads of each, fewer than 2^31 tokens, 2^46 values in all.
* The first ``2 n`` values of a head turn, ``n = len(inv_freq)`` (float32 or float64, on
  the GPU); the others pass.  Pair ``p`` turns by ``position * inv_freq[p]``, formed in 64
  bits, so that far positions keep their angles; ``scale`` multiplies what turns.
* ``pairing``: ``"half"`` pairs value ``p`` with ``n + p``, ``"adjacent"`` ``2 p`` with
  ``2 p + 1``.
* ``positions``: int32, int64 or float32, ``[batch, tokens]`` or ``[tokens]`` (one row for
  the whole batch).  With ``sections`` (how many frequencies each of 2 to 4 axes has:
  time, height, width ...) ``[axes, batch, tokens]`` or ``[axes, tokens]``;
  ``section_order`` ``"blocks"`` gives axis 0 the first ``sections[0]`` frequencies and so
  on, ``"cycle"`` gives frequency ``p`` to axis ``p % axes`` while that axis has some left,
  the rest to axis 0.

One read and one write of each vector per call (libvbhip ``vbh_rope_fwd`` /
``vbh_rope_bwd``), on torch's current stream.  No reference counterpart: the
reference has no operator that takes positions.
"""
import os
import sys

_ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
if _ROOT not in sys.path:
    sys.path.insert(0, _ROOT)

from dslperfgap_amd import _rope  # noqa: E402


def rope_fwd(q, k, positions, inv_freq, sections=None, section_order="blocks", pairing="half",
             scale=1.0):
    """Rotate queries and keys by their positions."""
    return _rope.rotate("rope_fwd", q, k, positions, inv_freq, sections, section_order, pairing,
                        scale)


def rope_bwd(dq_out, dk_out, positions, inv_freq, sections=None, section_order="blocks",
             pairing="half", scale=1.0):
    """The gradients of rope_fwd's q and k from those of its outputs."""
    return _rope.rotate("rope_bwd", dq_out, dk_out, positions, inv_freq, sections, section_order,
                        pairing, scale)
