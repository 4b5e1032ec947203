"""What the query / key operators refuse does not depend on the calls before, and is refused
before anything is allocated."""
import decimal

import pytest
import torch

from dslperfgap_amd import _rope
from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
from dslperfgap_amd.viperbench.rope.hip_impl import rope_bwd, rope_fwd

Q, K = torch.randn(5, 4, 16), torch.randn(5, 2, 16)
POS, FREQ = torch.arange(5), torch.ones(8)
W = torch.ones(16)


def _calls(q=Q, k=K, pos=POS, **how):
    norm = [lambda: qk_norm_rope_fwd(q, k, W, W, pos, FREQ, **how),
            lambda: qk_norm_rope_bwd(q, k, q, k, W, W, pos, FREQ, **how)]
    if "eps" in how:
        return norm
    return [lambda: rope_fwd(q, k, pos, FREQ, **how), lambda: rope_bwd(q, k, pos, FREQ, **how),
            *norm]


def _planned(**how):
    """Right arguments: the device check is reached (the tensors lie on the CPU), and the
    plan is kept."""
    for call in _calls(**how):
        with pytest.raises(ValueError, match="GPU tensors"):
            call()


@pytest.mark.parametrize("right,wrong,name", [
    ({"sections": (8,)}, {"sections": (8.0,)}, "sections"),
    ({"sections": [8]}, {"sections": [8.0]}, "sections"),
    ({"sections": (4, 4)}, {"sections": (4, 4.0)}, "sections"),
    ({"scale": 1.0}, {"scale": 1 + 0j}, "scale"),
    ({"scale": 2}, {"scale": decimal.Decimal(2)}, "scale"),
    ({"eps": 0.5}, {"eps": 0.5 + 0j}, "eps"),
], ids=str)
def test_values_that_equal_right_ones_are_refused_as_before_them(right, wrong, name):
    pos = POS.expand(2, 5) if right.get("sections") == (4, 4) else POS
    _rope._PLANS.cache_clear()
    for _ in range(2):
        for call in _calls(pos=pos, **wrong):
            with pytest.raises(TypeError, match=f"{name} must be"):
                call()
        _planned(pos=pos, **right)


def test_scales_of_either_zero_have_plans_of_their_own():
    """-0 * x and 0 * x differ in the sign of zero."""
    _rope._PLANS.cache_clear()
    signs = []
    for scale in (0.0, -0.0, 0, False):
        with pytest.raises(ValueError, match="GPU tensors"):
            rope_fwd(Q, K, POS, FREQ, scale=scale)
        signs.append(len(_rope._PLANS))
    assert signs == [1, 2, 2, 2]


@pytest.mark.parametrize("how,match", [
    ({"scale": 1e300}, "scale must be finite in 32 bits"),
    ({"scale": -3.5e38}, "scale must be finite in 32 bits"),
    ({"eps": 1e300}, "eps must be finite in 32 bits"),
], ids=str)
def test_numbers_beyond_32_bits_are_refused_and_leave_no_plan(how, match):
    _rope._PLANS.cache_clear()
    for call in _calls(**how):
        with pytest.raises(ValueError, match=match):
            call()
    assert not _rope._PLANS
    _planned(scale=3.4028234e38)
    _planned(eps=3.4028234e38)
