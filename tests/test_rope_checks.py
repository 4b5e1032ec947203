"""What the query / key operators refuse does not depend on the calls before, and is refused
before anything is allocated."""
import decimal
import importlib
import re
from pathlib import Path

import pytest
import torch

from dslperfgap_amd import _lib, _rope
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


def _sizes(lead, hq, hk, dim=16):
    """Operands of any size in one vector of memory."""
    one = torch.zeros(dim)
    return {"q": one.expand(*lead, hq, dim), "k": one.expand(*lead, hk, dim),
            "pos": torch.zeros(1, dtype=torch.int32).expand(lead)}


@pytest.mark.parametrize("sizes,match", [
    (((5,), 65537, 1), "at most 65536 heads"), (((5,), 1, 65537), "at most 65536 heads"),
    (((1 << 31,), 1, 1), "fewer than 2\\^31 tokens"),
    (((1 << 16, 1 << 15), 1, 1), "fewer than 2\\^31 tokens"),
    (((1 << 30,), 1 << 12, 1), "at most 2\\^46 values"),
], ids=str)
def test_sizes_beyond_the_kernels_are_refused_and_leave_no_plan(sizes, match):
    _rope._PLANS.cache_clear()
    for call in _calls(**_sizes(*sizes)):
        with pytest.raises(ValueError, match=match):
            call()
    assert not _rope._PLANS


@pytest.mark.parametrize("sizes", [((5,), 65536, 65536), (((1 << 31) - 1,), 1, 1),
                                   ((1 << 15, 1 << 15), 4095, 1)], ids=str)
def test_the_largest_sizes_are_taken(sizes):
    _planned(**_sizes(*sizes))


def test_the_limits_are_the_headers():
    header = (Path(__file__).parents[1] / "include" / "vbhip.h").read_text()
    limits = dict(re.findall(r"#define VBH_(ROPE_MAX_\w+) +(\(.*?\) << \d+\)|\d+)", header))
    assert len(limits) == 5
    for name, text in limits.items():
        value = text.replace("INT64_C(1)", "1")
        a, _, b = value.strip("()").partition(" << ")
        assert getattr(_lib, name) == int(a) << int(b or 0), name


@pytest.mark.parametrize("name", ["rope", "qk_norm_rope"])
def test_packages_say_what_they_hold(name):
    """Neither is an operator of ViperBench."""
    doc = importlib.import_module(f"dslperfgap_amd.viperbench.{name}").__doc__
    assert doc.startswith(name + ":") and "ViperBench" not in doc
