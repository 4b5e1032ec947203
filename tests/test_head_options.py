"""Options of the norms' gradients and of the projection's cross entropy that 32 bits cannot hold are
refused (nothing is launched)."""
import pytest
import torch

from dslperfgap_amd import _lib
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd

NOT_FINITE = [float("nan"), float("inf"), -float("inf"), 1e39, -1e39]


@pytest.mark.parametrize("eps", NOT_FINITE + [-1e-6, 3.5e38])
def test_rms_norm_bwd_eps(eps):
    x = torch.randn(4, 8)
    with pytest.raises(ValueError, match="finite in 32 bits"):
        rms_norm_bwd(x, x, (8,), torch.ones(8), eps)


@pytest.mark.parametrize("eps", NOT_FINITE + [-1e-6])
def test_entry_points_of_the_norms(eps):
    for name, outs in (("vbh_layer_norm_bwd", 3), ("vbh_rms_norm_bwd", 2)):
        with pytest.raises(_lib.VbhError, match="eps must be finite") as e:
            _lib.call(name, *[16] * (3 + outs), 4, 8, eps, 0, 0, 16, 1 << 30, None)
        assert e.value.code == _lib.E_INVALID


@pytest.mark.parametrize("value", NOT_FINITE)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_entry_points_of_the_cross_entropy(which, value):
    options = [0.1, 1.0, 1e-4]
    options[which] = value
    for name, pointers, more in (("vbh_linear_cross_entropy_fwd", 6, [0]),
                                 ("vbh_linear_cross_entropy_bwd", 7, [])):
        with pytest.raises(_lib.VbhError, match="finite in 32 bits") as e:
            _lib.call(name, *[256] * pointers, 4, 8, 10, 8, 8, *options, -100, 10, 0, 0, _lib.I64,
                      *more, 256, 1 << 40, None)
        assert e.value.code == _lib.E_INVALID
