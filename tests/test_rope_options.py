"""Options of the query / key operators that are no plain numbers: refused before a plan is
kept by them, since a tensor's value may change behind its identity."""
import pytest
import torch

from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
from dslperfgap_amd.viperbench.rope.hip_impl import rope_bwd, rope_fwd

Q, K = torch.randn(5, 4, 16), torch.randn(5, 2, 16)
POS, FREQ = torch.arange(5), torch.ones(8)


def _calls(**how):
    yield lambda: rope_fwd(Q, K, POS, FREQ, **how)
    yield lambda: rope_bwd(Q, K, POS, FREQ, **how)
    yield lambda: qk_norm_rope_fwd(Q, K, None, None, POS, FREQ, **how)
    yield lambda: qk_norm_rope_bwd(Q, K, Q, K, None, None, POS, FREQ, **how)


@pytest.mark.parametrize("how,name", [
    ({"scale": torch.tensor(2.0)}, "scale"), ({"scale": "2"}, "scale"),
    ({"scale": None}, "scale"), ({"sections": (torch.tensor(8),)}, "sections"),
    ({"sections": [4.0, 4.0]}, "sections"), ({"sections": 8}, "sections")])
def test_options_that_are_no_numbers_are_refused(how, name):
    for call in _calls(**how):
        with pytest.raises(TypeError, match=f"{name} must be"):
            call()


def test_an_eps_that_is_no_number_is_refused():
    for fn, args in ((qk_norm_rope_fwd, (Q, K)), (qk_norm_rope_bwd, (Q, K, Q, K))):
        with pytest.raises(TypeError, match="eps must be"):
            fn(*args, None, None, POS, FREQ, eps=torch.tensor(1e-6))


def test_numbers_of_other_types_are_taken():
    """They reach the device check: the tensors here lie on the CPU."""
    for how in ({"scale": 2}, {"sections": [8]}, {"sections": (8,)}):
        for call in _calls(**how):
            with pytest.raises(ValueError, match="GPU tensors"):
                call()
