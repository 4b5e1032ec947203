"""The norms' gradients on the CPU: the oracle against automatic differentiation and differences,
and every call they refuse, in Python and at the C entry points (nothing is launched)."""
import pytest
import torch

from dslperfgap_amd import _lib
from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd
from oracle import norm_grads as ref

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("layer_norm", [True, False])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (4, 64)])
def test_oracle_gradients_are_autograds_and_the_differences(layer_norm, rows, cols):
    g = torch.Generator().manual_seed(5)
    x, dy = (torch.randn(rows, cols, generator=g, dtype=torch.float64) for _ in range(2))
    w = 1 + 0.2 * torch.randn(cols, generator=g, dtype=torch.float64)
    b = torch.zeros(cols, dtype=torch.float64)

    def f(x, w, b):
        d = x - x.mean(1, keepdim=True) if layer_norm else x
        return (d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b).mul(dy).sum()

    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(f(*leaves), leaves)
    (dx, dw, db), _ = ref.backward(dy, x, w, 1e-5, layer_norm)
    assert torch.allclose(dx, want[0], atol=1e-10)
    assert torch.allclose(dw, want[1], atol=1e-10)
    if layer_norm:
        assert torch.allclose(db, want[2], atol=1e-12)
    v, e = torch.randn(x.shape, generator=g, dtype=torch.float64), 1e-7
    slope = (f(x + e * v, w, b) - f(x - e * v, w, b)) / (2 * e)
    assert abs(float(slope - (dx * v).sum())) < 1e-4 * (1 + float(dx.abs().sum()))


def test_layer_norm_bwd_refusals():
    x, w = torch.randn(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="GPU tensors"):
        layer_norm_bwd(x, x, w, w)
    with pytest.raises(ValueError, match="GPU tensors"):
        layer_norm_bwd(x, x, torch.ones(4, 8), None)
    with pytest.raises(ValueError, match="eps=1e-5"):
        layer_norm_bwd(x, x, w, w, 1e-6)
    with pytest.raises(RuntimeError, match="does not match"):
        layer_norm_bwd(x, x, torch.ones(7), None)
    with pytest.raises(RuntimeError, match="does not match"):
        layer_norm_bwd(x, x, torch.ones(2, 4, 8), None)
    with pytest.raises(RuntimeError, match="bias shape"):
        layer_norm_bwd(x, x, w, torch.ones(7))
    with pytest.raises(ValueError, match="dy must have shape"):
        layer_norm_bwd(x[:3], x, w, w)
    with pytest.raises(TypeError, match="dy dtype"):
        layer_norm_bwd(x.half(), x, w, w)
    with pytest.raises(TypeError, match="weight dtype"):
        layer_norm_bwd(x, x, w.half(), None)
    with pytest.raises(TypeError, match="dtypes differ"):
        layer_norm_bwd(x.half(), x.half(), w, w.half())
    with pytest.raises(TypeError, match="not supported"):
        layer_norm_bwd(x.double(), x.double(), w.double(), None)


def test_rms_norm_bwd_refusals():
    x, w = torch.randn(4, 8), torch.ones(8)
    with pytest.raises(ValueError, match="GPU tensors"):
        rms_norm_bwd(x, x, (8,), w)
    with pytest.raises(RuntimeError, match="more dims"):
        rms_norm_bwd(x, x, (2, 4, 8), w)
    with pytest.raises(RuntimeError, match="weight has"):
        rms_norm_bwd(x, x, (8,), w[:7])
    with pytest.raises(ValueError, match="dy must have shape"):
        rms_norm_bwd(x[:3], x, (8,), w)
    with pytest.raises(TypeError, match="dy dtype"):
        rms_norm_bwd(x.half(), x, (8,), w)
    with pytest.raises(TypeError, match="not supported"):
        rms_norm_bwd(x.double(), x.double(), (8,), w)
    for bad in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps must be"):
            rms_norm_bwd(x, x, (8,), w, bad)


def _fails(code, match, name, *args):
    with pytest.raises(_lib.VbhError, match=match) as e:
        _lib.call(name, *args)
    assert e.value.code == code


def _ln(dy=16, x=16, w=16, dx=16, dw=16, db=16, rows=4, cols=8, dt=0, wdt=0, ws=16, nbytes=1 << 30):
    return ("vbh_layer_norm_bwd", dy, x, w, dx, dw, db, rows, cols, 1e-5, dt, wdt, ws, nbytes, None)


def test_entry_point_errors_before_launch():
    _fails(_lib.E_DTYPE, "unsupported dtype", *_ln(dt=5))
    _fails(_lib.E_DTYPE, "weight dtype", *_ln(dt=_lib.BF16, wdt=_lib.F16))
    _fails(_lib.E_INVALID, "negative", *_ln(rows=-1))
    _fails(_lib.E_INVALID, "negative", *_ln(cols=-1))
    _fails(_lib.E_RANGE, "too large", *_ln(cols=1 << 31))
    _fails(_lib.E_RANGE, "more than one launch", *_ln(rows=1 << 40))
    for name in ("dy", "x", "w", "dx"):
        _fails(_lib.E_INVALID, "null pointer", *_ln(**{name: None}))
    _fails(_lib.E_INVALID, "workspace", *_ln(ws=None))
    _fails(_lib.E_INVALID, "workspace", *_ln(ws=24))
    _fails(_lib.E_INVALID, "workspace", *_ln(nbytes=16))
    _fails(_lib.E_INVALID, "workspace", *_ln(cols=100000, dw=None, db=None, ws=None))
    _fails(_lib.E_INVALID, "null pointer", "vbh_rms_norm_bwd", None, 16, 16, 16, 16, 4, 8, 1e-5, 0,
           0, 16, 1 << 30, None)
    # nothing to do
    _lib.call(*_ln(dy=None, x=None, w=None, dx=None, dw=None, db=None, rows=0, ws=None, nbytes=0))
    _lib.call(*_ln(dy=None, x=None, w=None, dx=None, cols=0, ws=None, nbytes=0))


def test_workspace_is_a_function_of_the_sizes():
    size = _lib.lib().vbh_norm_bwd_workspace_bytes
    assert size(8, 64, 0, 1) == 2 * size(8, 64, 0, 0) > 0
    assert size(0, 64, 0, 1) > 0  # dw and db of no rows
    assert size(8, 0, 0, 1) == size(-1, 8, 0, 1) == size(8, 8, 4, 1) == size(8, 1 << 31, 0, 1) == 0
