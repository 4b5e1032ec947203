"""The projection's cross entropy on the CPU: the oracle against the logits' own golden, automatic
differentiation and differences, and every call that is refused, in Python and at the C entry
points (nothing is launched)."""
import pytest
import torch

from dslperfgap_amd import _lib
from dslperfgap_amd.viperbench.linear_cross_entropy.hip_impl import (linear_cross_entropy_bwd,
                                                                     linear_cross_entropy_fwd)
from oracle import linear_ce as ref
from oracle import pytorch_impl as golden

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _make(tokens=9, hidden=12, vocab=21, dtype=torch.float64, seed=6):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g, dtype=torch.float64).to(dtype)
    w = torch.randn(vocab, hidden, generator=g, dtype=torch.float64).to(dtype)
    labels = torch.randint(0, vocab, (tokens,), generator=g)
    labels[2] = -100
    return x, w, labels


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("smoothing,scale,z,start,total", [
    (0.0, 1.0, 0.0, 0, 21), (0.1, 0.7, 1e-2, 0, 21), (0.2, 1.5, 0.0, 4, 40)])
def test_oracle_is_the_golden_of_its_logits(smoothing, scale, z, start, total, split):
    x, w, labels = _make()
    logits = (x @ w.T).float()
    got, _ = ref.forward(x, w, labels, smoothing, scale, z, -100, total, start, split)
    want = golden.cross_entropy_fwd(logits, labels, smoothing, scale, z, -100, total, start, 32,
                                    smoothing > 0, split)
    keep = labels != -100
    for p, q in zip(got, want):
        assert torch.allclose(p[keep].float(), q.reshape(-1)[:9][keep], atol=2e-4)
        assert float(p[~keep].abs().max()) == 0.0


@pytest.mark.parametrize("smoothing,scale,z", [(0.0, 1.0, 0.0), (0.1, 0.7, 1e-2)])
def test_oracle_gradients_are_autograds_and_the_differences(smoothing, scale, z):
    x, w, labels = _make()
    dloss = torch.rand(9, dtype=torch.float64, generator=torch.Generator().manual_seed(1))

    def f(x, w):
        return (ref.forward(x, w, labels, smoothing, scale, z)[0][0] * dloss).sum()

    lse = torch.logsumexp(scale * x @ w.T, 1)
    (dx, dw), _ = ref.backward(dloss, x, w, lse, labels, smoothing, scale, z)
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    want = torch.autograd.grad(f(*leaves), leaves)
    assert torch.allclose(dx, want[0], atol=1e-12) and torch.allclose(dw, want[1], atol=1e-12)
    v = torch.randn(w.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    slope = (f(x, w + 1e-6 * v) - f(x, w - 1e-6 * v)) / 2e-6
    assert abs(float(slope - (dw * v).sum())) < 1e-6


def _refused(error, match, x, w, labels, dloss=None, lse=None, **how):
    n = labels.shape[0] if labels.dim() == 1 else 1
    dloss = torch.ones(n) if dloss is None else dloss
    lse = torch.ones(n) if lse is None else lse
    with pytest.raises(error, match=match):
        linear_cross_entropy_fwd(x, w, labels, **how)
    with pytest.raises(error, match=match):
        linear_cross_entropy_bwd(dloss, x, w, lse, labels, **how)


def test_calls_are_refused():
    x, w, labels = _make(dtype=F32)
    _refused(ValueError, "GPU tensors", x, w, labels)
    _refused(ValueError, "GPU tensors", x, w.T.contiguous().T, labels.to(torch.int16))
    _refused(ValueError, "GPU tensors", x[:0], w, labels[:0])
    _refused(ValueError, "x must be 2-D", x[None], w, labels)
    _refused(ValueError, "weight must be 2-D", x, w[0], labels)
    _refused(ValueError, "values per token", x, w[:, :11], labels)
    _refused(ValueError, "weight is empty", x, w[:0], labels)
    _refused(ValueError, "weight is empty", x[:, :0], w[:, :0], labels)
    _refused(ValueError, "labels must have shape", x, w, labels[:8])
    _refused(ValueError, "labels must have shape", x, w, labels[None])
    _refused(TypeError, "integer tensor", x, w, labels.float())
    _refused(TypeError, "integer tensor", x, w, labels > 0)
    _refused(TypeError, "weight dtype", x, w.half(), labels)
    _refused(TypeError, "not supported", x.double(), w.double(), labels)
    one = torch.ones(9)
    for bad in ({"dloss": one[:8]}, {"lse": one[:8]}, {"dloss": one[None]}):
        with pytest.raises(ValueError, match="must have shape"):
            linear_cross_entropy_bwd(**{"dloss": one, "lse": one, **bad}, x=x, weight=w, labels=labels)
    with pytest.raises(TypeError, match="float tensor"):
        linear_cross_entropy_bwd(one.long(), x, w, one, labels)


def _fails(code, match, name, *args):
    with pytest.raises(_lib.VbhError, match=match) as e:
        _lib.call(name, *args)
    assert e.value.code == code


P = 4096  # a pointer that nothing reads


def _fwd(x=P, w=P, labels=P, loss=P, lse=P, z=P, tokens=4, hidden=8, vocab=16, xs=8, ws=8, total=16,
         start=0, dt=0, ldt=4, work=P, nbytes=1 << 40):
    return ("vbh_linear_cross_entropy_fwd", x, w, labels, loss, lse, z, tokens, hidden, vocab, xs,
            ws, 0.0, 1.0, 0.0, -100, total, start, dt, ldt, 0, work, nbytes, None)


def _bwd(dloss=P, x=P, w=P, lse=P, labels=P, dx=P, dw=P, tokens=4, hidden=8, vocab=16, xs=8, ws=8,
         total=16, start=0, dt=0, ldt=4, work=P, nbytes=1 << 40):
    return ("vbh_linear_cross_entropy_bwd", dloss, x, w, lse, labels, dx, dw, tokens, hidden, vocab,
            xs, ws, 0.0, 1.0, 0.0, -100, total, start, dt, ldt, work, nbytes, None)


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_entry_point_errors_before_launch(call):
    _fails(_lib.E_DTYPE, "unsupported dtype", *call(dt=4))
    _fails(_lib.E_DTYPE, "int32 or int64", *call(ldt=0))
    for bad in ({"tokens": -1}, {"hidden": 0}, {"vocab": 0}):
        _fails(_lib.E_INVALID, "negative size", *call(**bad))
    for bad in ({"tokens": (1 << 24) + 1}, {"hidden": (1 << 16) + 8, "xs": 1 << 17, "ws": 1 << 17},
                {"vocab": (1 << 24) + 1},
                {"vocab": 1 << 24, "hidden": 1 << 16, "xs": 1 << 16, "ws": 1 << 16}):
        _fails(_lib.E_RANGE, "out of range", *call(**bad))
    for bad in ({"xs": 7}, {"ws": 7}):
        _fails(_lib.E_INVALID, "row stride", *call(**bad))
    _fails(_lib.E_RANGE, "row stride", *call(xs=1 << 33))
    _fails(_lib.E_INVALID, "total_classes", *call(total=0))
    _fails(_lib.E_INVALID, "class_start_idx", *call(start=-1))
    for name in ("x", "w", "labels", "lse"):
        _fails(_lib.E_INVALID, "null pointer", *call(**{name: None}))
    _fails(_lib.E_INVALID, "workspace", *call(work=None))
    _fails(_lib.E_INVALID, "workspace", *call(work=P + 16))
    _fails(_lib.E_INVALID, "workspace", *call(nbytes=100))


def test_nothing_to_do():
    _lib.call(*_fwd(tokens=0, x=None, w=None, labels=None, work=None))
    _lib.call(*_bwd(tokens=0, dw=None, x=None, work=None))
    _lib.call(*_bwd(dx=None, dw=None, work=None))


def test_workspace_is_a_function_of_the_sizes():
    size = _lib.lib().vbh_linear_cross_entropy_workspace_bytes
    assert 0 < size(8, 64, 100, 2, 0, 0) < size(8, 64, 100, 2, 1, 0)
    assert size(0, 64, 100, 2, 0, 1) == size(8, 0, 100, 2, 0, 1) == size(8, 8, 8, 3, 0, 1) == 0
    # pieces of the vocabulary bound the gradients of the logits, not the vocabulary
    whole = 8192 * 128000 * 2
    assert size(8192, 4096, 128000, 2, 0, 1) < whole
    # and the forward keeps a hundredth of the logits
    assert size(8192, 4096, 128000, 2, 0, 0) - 8192 * 4096 * 2 < whole / 20


@pytest.mark.parametrize("dtype,logits", [(2, 1 << 39), (1, 1 << 39), (0, 1 << 37)])
def test_more_logits_than_one_launch_takes(dtype, logits):
    size = _lib.lib().vbh_linear_cross_entropy_workspace_bytes
    for tokens in (1 << 24, 1 << 20):
        assert size(tokens, 64, logits // tokens // 2, dtype, 0, 0) > 0
        vocab = min(logits // tokens * 2, 1 << 24)
        assert size(tokens, 64, vocab, dtype, 0, 0) == 0
        _fails(_lib.E_RANGE, "more than one launch", *_fwd(tokens=tokens, hidden=64, vocab=vocab,
                                                           xs=64, ws=64, dt=dtype))
        # the gradients come in pieces
        assert size(tokens, 64, vocab, dtype, 0, 1) > 0
