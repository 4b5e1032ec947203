"""Calls of the training head's operators that their documents allow beside the usual ones: rows far
apart, and the entry points' outputs that are not wanted."""
import pytest
import torch

from dslperfgap_amd import _lib
from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd
from dslperfgap_amd.viperbench.linear_cross_entropy.hip_impl import (linear_cross_entropy_bwd,
                                                                     linear_cross_entropy_fwd)
from oracle import linear_ce as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _make(tokens, hidden, vocab, dtype, ignored=0.0):
    g = torch.Generator(DEV).manual_seed(tokens + 7 * hidden + 13 * vocab)
    w = (1.5 / hidden ** 0.5 * torch.randn(vocab, hidden, generator=g, device=DEV)).to(dtype)
    x = torch.randn(tokens, hidden, generator=g, device=DEV).to(dtype)
    lab = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
    lab[torch.randperm(tokens, generator=g, device=DEV)[:round(ignored * tokens)]] = -100
    return x, w, lab, torch.rand(tokens, generator=g, device=DEV) / tokens


def _apart(t, values):
    """t's rows `values` apart, with what is no number between them."""
    wide = torch.full((t.shape[0] * values,), float("nan"), device=DEV, dtype=t.dtype)
    rows = wide.view(t.shape[0], values)[:, :t.shape[1]]
    rows.copy_(t)
    return rows


# the farthest apart that is read in place (1 MiB), and farther; tiles of 32, 64, 128 and 256 rows
@pytest.mark.parametrize("more", [0, 16])
@pytest.mark.parametrize("dtype,tokens,hidden,vocab", [
    (BF16, 20, 128, 1500), (F32, 300, 72, 700), (BF16, 1100, 264, 1700), (F16, 300, 64, 1300)])
def test_rows_a_mebibyte_apart(dtype, tokens, hidden, vocab, more):
    print(f"[gpu] far rows {dtype} {tokens} {hidden} {vocab} {more}", flush=True)
    x, w, lab, dloss = _make(tokens, hidden, vocab, dtype, 0.1)
    loss, lse, z = linear_cross_entropy_fwd(x, w, lab)
    want = (loss, lse, z, *linear_cross_entropy_bwd(dloss, x, w, lse, lab))
    apart = ((1 << 20) + more) // x.element_size()
    for xs, ws in ((_apart(x, apart), w), (x, _apart(w, apart))):
        got = linear_cross_entropy_fwd(xs, ws, lab)
        got = (*got, *linear_cross_entropy_bwd(dloss, xs, ws, lse, lab))
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def _workspace(size):
    return torch.empty(size, dtype=torch.uint8, device=DEV)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("tokens", [20, 700])
def test_gradients_that_are_not_wanted(dtype, tokens):
    """dw without dx (in fp16 at the common scale at once), and dx without dw."""
    hidden, vocab = 72, 3001
    x, w, lab, _ = _make(tokens, hidden, vocab, dtype, 0.2)
    dloss = torch.exp2(-18 * torch.rand(tokens, device=DEV))
    lse = linear_cross_entropy_fwd(x, w, lab)[1]
    both = linear_cross_entropy_bwd(dloss, x, w, lse, lab)
    code = {F32: _lib.F32, F16: _lib.F16, BF16: _lib.BF16}[dtype]
    nbytes = _lib.lib().vbh_linear_cross_entropy_workspace_bytes(tokens, hidden, vocab, code, 0, 1)
    ws, stream = _workspace(nbytes), torch.cuda.current_stream().cuda_stream
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    for a, b in ((None, dw), (dx, None), (None, None)):
        _lib.call("vbh_linear_cross_entropy_bwd", dloss.data_ptr(), x.data_ptr(), w.data_ptr(),
                  lse.data_ptr(), lab.data_ptr(), a.data_ptr() if a is not None else None,
                  b.data_ptr() if b is not None else None, tokens, hidden, vocab, hidden, hidden, 0.0,
                  1.0, 0.0, -100, vocab, 0, code, _lib.I64, ws.data_ptr(), nbytes, stream)
    assert torch.equal(dx, both[0])
    if dtype != F16:
        assert torch.equal(dw, both[1])
    want, bounds = ref.backward(dloss, x, w, lse, lab)
    off = (dw.double() - want[1]).abs() - ref.rounded(bounds[1], want[1], dtype)
    assert float(off.max()) <= 0.0


@pytest.mark.parametrize("rows,cols", [(70, 100), (600, 5000), (300, 20480), (9, 40000)])
def test_norm_gradients_that_are_not_wanted(rows, cols):
    g = torch.Generator(DEV).manual_seed(rows)
    x, dy = (torch.randn(rows, cols, generator=g, device=DEV).to(BF16) for _ in range(2))
    w = torch.randn(cols, generator=g, device=DEV)
    want = layer_norm_bwd(dy, x, w, w)
    nbytes = _lib.lib().vbh_norm_bwd_workspace_bytes(rows, cols, _lib.BF16, 1)
    ws, stream = _workspace(nbytes), torch.cuda.current_stream().cuda_stream
    for wanted in ((True, False), (False, True), (False, False)):
        got = [torch.full_like(t, 7.0) for t in want]
        ptr = [t.data_ptr() if on else None for t, on in zip(got[1:], wanted)]
        _lib.call("vbh_layer_norm_bwd", dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                  got[0].data_ptr(), *ptr, rows, cols, 1e-5, _lib.BF16, _lib.F32, ws.data_ptr(),
                  nbytes, stream)
        assert torch.equal(got[0], want[0])
        for t, q, on in zip(got[1:], want[1:], wanted):
            assert torch.equal(t, q if on else torch.full_like(q, 7.0))
    if cols <= 32768:  # rows in registers need no workspace without the weights' gradients
        got = torch.empty_like(x)
        _lib.call("vbh_layer_norm_bwd", dy.data_ptr(), x.data_ptr(), w.data_ptr(), got.data_ptr(),
                  None, None, rows, cols, 1e-5, _lib.BF16, _lib.F32, None, 0, stream)
        assert torch.equal(got, want[0])
