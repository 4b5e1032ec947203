"""The norms' gradients on the GPU against the oracle, within the bounds derived there."""
import pytest
import torch

from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd
from oracle import norm_grads as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# one value; less than an access; slices of a wave; a wave; ragged; several waves with one to four
# accesses a lane; the widest rows in registers (16384 fp32, 32768 16-bit values); beyond them
SIZES = [(1, 1), (3, 5), (7, 8), (129, 40), (1000, 64), (513, 100), (4097, 33), (258, 768),
         (5003, 1001), (300, 4096), (2048, 4100), (65, 9000), (77, 20480), (40, 20481),
         (20, 32768), (10, 40000), (67, 70001)]


def _held(got, want, bound, what):
    assert got.shape == want.shape
    off = (got.cpu().double() - want).abs() - ref.rounded(bound, want, got.dtype)
    assert float(off.max()) <= 0.0, (what, float(off.max()))


def _check(x, dy, w, b, layer_norm, eps=1e-5):
    if layer_norm:
        got = layer_norm_bwd(dy, x, w, b, eps)
    else:
        got = (*rms_norm_bwd(dy, x, (x.shape[-1],), w, eps), None)
    cols = x.shape[-1]
    want, bounds = ref.backward(dy.reshape(-1, cols).cpu(), x.reshape(-1, cols).cpu(), w.cpu(), eps,
                                layer_norm)
    assert got[0].dtype == x.dtype and got[1].dtype == w.dtype and got[0].shape == x.shape
    _held(got[0].reshape(-1, cols), want[0], bounds[0], "dx")
    _held(got[1], want[1], bounds[1], "dw")
    if got[2] is not None:
        _held(got[2], want[2], bounds[2], "db")
    return got


def _make(rows, cols, dtype, wdtype, seed=0, mean=0.5):
    g = torch.Generator(DEV).manual_seed(seed + rows * 7 + cols)
    x = 2 * torch.randn(rows, cols, generator=g, device=DEV) + mean
    dy = torch.randn(rows, cols, generator=g, device=DEV)
    w = 1 + 0.2 * torch.randn(cols, generator=g, device=DEV)
    return x.to(dtype), dy.to(dtype), w.to(wdtype), torch.zeros(cols, device=DEV, dtype=wdtype)


@pytest.mark.parametrize("layer_norm", [True, False])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16),
                                          (F16, F32)])
def test_sizes(dtype, wdtype, layer_norm):
    for rows, cols in SIZES:
        print(f"[gpu] norm_bwd {dtype} {wdtype} {rows} x {cols}", flush=True)
        _check(*_make(rows, cols, dtype, wdtype), layer_norm)


@pytest.mark.parametrize("layer_norm", [True, False])
@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("rows,cols", [(700, 20480), (513, 24580), (300, 12000), (600, 16384),
                                       (3000, 2048), (9001, 72), (2049, 520)])
def test_several_rows_after_each_other(rows, cols, dtype, wdtype, layer_norm):
    """More rows than the launch holds at once, in each way that rows lie over lanes."""
    _check(*_make(rows, cols, dtype, wdtype), layer_norm)


@pytest.mark.parametrize("layer_norm", [True, False])
def test_many_short_rows(layer_norm):
    """More rows than a launch of one workgroup per row could have."""
    _check(*_make((1 << 22) + 5, 8, BF16, BF16), layer_norm)


@pytest.mark.parametrize("layer_norm", [True, False])
def test_no_rows_give_zero_weight_gradients(layer_norm):
    x, dy, w, b = _make(0, 96, BF16, F32)
    got = layer_norm_bwd(dy, x, w, b) if layer_norm else rms_norm_bwd(dy, x, (96,), w)
    assert got[0].shape == (0, 96)
    for t in got[1:]:
        assert torch.equal(t, torch.zeros_like(w))


def test_without_bias_and_over_several_axes():
    x, dy, w, _ = _make(24, 6 * 50, F32, F32)
    dx, dw, db = layer_norm_bwd(dy.view(4, 6, 6, 50), x.view(4, 6, 6, 50), w.view(6, 50), None)
    assert db is None and dw.shape == (6, 50) and dx.shape == (4, 6, 6, 50)
    flat = layer_norm_bwd(dy, x, w, torch.zeros_like(w))
    assert torch.equal(dx.reshape(24, 300), flat[0]) and torch.equal(dw.reshape(-1), flat[1])


def test_other_layouts_and_offsets():
    """Rows apart from each other, columns ahead of rows, expanded gradients, and tensors that do
    not begin at a multiple of 16 bytes."""
    x, dy, w, b = _make(70, 128, BF16, BF16)
    want = layer_norm_bwd(dy, x, w, b)
    wide = torch.zeros(70, 200, device=DEV, dtype=BF16)
    wide[:, 3:131] = x
    got = layer_norm_bwd(dy.T.contiguous().T, wide[:, 3:131], w, b)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    flat = torch.zeros(70 * 128 + 1, device=DEV, dtype=BF16)
    flat[1:] = x.reshape(-1)
    wf = torch.zeros(129, device=DEV, dtype=BF16)
    wf[1:] = w
    got = layer_norm_bwd(dy, flat[1:].view(70, 128), wf[1:], b)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    _check(x, dy[:1].expand(70, 128), w, b, True)


@pytest.mark.parametrize("layer_norm", [True, False])
def test_equal_rows_large_means_and_eps(layer_norm):
    x, dy, w, b = _make(33, 1024, F32, F32, mean=300.0)
    _check(x, dy, w, b, layer_norm)
    _check(torch.full_like(x, 3.0), dy, w, b, layer_norm)
    _check(torch.zeros_like(x), dy, w, b, layer_norm)
    if not layer_norm:
        _check(x, dy, w, b, False, 0.0)
        _check(x * 1e-4, dy, w, b, False, 1e-6)


@pytest.mark.parametrize("cols", [64, 1024])
@pytest.mark.parametrize("layer_norm", [True, False])
def test_a_row_that_is_not_finite_stays_alone(layer_norm, cols):
    x, dy, w, b = _make(600, cols, F32, F32)
    clean = _check(x, dy, w, b, layer_norm)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[5, 3] = bad
        got = layer_norm_bwd(dy, y, w, b) if layer_norm else rms_norm_bwd(dy, y, (cols,), w)
        rows = torch.arange(600, device=DEV) != 5
        assert torch.equal(got[0][rows], clean[0][rows])
        assert not torch.isfinite(got[0][5]).all()


@pytest.mark.parametrize("size,scale", [(1e17, 1e17), (1e-12, 1e-30)])
@pytest.mark.parametrize("cols", [64, 1024, 5000])
def test_dots_beyond_the_range_of_32_bits(cols, size, scale):
    """sum(g x) is infinite, or below the smallest 32-bit number, where the gradients are not."""
    x, dy, w, b = _make(40, cols, F32, F32, mean=0.0)
    x[::2] *= size
    dy[::2] *= scale
    got = rms_norm_bwd(dy, x, (cols,), w, 0.0)
    (dx, dw, _), bounds = ref.backward(dy.cpu(), x.cpu(), w.cpu(), 0.0, False)
    # results below the smallest normal number may be flushed
    _held(got[0], dx, bounds[0] + 2.0 ** -126, "dx")
    _held(got[1], dw, bounds[1] + 2.0 ** -126, "dw")


def test_same_bits_each_time_and_in_a_replayed_graph():
    x, dy, w, b = _make(3001, 1000, BF16, BF16)
    want = layer_norm_bwd(dy, x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = layer_norm_bwd(dy, x, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer_norm_bwd(dy, x, w, b)
    for seed in (1, 2, 3):
        y = _make(3001, 1000, BF16, BF16, seed=seed)[0]
        x.copy_(y)
        eager = layer_norm_bwd(dy, y, w, b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager))
