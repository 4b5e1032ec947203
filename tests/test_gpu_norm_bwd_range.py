"""The norms' gradients of rows whose sum(g x) is beyond the range of 32 bits, among rows whose is
not, in each way that rows lie over lanes."""
import pytest
import torch

from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd
from oracle import norm_grads as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("scale", [2e21, 1e23])
@pytest.mark.parametrize("layer_norm", [True, False])
@pytest.mark.parametrize("dtype,rows,cols", [
    (F32, 40, 64), (F32, 2100, 100), (F32, 40, 1024), (BF16, 600, 1001), (F32, 600, 5000),
    (F32, 300, 12000), (F32, 300, 16384), (BF16, 700, 20480), (BF16, 600, 24576), (BF16, 300, 32768),
    (BF16, 300, 20481), (F32, 10, 40000)])
def test_sums_beyond_the_largest_number(dtype, rows, cols, layer_norm, scale):
    g = torch.Generator(DEV).manual_seed(rows + 7 * cols)
    x, dy = (torch.randn(rows, cols, generator=g, device=DEV) for _ in range(2))
    w = 1 + 0.2 * torch.randn(cols, generator=g, device=DEV)
    x[::2] *= 2e16
    # g in line with x, so that its products with x add up
    dy[::2] = scale * (dy[::2] + x[::2].sign())
    x, dy, w = x.to(dtype), dy.to(dtype), w.to(dtype)
    dots = (dy.double() * w.double() * x.double()).sum(1).abs()
    assert float(dots[::2].min()) > 2.0 ** 127 > float(dots[1::2].max())
    assert float(x.double().square().sum(1).max()) < 2.0 ** 127
    if layer_norm:
        got = layer_norm_bwd(dy, x, w, w)
    else:
        got = rms_norm_bwd(dy, x, (cols,), w)
    want, bounds = ref.backward(dy.cpu(), x.cpu(), w.cpu(), 1e-5, layer_norm)
    for name, p, q, b in zip(("dx", "dw", "db"), got, want, bounds):
        assert torch.isfinite(q).all() and torch.isfinite(p).all(), name
        off = (p.cpu().double() - q).abs() - ref.rounded(b, q, p.dtype)
        assert float(off.max()) <= 0.0, (name, float(off.max()))


@pytest.mark.parametrize("layer_norm", [True, False])
@pytest.mark.parametrize("dtype,rows,cols", [
    (F32, 40, 64), (BF16, 600, 1001), (F32, 300, 12000), (BF16, 700, 20480), (BF16, 300, 20481),
    (F32, 10, 40000)])
def test_rows_whose_squares_are_infinite_have_no_gradient(dtype, rows, cols, layer_norm):
    """Their forward is constant in 32 bits: rows of dx are 0, and nothing of them enters dw."""
    g = torch.Generator(DEV).manual_seed(rows + 7 * cols)
    x, dy = (torch.randn(rows, cols, generator=g, device=DEV).to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(cols, generator=g, device=DEV)).to(dtype)
    x[::2] *= 1e25
    far = torch.arange(rows, device=DEV) % 2 == 0
    kept = dy.clone()
    kept[far] = 0.0
    small = x.clone()
    small[far] = 0.0

    def run(dy, x):
        return layer_norm_bwd(dy, x, w, w) if layer_norm else rms_norm_bwd(dy, x, (cols,), w)

    got, want = run(dy, x), run(kept, small)
    assert float(got[0][far].abs().max()) == 0.0
    assert torch.equal(got[0], want[0])
    assert torch.equal(got[1], want[1])
