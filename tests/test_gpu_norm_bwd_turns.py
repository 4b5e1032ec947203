"""The norms' gradients where a workgroup goes over three rows and more of five to eight vectors a
lane, with the next row on its way into the LDS (whole rows) or in registers (ragged ones)."""
import pytest
import torch

from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd
from oracle import norm_grads as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("layer_norm", [True, False])
@pytest.mark.parametrize("dtype,wdtype,rows,cols", [
    (BF16, BF16, 700, 24576), (F16, F32, 700, 24568), (BF16, F32, 700, 32768), (F16, F16, 700, 28680),
    (BF16, F32, 1030, 16392), (BF16, BF16, 600, 16393), (F16, F32, 600, 24570), (BF16, BF16, 600, 30001),
    (F32, F32, 700, 12288), (F32, F32, 700, 16384), (F32, F32, 600, 8201), (F32, F32, 600, 12001),
    (F32, F32, 600, 16381)])
def test_rows_of_many_vectors_in_turn(dtype, wdtype, rows, cols, layer_norm):
    print(f"[gpu] norm_bwd turns {dtype} {wdtype} {rows} x {cols}", flush=True)
    g = torch.Generator(DEV).manual_seed(rows + 7 * cols)
    x = (2 * torch.randn(rows, cols, generator=g, device=DEV) + 0.5).to(dtype)
    dy = torch.randn(rows, cols, generator=g, device=DEV).to(dtype)
    w = (1 + 0.2 * torch.randn(cols, generator=g, device=DEV)).to(wdtype)
    if layer_norm:
        got = layer_norm_bwd(dy, x, w, w)
        again = layer_norm_bwd(dy, x, w, w)
    else:
        got = rms_norm_bwd(dy, x, (cols,), w)
        again = rms_norm_bwd(dy, x, (cols,), w)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    want, bounds = ref.backward(dy.cpu(), x.cpu(), w.cpu(), 1e-5, layer_norm)
    for name, p, q, b in zip(("dx", "dw", "db"), got, want, bounds):
        off = (p.cpu().double() - q).abs() - ref.rounded(b, q, p.dtype)
        assert float(off.max()) <= 0.0, (name, float(off.max()))
