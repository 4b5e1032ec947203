"""The norms' gradients of rows so wide that 16 lanes to a column are 2^32 of them and more."""
import pytest
import torch

from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm_bwd
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm_bwd
from oracle import norm_grads as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
PART = 1 << 25


def _row(cols, seed, size, mean):
    g = torch.Generator(DEV).manual_seed(seed)
    return (size * torch.randn(1, cols, generator=g, device=DEV) + mean).to(BF16)


def _sum(f, cols):
    """Of f(slice) over the columns, in 64 bits."""
    return sum(float(f(slice(i, min(i + PART, cols))).sum(dtype=torch.float64))
               for i in range(0, cols, PART))


@pytest.mark.parametrize("layer_norm", [True, False])
@pytest.mark.parametrize("cols", [(1 << 21) + 5, (1 << 28) + 33])
def test_columns_beyond_one_launch(cols, layer_norm):
    """The bounds of oracle/norm_grads.py for one row, part by part; a lane adds up the 1024th part of
    the row, one value after the other."""
    x, dy, w = _row(cols, 1, 2.0, 0.5), _row(cols, 2, 1.0, 0.0), _row(cols, 3, 0.2, 1.0)[0]
    print(f"[gpu] norm_bwd 1 x {cols}, LayerNorm {layer_norm}", flush=True)
    if layer_norm:
        dx, dw, db = layer_norm_bwd(dy, x, w, w)
        assert torch.equal(db, dy[0])  # one row: nothing is added to it
    else:
        dx, dw = rms_norm_bwd(dy, x, (cols,), w)
    steps = ref.STEPS + cols // 1024
    xd, gd = (lambda s: x[0, s].double()), (lambda s: dy[0, s].double() * w[s].double())
    m = _sum(xd, cols) / cols if layer_norm else 0.0
    far = _sum(lambda s: xd(s).abs(), cols) / cols if layer_norm else 0.0
    r = (_sum(lambda s: (xd(s) - m).square(), cols) / cols + 1e-5) ** -0.5
    mean_g = _sum(gd, cols) / cols if layer_norm else 0.0
    mean_gu = _sum(lambda s: gd(s) * (xd(s) - m) * r, cols) / cols
    spread = 1.0 + _sum(lambda s: ((xd(s).abs() + far) * r).square(), cols) / cols
    size_g = _sum(lambda s: gd(s).abs(), cols) / cols
    size_gu = _sum(lambda s: gd(s).abs() * (xd(s).abs() + far) * r, cols) / cols
    for i in range(0, cols, PART):
        s = slice(i, min(i + PART, cols))
        u, big, g = (xd(s) - m) * r, (xd(s).abs() + far) * r, gd(s)
        want = r * (g - mean_g - u * mean_gu)
        bound = steps * ref.ULP * r * spread * (
            g.abs() + big * size_gu + (size_g if layer_norm else 0.0))
        off = (dx[0, s].double() - want).abs() - ref.rounded(bound, want, BF16)
        assert float(off.max()) <= 0.0, ("dx", i, float(off.max()))
        want = dy[0, s].double() * u
        bound = steps * ref.ULP * spread * dy[0, s].double().abs() * big
        off = (dw[s].double() - want).abs() - ref.rounded(bound, want, BF16)
        assert float(off.max()) <= 0.0, ("dw", i, float(off.max()))


def test_more_lanes_in_both_directions():
    """Columns by rows of workgroups, 2^32 lanes and more together: parts of rows against the
    definition, with the rows' statistics in 64 bits."""
    rows, cols = 66, (1 << 26) + 40
    g = torch.Generator(DEV).manual_seed(4)
    x = torch.empty(rows, cols, device=DEV, dtype=BF16).normal_(generator=g)
    dy = torch.empty(rows, cols, device=DEV, dtype=BF16).normal_(generator=g)
    w = _row(cols, 3, 0.2, 1.0)[0]
    print(f"[gpu] layer_norm_bwd {rows} x {cols}", flush=True)
    dx, dw, db = layer_norm_bwd(dy, x, w, w)
    steps = ref.STEPS + cols // 1024
    ends = [slice(0, 4096), slice(cols // 2, cols // 2 + 4096), slice(cols - 4096, cols)]
    want_dw = [torch.zeros(4096, dtype=torch.float64, device=DEV) for _ in ends]
    bound_dw = [torch.zeros_like(t) for t in want_dw]
    for row in range(rows):
        xd, gd = (lambda s: x[row, s].double()), (lambda s: dy[row, s].double() * w[s].double())
        m, far = _sum(xd, cols) / cols, _sum(lambda s: xd(s).abs(), cols) / cols
        r = (_sum(lambda s: (xd(s) - m).square(), cols) / cols + 1e-5) ** -0.5
        mean_g = _sum(gd, cols) / cols
        mean_gu = _sum(lambda s: gd(s) * (xd(s) - m) * r, cols) / cols
        size_g = _sum(lambda s: gd(s).abs(), cols) / cols
        size_gu = _sum(lambda s: gd(s).abs() * (xd(s).abs() + far) * r, cols) / cols
        spread = 1.0 + _sum(lambda s: ((xd(s).abs() + far) * r).square(), cols) / cols
        for i, s in enumerate(ends):
            u, big, gs = (xd(s) - m) * r, (xd(s).abs() + far) * r, gd(s)
            want = r * (gs - mean_g - u * mean_gu)
            bound = steps * ref.ULP * r * spread * (gs.abs() + big * size_gu + size_g)
            off = (dx[row, s].double() - want).abs() - ref.rounded(bound, want, BF16)
            assert float(off.max()) <= 0.0, ("dx", row, i, float(off.max()))
            want_dw[i] += dy[row, s].double() * u
            bound_dw[i] += steps * ref.ULP * spread * dy[row, s].double().abs() * big
    for i, s in enumerate(ends):
        off = (dw[s].double() - want_dw[i]).abs() - ref.rounded(bound_dw[i], want_dw[i], BF16)
        assert float(off.max()) <= 0.0, ("dw", i, float(off.max()))
        want = dy[:, s].double().sum(0)
        bound = 2 * rows * ref.ULP * dy[:, s].double().abs().sum(0)
        off = (db[s].double() - want).abs() - ref.rounded(bound, want, BF16)
        assert float(off.max()) <= 0.0, ("db", i, float(off.max()))
