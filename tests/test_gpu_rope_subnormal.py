"""qk_norm_rope of 16-bit vectors so small that their squares, or they themselves, are
subnormal numbers, without eps or with one of their squares' size, against the definition
in 64 bits (oracle/rope.py, whose bounds count the rounding of subnormal sums)."""
import pytest
import torch

from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
from oracle import rope as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _held(got, want, bound, dtype, what):
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all()), what
    off = float(((got - want).abs() / ref.rounded(bound, want, dtype)).max())
    assert off <= 1.0, (what, off)


# accesses of 16 bytes (a power of two of lanes or not), of 4 over the LDS, pair by pair
@pytest.mark.parametrize("dim,n", [(64, 32), (80, 40), (96, 40), (50, 25), (33, 16), (130, 65)])
@pytest.mark.parametrize("dtype,size,eps", [
    (BF16, 1e-21, 0.0),     # squares 1e-42, subnormal in 32 bits
    (BF16, 3e-19, 0.0),     # 9e-38: some above 2^-126, some below
    (BF16, 1e-17, 0.0),
    (BF16, 1e-21, 1e-42),   # an eps of the squares' size
    (F16, 3e-7, 0.0),       # five times the smallest subnormal number
    (F16, 3e-7, 1e-13),
    (F16, 2e-5, 1e-10),
], ids=str)
def test_vectors_of_tiny_values(dim, n, dtype, size, eps):
    print(f"[gpu] {dtype} vectors of {size}, eps {eps}, heads of {dim}", flush=True)
    g = torch.Generator().manual_seed(dim)
    x = (size * (1 + torch.rand(1, 9, 3, dim, generator=g)) *
         torch.randn(1, 9, 3, dim, generator=g).sign()).to(dtype)
    dy = (size * torch.randn(1, 9, 3, dim, generator=g)).to(BF16).to(dtype)
    if dtype == F16:  # gradients of dx's size times the vectors'
        dy = torch.full_like(dy, size)
    w = 1 + 0.3 * torch.randn(dim, generator=g)
    pos, freq = torch.arange(9) * 7, ref.inv_freq(n)
    theta = ref.angles(pos, freq, (1, 9))
    where = (pos.to(DEV), freq.to(DEV))
    for pairing in ("half", "adjacent"):
        got = qk_norm_rope_fwd(x.to(DEV), x.to(DEV), w.to(DEV), w.to(DEV), *where, eps,
                               pairing=pairing)
        want, bound = ref.forward(x, theta, pairing, 1.0, w, eps)
        for out in got:
            _held(out, want, bound, dtype, ("forward", pairing))
        dx, dw, bx, bw = ref.backward(dy, x, theta, pairing, 1.0, w, eps)
        got = qk_norm_rope_bwd(*[t.to(DEV) for t in (dy, dy, x, x, w, w)], *where, eps,
                               pairing=pairing)
        for side in (0, 1):
            _held(got[side], dx, bx, dtype, ("backward", pairing))
            _held(got[2 + side], dw, bw, F32, ("weight", pairing))
