"""qk_norm_rope where products of its formula pass the range of 32 bits though its values
do not: large vectors with large weights or gradients against the definition in 64 bits
(oracle/rope.py), and vectors whose squares pass it, such as rows filled with the type's
lowest value, against rms_norm and rope_fwd one after the other."""
import pytest
import torch

from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_fwd
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm
from dslperfgap_amd.viperbench.rope.hip_impl import rope_fwd
from oracle import rope as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-6
# accesses of 16 bytes (a power of two of lanes or not, a part that passes), of 4 over the
# LDS, pair by pair
SIZES = [(64, 32), (80, 40), (96, 40), (50, 25), (33, 16), (130, 65)]
HOW = [("half", F32), ("half", BF16), ("adjacent", F32), ("adjacent", BF16)]


def _held(got, want, bound, dtype, what):
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all()), what
    off = float(((got - want).abs() / ref.rounded(bound, want, dtype)).max())
    assert off <= 1.0, (what, off)


def _case(dim, n, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    x, dy = (torch.randn(1, 11, 3, dim, generator=g).to(dtype) for _ in range(2))
    pos, freq = torch.arange(11) * 5, ref.inv_freq(n)
    return x, dy, pos, freq, ref.angles(pos, freq, (1, 11)), g


@pytest.mark.parametrize("pairing,dtype", HOW, ids=str)
@pytest.mark.parametrize("dim,n", SIZES)
def test_large_vectors_with_large_weights(dim, n, pairing, dtype):
    """|x w| reaches 1e39 and more, the outputs 1e22."""
    print(f"[gpu] large weights, heads of {dim}, {pairing}, {dtype}", flush=True)
    x, _, pos, freq, theta, g = _case(dim, n, dtype)
    x = (x.float() * 3e17).to(dtype)
    w = (1e21 * (1 + torch.rand(dim, generator=g))).to(dtype)
    got = qk_norm_rope_fwd(*[t.to(DEV) for t in (x, x, w, w, pos, freq)], EPS, pairing=pairing)
    for out in got:
        _held(out, *ref.forward(x, theta, pairing, 1.0, w, EPS), dtype, "forward")


def _with_lowest_rows(dim, n, dtype):
    """_case with seven vectors whose squares pass the range of 32 bits; which ones."""
    x, dy, pos, freq, theta, g = _case(dim, n, dtype)
    x[0, 3:5] = torch.finfo(dtype).min
    x[0, 7, 1] = torch.finfo(dtype).max
    w = (2 + torch.rand(dim, generator=g)).to(dtype)
    low = (x.abs() > 1e30).all(-1)
    assert int(low.sum()) == 7
    return x, dy, w, pos, freq, theta, low


@pytest.mark.parametrize("pairing,dtype", HOW, ids=str)
@pytest.mark.parametrize("dim,n", SIZES)
def test_rows_of_the_lowest_value(dim, n, pairing, dtype):
    """1 / sqrt(infinity) is 0, as in rms_norm, and so are the outputs of such vectors; the
    others keep theirs."""
    print(f"[gpu] lowest values, heads of {dim}, {pairing}, {dtype}", flush=True)
    x, _, w, pos, freq, theta, low = _with_lowest_rows(dim, n, dtype)
    xd, wd, pd, fd = (t.to(DEV) for t in (x, w, pos, freq))
    apart = rope_fwd(rms_norm(xd, (dim,), wd, EPS), xd, pd, fd, pairing=pairing)[0].cpu()
    assert not bool(apart[low].any())
    want, bound = ref.forward(x, theta, pairing, 1.0, w, EPS)
    for out in qk_norm_rope_fwd(xd, xd, wd, wd, pd, fd, EPS, pairing=pairing):
        assert not bool(out.cpu()[low].any())
        _held(out.cpu()[~low], want[~low], bound[~low], dtype, "forward")
