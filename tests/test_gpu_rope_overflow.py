"""qk_norm_rope where products of its formula pass the range of 32 bits though its values
do not: large vectors with large weights or gradients against the definition in 64 bits
(oracle/rope.py), and vectors whose squares pass it, such as rows filled with the type's
lowest value, against rms_norm and rope_fwd one after the other."""
import pytest
import torch

from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
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


@pytest.mark.parametrize("pairing,dtype", HOW, ids=str)
@pytest.mark.parametrize("dim,n", SIZES)
def test_large_vectors_with_large_gradients(dim, n, pairing, dtype):
    """sum(dn w x) passes 1e39, mean(dn w u) is 1e22 at most."""
    print(f"[gpu] large gradients, heads of {dim}, {pairing}, {dtype}", flush=True)
    x, dy, pos, freq, theta, g = _case(dim, n, dtype)
    x, dy = (x.float() * 3e17).to(dtype), (dy.float() * 1e21).to(dtype)
    w = (1 + 0.3 * torch.rand(dim, generator=g)).to(dtype)
    got = qk_norm_rope_bwd(*[t.to(DEV) for t in (dy, dy, x, x, w, w, pos, freq)], EPS,
                           pairing=pairing)
    dx, dw, bx, bw = ref.backward(dy, x, theta, pairing, 1.0, w, EPS)
    for i in (0, 1):
        _held(got[i], dx, bx, dtype, "backward")
        _held(got[2 + i], dw, bw, dtype, "weight")


@pytest.mark.parametrize("pairing,dtype", HOW, ids=str)
@pytest.mark.parametrize("dim,n", SIZES)
def test_gradients_of_rows_of_the_lowest_value(dim, n, pairing, dtype):
    """They are zeros, and add nothing to the weights'; the others keep theirs."""
    print(f"[gpu] gradients at lowest values, heads of {dim}, {pairing}, {dtype}", flush=True)
    x, dy, w, pos, freq, theta, low = _with_lowest_rows(dim, n, dtype)
    got = qk_norm_rope_bwd(*[t.to(DEV) for t in (dy, dy, x, x, w, w, pos, freq)], EPS,
                           pairing=pairing)
    dx, _, bx, _ = ref.backward(dy, x, theta, pairing, 1.0, w, EPS)
    for t in (dy, x):
        t[low] = 0
    _, dw, _, bw = ref.backward(dy, x, theta, pairing, 1.0, w, EPS)
    for i in (0, 1):
        assert not bool(got[i].cpu()[low].any())
        _held(got[i].cpu()[~low], dx[~low], bx[~low], dtype, "backward")
        _held(got[2 + i], dw, bw, dtype, "weight")


# a wave takes one pass of a token, two, and eight, of several tokens
@pytest.mark.parametrize("tokens,hq,hk,dim", [(700, 6, 2, 128), (4200, 32, 8, 128),
                                              (14000, 16, 4, 192)])
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_lowest_rows_leave_the_others_as_they_are(tokens, hq, hk, dim, pairing):
    """The others' gradients are bit for bit those of a call in which such rows are zeros."""
    print(f"[gpu] {tokens} tokens of {hq} + {hk} heads of {dim}, {pairing}", flush=True)
    g = torch.Generator(DEV).manual_seed(dim)
    q, k, gq, gk = (torch.randn(tokens, h, dim, generator=g, device=DEV).to(BF16)
                    for h in (hq, hk, hq, hk))
    w = (1 + 0.3 * torch.randn(dim, generator=g, device=DEV)).to(BF16)
    pos, freq = torch.arange(tokens, device=DEV), ref.inv_freq(dim // 2).to(DEV)
    low = [torch.rand(t.shape[:2], generator=g, device=DEV) < 0.01 for t in (q, k)]
    outs = []
    for fill in (torch.finfo(BF16).min, 0.0):
        x = [t.clone() for t in (q, k)]
        for t, rows in zip(x, low):
            t[rows] = fill
        outs.append(qk_norm_rope_bwd(gq, gk, *x, w, w, pos, freq, EPS, pairing=pairing))
    for i, rows in enumerate(low):
        assert int(rows.sum()) > 0 and not bool(outs[0][i][rows].any())
        assert torch.equal(outs[0][i][~rows], outs[1][i][~rows])
        assert torch.equal(outs[0][2 + i], outs[1][2 + i])


@pytest.mark.parametrize("pairing,dtype", HOW, ids=str)
@pytest.mark.parametrize("dim,n", SIZES)
@pytest.mark.parametrize("size,weight", [(1e-18, 1e22), (1e18, 1e-22)])
def test_sizes_and_weights_of_which_one_is_large_and_one_small(dim, n, pairing, dtype, size,
                                                               weight):
    """1 / sqrt(mean) times the weight is 1e40 or 1e-40, the outputs are 1e22 or 1e-22."""
    print(f"[gpu] vectors of {size}, weights of {weight}, heads of {dim}, {pairing}, {dtype}",
          flush=True)
    x, _, pos, freq, theta, g = _case(dim, n, dtype)
    x = (x.float() * size).to(dtype)
    w = (weight * (1 + torch.rand(dim, generator=g))).to(dtype)
    got = qk_norm_rope_fwd(*[t.to(DEV) for t in (x, x, w, w, pos, freq)], 0.0, pairing=pairing)
    for out in got:
        _held(out, *ref.forward(x, theta, pairing, 1.0, w, 0.0), dtype, "forward")


@pytest.mark.parametrize("pairing,dtype", HOW, ids=str)
@pytest.mark.parametrize("dim,n", SIZES)
@pytest.mark.parametrize("size,gradient,weight", [
    (1e-18, 1e-26, 1.0),   # sum(dn w x) is 1e-42, mean(dn w u) 1e-26
    (1e-18, 1e-29, 1.0),   # its terms are 1e-47, less than the smallest number
    (1e-18, 1e22, 1e-22),  # dn / sqrt(mean) is 1e40, the gradients are 1e18
    (1e18, 1e-22, 1e20),   # dn / sqrt(mean) is 1e-40, the gradients are 1e-20
])
def test_gradients_of_large_and_small_parts(dim, n, pairing, dtype, size, gradient, weight):
    print(f"[gpu] vectors of {size}, gradients of {gradient}, weights of {weight}, heads of "
          f"{dim}, {pairing}, {dtype}", flush=True)
    x, dy, pos, freq, theta, g = _case(dim, n, dtype)
    x, dy = (x.float() * size).to(dtype), (dy.float() * gradient).to(dtype)
    w = (weight * (1 + torch.rand(dim, generator=g))).to(dtype)
    got = qk_norm_rope_bwd(*[t.to(DEV) for t in (dy, dy, x, x, w, w, pos, freq)], 0.0,
                           pairing=pairing)
    dx, dw, bx, bw = ref.backward(dy, x, theta, pairing, 1.0, w, 0.0)
    for i in (0, 1):
        _held(got[i], dx, bx, dtype, "backward")
        _held(got[2 + i], dw, bw, dtype, "weight")
