"""The query / key operators on launches large enough that a wave takes several passes of
a token, walks over several tokens and treats the memory as a stream, against the
definition in 64 bits (oracle/rope.py), which is evaluated on the GPU here: by plain
elementwise work and sums."""
import pytest
import torch

from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
from dslperfgap_amd.viperbench.rope.hip_impl import rope_bwd, rope_fwd
from oracle import rope as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-6


def _held(got, want, bound, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, what
    assert bool(torch.isfinite(got).all()), what
    off = float(((got.double() - want).abs() / ref.rounded(bound, want, dtype)).max())
    assert off <= 1.0, (what, off)


# (batch, tokens of each, query heads, key heads, head size, pairs, type): the passes of a
# token (16-byte accesses of 64 lanes) times the tokens say how many passes a wave takes
CASES = [
    (1, 2000, 32, 8, 128, 64, BF16),    # forward: shares of 4 and 2
    (2, 1500, 12, 4, 128, 64, BF16),    # forward: shares of 3 and 1
    (2, 2100, 32, 8, 128, 64, BF16),    # backward: shares of 2
    (2, 4100, 32, 8, 128, 64, BF16),    # backward: of 4, two at a time
    (1, 14000, 16, 4, 192, 96, BF16),   # backward: of 8, lanes without values
    (1, 14000, 16, 4, 256, 128, F16),   # two rounds of angles
    (1, 9000, 24, 8, 100, 50, BF16),    # accesses of 8 bytes
    (1, 9000, 24, 8, 50, 25, F16),      # accesses of 4 bytes, partners over the LDS
    (2, 10001, 32, 8, 72, 36, BF16),    # lanes no power of two apart: sums over the LDS
    (1, 9000, 15, 5, 96, 24, F32),      # a part that passes
    (1, 9000, 9, 3, 33, 16, F32),       # pair by pair
    (1, 30001, 24, 8, 128, 64, BF16),   # 246 MB written
]


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("b,s,hq,hk,dim,n,dtype", CASES)
def test_large_launches(b, s, hq, hk, dim, n, dtype, pairing):
    print(f"[gpu] large {b} x {s} of {hq} + {hk} heads of {dim}, {dtype} {pairing}", flush=True)
    g = torch.Generator(DEV).manual_seed(s + dim)

    def heads(h):  # heads ahead of the tokens in memory: batch and tokens stay two axes
        return torch.randn(b, h, s, dim, generator=g, device=DEV).to(dtype).transpose(1, 2)

    pos = torch.randint(0, 5000, (b, s), generator=g, device=DEV)
    freq = ref.inv_freq(n).to(DEV)
    theta = ref.angles(pos, freq, (b, s))
    x, dy = [heads(hq), heads(hk)], [heads(hq), heads(hk)]
    w = [1 + 0.3 * torch.randn(dim, generator=g, device=DEV) for _ in x]
    turned = rope_fwd(*x, pos, freq, pairing=pairing)
    back = rope_bwd(*dy, pos, freq, pairing=pairing)
    normed = qk_norm_rope_fwd(*x, *w, pos, freq, EPS, pairing=pairing)
    grads = qk_norm_rope_bwd(*dy, *x, *w, pos, freq, EPS, pairing=pairing)
    for i in range(2):
        _held(turned[i], *ref.forward(x[i], theta, pairing, 1.0), dtype, ("rope_fwd", i))
        _held(back[i], *ref.forward(dy[i], -theta, pairing, 1.0), dtype, ("rope_bwd", i))
        _held(normed[i], *ref.forward(x[i], theta, pairing, 1.0, w[i], EPS), dtype, ("norm", i))
        dx, dw, bx, bw = ref.backward(dy[i], x[i], theta, pairing, 1.0, w[i], EPS)
        _held(grads[i], dx, bx, dtype, ("norm_bwd", i))
        _held(grads[2 + i], dw, bw, F32, ("norm_bwd weight", i))


@pytest.mark.parametrize("dim,n", [(64, 32), (80, 40), (33, 16)])
def test_infinite_gradients_reach_the_weights_as_they_are(dim, n):
    """An infinite gradient of the first vector makes the weight gradients of its pair
    infinite, of the formula's signs (lanes without a vector add no 0 * infinity), and
    leaves the others as they are."""
    print(f"[gpu] infinite gradients, heads of {dim}", flush=True)
    g = torch.Generator().manual_seed(dim)
    x, dy = (torch.randn(1, 5, 3, dim, generator=g) for _ in range(2))
    dy[0, 0, 0, 2] = float("inf")
    w = torch.ones(dim)
    pos, freq = torch.arange(5) + 1, ref.inv_freq(n)
    theta = ref.angles(pos, freq, (1, 5))
    _, want, _, bound = ref.backward(dy, x, theta, "half", 1.0, w, EPS)
    assert int(want.isinf().sum()) == 2 and not bool(want.isnan().any())
    got = qk_norm_rope_bwd(*[t.to(DEV) for t in (dy, dy, x, x, w, w, pos, freq)], EPS)
    rest = want.isfinite()
    for dw in got[2:]:
        dw = dw.cpu()
        assert torch.equal(dw[~rest].double(), want[~rest])
        _held(dw[rest], want[rest], bound[rest], F32, "others")
