"""The projection's cross entropy on the GPU against the oracle, within the bounds derived there."""
import pytest
import torch

from dslperfgap_amd.viperbench.layer_norm.hip_impl import layer_norm, layer_norm_bwd
from dslperfgap_amd.viperbench.linear_cross_entropy.hip_impl import (linear_cross_entropy_bwd,
                                                                     linear_cross_entropy_fwd)
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm, rms_norm_bwd
from oracle import linear_ce as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# one value of everything; one token; less than a tile; each height of tiles and its borders; odd
# hidden sizes and vocabularies; several tiles of each kind
SIZES = [(1, 1, 1), (1, 64, 300), (3, 33, 5), (4, 1024, 3200), (31, 100, 1000), (32, 256, 128),
         (33, 256, 777), (64, 72, 130), (65, 128, 300), (256, 64, 256), (257, 200, 513),
         (300, 768, 5003), (700, 129, 1500), (1000, 512, 9000)]
OPTIONS = [dict(), dict(smoothing=0.1, lse_square_scale=1e-3, logit_scale=1.3)]


def _make(tokens, hidden, vocab, dtype, ignored=0.0, seed=0, labels=torch.int64):
    g = torch.Generator(DEV).manual_seed(seed + tokens + 7 * hidden + 13 * vocab)
    w = 1.5 / hidden ** 0.5 * torch.randn(vocab, hidden, generator=g, device=DEV)
    x = torch.randn(tokens, hidden, generator=g, device=DEV)
    lab = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
    drop = torch.randperm(tokens, generator=g, device=DEV)[:round(ignored * tokens)]
    lab[drop] = -100
    dloss = torch.rand(tokens, generator=g, device=DEV) / max(1, tokens)
    return x.to(dtype), w.to(dtype), lab.to(labels), dloss


def _held(got, want, bound, what):
    assert got.shape == want.shape, what
    if got.numel() == 0:
        return
    off = (got.double() - want).abs() - ref.rounded(bound, want, got.dtype)
    assert float(off.max()) <= 0.0, (what, float(off.max()))


def _check(x, w, labels, dloss, **how):
    got = linear_cross_entropy_fwd(x, w, labels, **how)
    want, bounds = ref.forward(x, w, labels, **how)
    for name, p, q, b in zip(("loss", "lse", "z_loss"), got, want, bounds):
        assert p.dtype == F32
        _held(p, q, b, name)
    grads = linear_cross_entropy_bwd(dloss, x, w, got[1], labels, **how)
    want, bounds = ref.backward(dloss, x, w, got[1], labels, **how)
    for name, p, q, b in zip(("dx", "dw"), grads, want, bounds):
        assert p.dtype == x.dtype
        _held(p, q, b, name)
    return got, grads


@pytest.mark.parametrize("ignored", [0.0, 0.4])
@pytest.mark.parametrize("how", OPTIONS)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sizes(dtype, how, ignored):
    for size in SIZES:
        print(f"[gpu] linear_ce {dtype} {size} {how} {ignored}", flush=True)
        _check(*_make(*size, dtype, ignored), **how)


def test_pieces_of_the_vocabulary():
    """dL of more than one piece's bytes: dx is summed over pieces, the last one is shorter."""
    _check(*_make(20001, 64, 16100, BF16, 0.1))


def test_int32_labels_and_other_ignored_values():
    x, w, lab, dloss = _make(300, 64, 500, BF16, 0.3)
    want = linear_cross_entropy_fwd(x, w, lab)
    got = linear_cross_entropy_fwd(x, w, lab.int())
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    lab[lab == -100] = 7
    _check(x, w, lab, dloss, ignored_index=7)


@pytest.mark.parametrize("tokens", [5, 300])
def test_labels_outside_count_nowhere(tokens):
    x, w, lab, dloss = _make(tokens, 64, 500, F32)
    lab[0], lab[1], lab[2] = -3, 500, 1 << 40
    for how in OPTIONS:
        _check(x, w, lab, dloss, **how)


@pytest.mark.parametrize("tokens", [40, 300])
def test_slices_of_the_classes_make_the_whole(tokens):
    x, w, lab, dloss = _make(tokens, 96, 1000, F32, 0.2)
    how = dict(smoothing=0.1, logit_scale=0.9, total_classes=1000)
    parts = [slice(0, 300), slice(300, 1000)]
    fwd = [linear_cross_entropy_fwd(x, w[s], lab, class_start_idx=s.start, SPLIT=True, **how)
           for s in parts]
    for s, got in zip(parts, fwd):
        want, bounds = ref.forward(x, w[s], lab, class_start_idx=s.start, split=True, **how)
        for p, q, b in zip(got, want, bounds):
            _held(p, q, b, "split")
    lse = torch.logaddexp(fwd[0][1], fwd[1][1])
    lse[lab == -100] = 0.0
    whole, bounds = ref.forward(x, w, lab, **how)
    # the two slices' loss parts, the lse's rounding and the sum's
    _held(lse, whole[1], 2 * bounds[1], "lse")
    for s in parts:
        got = linear_cross_entropy_bwd(dloss, x, w[s], lse, lab, class_start_idx=s.start, **how)
        want, b = ref.backward(dloss, x, w[s], lse, lab, class_start_idx=s.start, **how)
        _held(got[0], want[0], b[0], "dx")
        _held(got[1], want[1], b[1], "dw")


@pytest.mark.parametrize("tokens", [20, 300])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_other_layouts_and_offsets(dtype, tokens):
    """Rows apart, rows that are no whole 16-byte pieces, other orders of memory, expanded x."""
    x, w, lab, dloss = _make(tokens, 128, 500, dtype, 0.2)
    want = _check(x, w, lab, dloss)
    for off, width in ((0, 160), (8, 160), (3, 161)):
        xs = torch.full((tokens, width), float("nan"), device=DEV, dtype=dtype)
        ws = torch.full((500, width), float("nan"), device=DEV, dtype=dtype)
        xs[:, off:off + 128], ws[:, off:off + 128] = x, w
        xs, ws = xs[:, off:off + 128], ws[:, off:off + 128]
        for p, q in ((xs, w), (x, ws), (xs, ws)):
            got = linear_cross_entropy_fwd(p, q, lab), linear_cross_entropy_bwd(
                dloss, p, q, want[0][1], lab)
            assert all(torch.equal(s, t) for m, n in zip(got, want) for s, t in zip(m, n))
    got = linear_cross_entropy_fwd(x.T.contiguous().T, w.T.contiguous().T, lab)
    assert all(torch.equal(s, t) for s, t in zip(got, want[0]))
    got = linear_cross_entropy_bwd(dloss.double(), x, w, want[0][1], lab)
    assert all(torch.equal(s, t) for s, t in zip(got, want[1]))
    _check(x[:1].expand(tokens, 128), w, lab, dloss[:1].expand(tokens))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("tokens", [20, 300])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_ignored_tokens_reach_nothing(dtype, tokens, bad):
    x, w, lab, dloss = _make(tokens, 64, 500, dtype, 0.3)
    want = _check(x, w, lab, dloss)
    drop = lab == -100
    x[drop] = bad
    dloss[drop] = bad
    lse = want[0][1].clone()
    lse[drop] = bad
    got = linear_cross_entropy_fwd(x, w, lab), linear_cross_entropy_bwd(dloss, x, w, lse, lab)
    assert all(torch.equal(s, t) for m, n in zip(got, want) for s, t in zip(m, n))
    assert float(got[0][0][drop].abs().max()) == 0.0 and float(got[1][0][drop].abs().max()) == 0.0


@pytest.mark.parametrize("tokens", [0, 7, 300])
@pytest.mark.parametrize("hidden", [64, 33])
def test_no_token_counts(tokens, hidden):
    x, w, lab, dloss = _make(tokens, hidden, 500, BF16)
    lab[:] = -100
    got = linear_cross_entropy_fwd(x, w, lab)
    grads = linear_cross_entropy_bwd(dloss, x, w, got[1], lab)
    for t in (*got, *grads):
        assert torch.equal(t, torch.zeros_like(t))
    assert grads[1].shape == w.shape


def test_without_the_weights_gradient():
    x, w, lab, dloss = _make(300, 64, 5000, BF16, 0.1)
    lse = linear_cross_entropy_fwd(x, w, lab)[1]
    want = linear_cross_entropy_bwd(dloss, x, w, lse, lab)
    got = linear_cross_entropy_bwd(dloss, x, w, lse, lab, weight_grad=False)
    assert got[1] is None and torch.equal(got[0], want[0])


@pytest.mark.parametrize("tokens", [20, 300])
def test_a_token_that_is_not_finite_stays_alone(tokens):
    x, w, lab, dloss = _make(tokens, 64, 500, F32)
    clean = linear_cross_entropy_fwd(x, w, lab)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[3, 5] = bad
        got = linear_cross_entropy_fwd(y, w, lab)
        rows = torch.arange(tokens, device=DEV) != 3
        for p, q in zip(got, clean):
            assert torch.equal(p[rows], q[rows])
        assert torch.isnan(got[0][3]) and torch.isnan(got[1][3])
        dx, dw = linear_cross_entropy_bwd(dloss, y, w, got[1], lab)
        assert torch.isfinite(dx[rows]).all() and not torch.isfinite(dx[3]).any()


@pytest.mark.parametrize("size", [1e-7, 1.0, 1e4])
def test_gradients_of_small_and_large_losses_in_fp16(size):
    """The gradients of the logits lie far below fp16's normal numbers, those of the weights do not
    matter: relative to the loss's they stay as exact."""
    x, w, lab, _ = _make(200, 64, 5000, F16)
    dloss = torch.full((200,), size, device=DEV)
    lse = linear_cross_entropy_fwd(x, w, lab)[1]
    got = linear_cross_entropy_bwd(dloss, x, w, lse, lab)
    want, bounds = ref.backward(dloss, x, w, lse, lab)
    for p, q, b in zip(got, want, bounds):
        _held(p, q, b, "grads")


def test_peaked_and_shifted_logits():
    """Logits of hundreds: one class takes all, and many equal ones share."""
    x, w, lab, dloss = _make(300, 64, 700, F32)
    _check(200 * x, w, lab, dloss)
    _check(torch.zeros_like(x), w, lab, dloss)
    _check(x, 300 * w[:1].expand(700, 64).contiguous() + w, lab, dloss)


def test_weights_beyond_32_bit_offsets():
    tokens, hidden, vocab = 70, 8192, 270000  # 4.4 GB
    x, w, lab, dloss = _make(tokens, hidden, 1000, BF16)
    big = torch.zeros(vocab, hidden, device=DEV, dtype=BF16)
    at = torch.randperm(vocab, generator=torch.Generator().manual_seed(1))[:1000].to(DEV)
    at[0] = vocab - 1
    big[at] = w
    lab = at[lab]
    # the other classes' logits are 0: their exponentials are counted apart
    got = linear_cross_entropy_fwd(x, big, lab)
    logits = torch.matmul(x.double(), w.double().T)
    lse = torch.logaddexp(torch.logsumexp(logits, 1),
                          torch.log(torch.tensor(vocab - 1000.0, dtype=torch.float64, device=DEV)))
    assert float((got[1].double() - lse).abs().max()) < 1e-4
    dx, dw = linear_cross_entropy_bwd(dloss, x, big, got[1], lab)
    d = torch.exp(logits - got[1].double()[:, None])
    d[torch.arange(tokens, device=DEV), (at[None, :] == lab[:, None]).int().argmax(1)] -= 1.0
    d = d * dloss.double()[:, None]
    want = torch.matmul(d.T, x.double())
    size = torch.matmul(d.abs().T, x.double().abs())
    assert float(((dw[at].double() - want).abs() - 2.0 ** -7 * size).max()) <= 1e-9
    want = torch.matmul(d, w.double())
    size = torch.matmul(d.abs(), w.double().abs())
    assert float(((dx.double() - want).abs() - 2.0 ** -7 * size).max()) <= 1e-9


def test_same_bits_each_time_on_another_stream_and_in_a_replayed_graph():
    x, w, lab, dloss = _make(600, 256, 3000, BF16, 0.3)

    def step(x, lab):
        loss, lse, z = linear_cross_entropy_fwd(x, w, lab, lse_square_scale=1e-4)
        return (loss, lse, z, *linear_cross_entropy_bwd(dloss, x, w, lse, lab,
                                                        lse_square_scale=1e-4))

    want = step(x, lab)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x, lab)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(x, lab)
    # other inputs, with other numbers of tokens that count
    for seed, ignored in ((1, 0.0), (2, 0.9), (3, 1.0), (4, 0.5)):
        y, _, other, _ = _make(600, 256, 3000, BF16, ignored, seed)
        x.copy_(y)
        lab.copy_(other)
        eager = step(y, other)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, eager))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layer", [True, False])
def test_a_training_head_as_it_is_used(dtype, layer):
    """Final norm, projection and loss, and back, against automatic differentiation of the whole
    in 64 bits."""
    g = torch.Generator(DEV).manual_seed(9)
    tokens, hidden, vocab = 391, 320, 2003
    h = torch.randn(tokens, hidden, generator=g, device=DEV).to(dtype)
    gain = (1 + 0.1 * torch.randn(hidden, generator=g, device=DEV)).to(dtype)
    bias = (0.1 * torch.randn(hidden, generator=g, device=DEV)).to(dtype)
    w = (torch.randn(vocab, hidden, generator=g, device=DEV) / hidden ** 0.5).to(dtype)
    lab = torch.randint(0, vocab, (tokens,), generator=g, device=DEV)
    lab[::3] = -100
    n = int((lab != -100).sum())
    x = layer_norm(h, gain, bias) if layer else rms_norm(h, (hidden,), gain, 1e-5)
    loss, lse, _ = linear_cross_entropy_fwd(x, w, lab)
    dloss = torch.full((tokens,), 1.0 / n, device=DEV)
    dx, dw = linear_cross_entropy_bwd(dloss, x, w, lse, lab)
    if layer:
        dh, dgain, dbias = layer_norm_bwd(dx, h, gain, bias)
    else:
        (dh, dgain), dbias = rms_norm_bwd(dx, h, (hidden,), gain, 1e-5), None

    leaves = [t.double().requires_grad_() for t in (h, gain, bias, w)]
    hd, gd, bd, wd = leaves
    d = hd - hd.mean(1, keepdim=True) if layer else hd
    y = d / (d.square().mean(1, keepdim=True) + 1e-5).sqrt() * gd + (bd if layer else 0 * bd)
    whole = torch.nn.functional.cross_entropy(torch.matmul(y, wd.T), lab, ignore_index=-100)
    want = torch.autograd.grad(whole, leaves)
    eps = torch.finfo(dtype).eps
    assert abs(float(loss.sum() / n) - float(whole.detach())) < 8 * eps + 1e-5
    # each array is rounded to the type once where it is made: x, dL, dx, and the result, by half
    # a step each; in the norm of a whole array those are at most 4 half steps of relative size,
    # and the rounded x enters twice more (logits and dw): 8 half steps in all
    tol = 4 * eps + 1e-5
    for got, ref64 in zip((dh, dgain, dbias, dw), want):
        if got is None:
            continue
        assert float((got.double() - ref64).norm() / ref64.norm()) < tol
