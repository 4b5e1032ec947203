"""The query / key operators on the GPU against the definition in 64 bits, value by value
within bounds that follow from the arithmetic (oracle/rope.py): every width of piece, both
pairings, one to four axes, the layouts that users hold their projections in, and what
lies at the edges (no tokens, one token, infinities, far positions, other streams and
graphs).
"""
import ctypes

import pytest
import torch

from dslperfgap_amd import _lib, _rope
from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
from dslperfgap_amd.viperbench.rms_norm.hip_impl import rms_norm
from dslperfgap_amd.viperbench.rope.hip_impl import rope_bwd, rope_fwd
from dslperfgap_amd.viperbench.softmax.hip_impl import softmax
from oracle import rope as ref

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EPS = 1e-6


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _heads(shape, dtype, g, layout="separate", scale=1.0):
    b, s, h, d = shape
    x = (scale * torch.randn(b, s, h, d, generator=g)).to(dtype)
    if layout == "heads_first":
        return x, x.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "packed":  # a slice of a wider projection, off the 16-byte boundary
        whole = torch.zeros(b, s, h + 3, d, dtype=dtype, device=DEV)
        whole[:, :, 2:2 + h] = x.to(DEV)
        return x, whole[:, :, 2:2 + h]
    if layout == "strided":  # vectors that are not contiguous
        whole = torch.zeros(b, s, h, d, 2, dtype=dtype, device=DEV)
        whole[..., 1] = x.to(DEV)
        return x, whole[..., 1]
    return x, x.to(DEV)


def _held(got, want, bound, dtype, what):
    assert got.dtype == dtype and got.shape == want.shape, what
    got = got.cpu().double()
    assert bool(torch.isfinite(got).all()), what
    off = (got - want).abs() / ref.rounded(bound, want, dtype)
    assert float(off.max() if off.numel() else 0.0) <= 1.0, (what, float(off.max()))


def _check(lead=(2, 37), hq=4, hk=2, dim=64, n=None, dtype=F32, wdtype=None, pairing="half",
           sections=None, order="blocks", pos_dtype=torch.int64, first=0, one_row=False,
           layout="separate", scale=1.0, weights=(True, True), freq_dtype=F32, eps=EPS, seed=0):
    g = _gen(seed)
    b, s = lead
    n = dim // 2 if n is None else n
    axes = 1 if sections is None else len(sections)
    rows = (s,) if one_row else (b, s)
    pos = torch.randint(0, 5000, (axes, *rows) if axes > 1 else rows, generator=g)
    pos = (pos + first).to(pos_dtype)
    freq = ref.inv_freq(n, dtype=freq_dtype)
    theta = ref.angles(pos, freq, (b, s), sections, order)
    where = (pos.to(DEV), freq.to(DEV))
    how = dict(sections=sections, section_order=order, pairing=pairing, scale=scale)
    (q, qd), (k, kd) = (_heads((b, s, h, dim), dtype, g, layout, 2.0) for h in (hq, hk))
    (gq, gqd), (gk, gkd) = (_heads((b, s, h, dim), dtype, g, layout) for h in (hq, hk))
    wd = dtype if wdtype is None else wdtype
    ws = [(1 + 0.3 * torch.randn(dim, generator=g)).to(wd) if there else None for there in weights]
    wsd = [None if w is None else w.to(DEV) for w in ws]

    def both(got, x, op, **kw):
        for out, xx, w, name in zip(got, x, ws, "qk"):
            want, bound = ref.forward(xx, kw.pop("theta", theta), pairing, scale,
                                      w if "eps" in kw else None, kw.get("eps"))
            assert out.is_contiguous()
            _held(out, want, bound, dtype, (op, name))

    both(rope_fwd(qd, kd, *where, **how), (q, k), "rope_fwd")
    for out, x, name in zip(rope_bwd(gqd, gkd, *where, **how), (gq, gk), "qk"):
        want, bound = ref.forward(x, -theta, pairing, scale)
        _held(out, want, bound, dtype, ("rope_bwd", name))
    both(qk_norm_rope_fwd(qd, kd, *wsd, *where, eps, **how), (q, k), "norm_fwd", eps=eps)
    got = qk_norm_rope_bwd(gqd, gkd, qd, kd, *wsd, *where, eps, **how)
    for i, (dy, x, w) in enumerate(((gq, q, ws[0]), (gk, k, ws[1]))):
        dx, dw, bx, bw = ref.backward(dy, x, theta, pairing, scale, w, eps)
        _held(got[i], dx, bx, dtype, ("norm_bwd", "qk"[i]))
        if w is None:
            assert got[2 + i] is None
        else:
            _held(got[2 + i], dw, bw, wd, ("norm_bwd weight", "qk"[i]))


# every width of piece: 8, 4, 2 and 1 values, one to 64 lanes a vector, lanes that hold
# nothing (80, 96, 192), value by value along a wave (250, 510, 1023), partial rotation
SIZES = [(2, 1), (3, 1), (8, 4), (16, 8), (20, 10), (33, 16), (64, 32), (65, 32), (72, 36),
         (80, 40), (80, 10), (96, 48), (100, 50), (128, 64), (128, 32), (128, 3), (192, 96),
         (250, 125), (256, 128),
         (50, 25), (66, 33), (24, 6), (120, 15), (104, 52), (36, 7), (42, 10), (126, 63), (510, 255), (512, 256), (1023, 511), (1024, 512), (1024, 100)]


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("dim,n", SIZES)
def test_head_sizes(dim, n, dtype, pairing):
    print(f"[gpu] head size {dim}, {n} pairs, {dtype}, {pairing}", flush=True)
    _check(lead=(1, 19), hq=3, hk=2, dim=dim, n=n, dtype=dtype, pairing=pairing, seed=dim)


@pytest.mark.parametrize("lead", [(1, 1), (1, 2), (5, 1), (1, 63), (64, 1), (3, 33), (7, 3),
                                  (1, 1000), (2, 1025)])
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 8), (32, 8), (7, 1), (33, 2), (2, 30)])
def test_tokens_and_heads(lead, hq, hk):
    print(f"[gpu] tokens {lead}, heads {hq} + {hk}", flush=True)
    _check(lead=lead, hq=hq, hk=hk, dim=64, dtype=BF16, seed=hq)


@pytest.mark.parametrize("layout", ["separate", "packed", "heads_first", "strided"])
@pytest.mark.parametrize("one_row", [False, True])
@pytest.mark.parametrize("dtype,dim", [(F32, 48), (BF16, 128), (F16, 72), (BF16, 33)])
def test_layouts(layout, one_row, dtype, dim):
    print(f"[gpu] layout {layout}, {dtype}, {dim}", flush=True)
    _check(lead=(3, 29), hq=6, hk=3, dim=dim, dtype=dtype, layout=layout, one_row=one_row)


@pytest.mark.parametrize("sections,order", [((16, 24, 24), "blocks"), ((24, 20, 20), "cycle"),
                                            ((32, 32), "cycle"), ((10, 54), "blocks"),
                                            ((0, 64), "blocks"), ((40, 8, 10, 6), "blocks"),
                                            ((52, 4, 0, 8), "cycle"), ((64,), "blocks")])
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("one_row", [False, True])
def test_axes(sections, order, pairing, one_row):
    print(f"[gpu] sections {sections} {order} {pairing}", flush=True)
    _check(lead=(2, 31), dim=144, n=64, dtype=F32, sections=sections, order=order,
           pairing=pairing, one_row=one_row)


@pytest.mark.parametrize("how", [
    {"wdtype": F32}, {"wdtype": F32, "pairing": "adjacent"}, {"weights": (False, True)},
    {"weights": (True, False)}, {"weights": (False, False)}, {"scale": 1.2079}, {"scale": -0.5},
    {"freq_dtype": torch.float64}, {"pos_dtype": torch.int32}, {"pos_dtype": F32},
    {"eps": 0.0}, {"eps": 1e-2}], ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_options(how, dtype):
    print(f"[gpu] options {how}", flush=True)
    _check(dim=128, dtype=dtype, **how)


def test_weights_of_other_types_are_widened_and_their_gradients_narrowed():
    print("[gpu] weight types", flush=True)
    g = _gen(5)
    q, k = (torch.randn(9, 2, 32, generator=g).bfloat16().to(DEV) for _ in "qk")
    pos, freq = torch.arange(9, device=DEV), ref.inv_freq(16).to(DEV)
    w = torch.randn(32, generator=g)
    want = qk_norm_rope_bwd(q, k, q, k, w.to(DEV), w.to(DEV), pos, freq)
    for qw, kw in ((w.double(), w), (w, w.double()), (w.double(), w.double())):
        got = qk_norm_rope_bwd(q, k, q, k, qw.to(DEV), kw.to(DEV), pos, freq)
        assert [t.dtype for t in got[2:]] == [qw.dtype, kw.dtype]
        for a, b in zip(got, want):
            assert torch.equal(a.to(b.dtype), b)
    got = qk_norm_rope_fwd(q, k, w.half().to(DEV), w.bfloat16().to(DEV), pos, freq)
    want = qk_norm_rope_fwd(q, k, w.half().float().to(DEV), w.bfloat16().float().to(DEV), pos, freq)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    strided = torch.stack([w, w], 1).to(DEV)[:, 0]
    got = qk_norm_rope_fwd(q, k, strided, strided, pos, freq)
    want = qk_norm_rope_fwd(q, k, w.to(DEV), w.to(DEV), pos, freq)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("first", [-4000, 1 << 20, (1 << 31) - 5001, 1 << 40, -(1 << 40)])
def test_far_positions(first):
    """A position times a frequency is formed with a relative error of 2^-52: at 2^40 the
    angle (2^40 radians at most) is off by 2^-12, below that in proportion."""
    print(f"[gpu] positions from {first}", flush=True)
    if abs(first) < 1 << 32:
        _check(dim=64, first=first, seed=3)
        return
    g = _gen(8)
    q, k = (torch.randn(33, 2, 64, generator=g) for _ in "qk")
    pos, freq = torch.arange(33) + first, ref.inv_freq(32)
    theta = ref.angles(pos, freq, (1, 33))
    got = rope_fwd(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV))
    for out, x in zip(got, (q, k)):
        want = ref.forward(x[None], theta, "half")[0][0]
        size = ref.turn(x[None].double(), theta, "half", size=True)[0]
        bound = 2.0 ** -52 * 2.2 * theta[0].abs()[:, None].repeat(1, 1, 2) * size + 1e-6 * size
        assert bool(((out.cpu().double() - want).abs() <= bound).all())


def test_positions_are_read_through_their_strides():
    print("[gpu] strided positions", flush=True)
    g = _gen(9)
    q, k = (torch.randn(2, 5, h, 32, generator=g).to(DEV) for h in (3, 1))
    freq = ref.inv_freq(16).to(DEV)
    wide = torch.randint(0, 900, (5, 2, 3, 4), generator=g).to(DEV)
    pos = wide.permute(2, 1, 0, 3)[..., 1]  # [3, 2, 5] of strides 4, 12, 24
    how = dict(sections=(6, 5, 5))
    got = rope_fwd(q, k, pos, freq, **how)
    want = rope_fwd(q, k, pos.contiguous(), freq, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = rope_fwd(q, k, pos[0, :1].expand(2, 5), freq)
    want = rope_fwd(q, k, pos[0, 0].contiguous(), freq)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = q[:, :, :1].expand(2, 5, 4, 32)  # one stored head for all
    got = rope_fwd(one, k, pos, freq, **how)[0]
    assert torch.equal(got, rope_fwd(one.contiguous(), k, pos, freq, **how)[0])


@pytest.mark.parametrize("shape", [(0, 4, 2), (2, 0, 4), (3, 0, 0)])
def test_nothing_to_do(shape):
    print(f"[gpu] empty {shape}", flush=True)
    s, hq, hk = shape
    q, k = (torch.ones(s, h, 64, device=DEV) for h in (hq, hk))
    pos, freq = torch.arange(s, device=DEV), ref.inv_freq(32).to(DEV)
    w = torch.ones(64, device=DEV)
    for out in (rope_fwd(q, k, pos, freq), rope_bwd(q, k, pos, freq),
                qk_norm_rope_fwd(q, k, w, w, pos, freq)):
        assert out[0].shape == q.shape and out[1].shape == k.shape
    dq, dk, dqw, dkw = qk_norm_rope_bwd(q, k, q, k, w, w, pos, freq)
    assert dq.shape == q.shape and dk.shape == k.shape
    if hq == 0 or s == 0:
        assert not bool(dqw.any())
    if hk == 0 or s == 0:
        assert not bool(dkw.any())
    if s and hk:  # the other side's work is done
        want = rope_fwd(k, k, pos, freq)[1]
        assert torch.equal(rope_fwd(q, k, pos, freq)[1], want)


@pytest.mark.parametrize("dim,n,pairing", [(128, 32, "half"), (128, 32, "adjacent"),
                                           (65, 20, "half"), (65, 20, "adjacent"),
                                           (96, 44, "adjacent")])
def test_infinities_stay_where_they_belong(dim, n, pairing):
    """A rotation's infinity reaches its pair and no other value, in the part that passes
    itself alone; a norm's reaches its vector alone.  NaN likewise."""
    print(f"[gpu] infinities {dim} {n} {pairing}", flush=True)
    g = _gen(11)
    x = torch.randn(6, 3, dim, generator=g)
    how = {"pairing": pairing}
    pos, freq = torch.arange(6) + 1, ref.inv_freq(n)
    clean = rope_fwd(x.to(DEV), x.to(DEV), pos.to(DEV), freq.to(DEV), **how)[0].cpu()
    w = torch.ones(dim, device=DEV)
    clean_n = qk_norm_rope_fwd(x.to(DEV), x.to(DEV), w, w, pos.to(DEV), freq.to(DEV), **how)[0].cpu()
    clean_b = qk_norm_rope_bwd(*[x.to(DEV)] * 4, w, w, pos.to(DEV), freq.to(DEV), **how)[0].cpu()
    first, second = ref.pairs(n, pairing)
    for bad in (float("inf"), float("-inf"), float("nan")):
        for at in (0, 3, 2 * n - 1, 2 * n, dim - 1):
            y = x.clone()
            y[2, 1, at] = bad
            yd = y.to(DEV)
            got = rope_fwd(yd, yd, pos.to(DEV), freq.to(DEV), **how)[0].cpu()
            touched = {at}
            for a, b in zip(first, second):
                if at in (a, b):
                    touched = {a, b}
            rest = [i for i in range(dim) if i not in touched]
            assert torch.equal(got[2, 1, rest], clean[2, 1, rest])
            assert not bool(torch.isfinite(got[2, 1, list(touched)]).any())
            got_n = qk_norm_rope_fwd(yd, yd, w, w, pos.to(DEV), freq.to(DEV), **how)[0].cpu()
            got_b = qk_norm_rope_bwd(*[yd] * 4, w, w, pos.to(DEV), freq.to(DEV), **how)[0].cpu()
            assert not bool(torch.isfinite(got_n[2, 1, at]))
            assert not bool(torch.isfinite(got_b[2, 1, at]))
            for o, c in ((got, clean), (got_n, clean_n), (got_b, clean_b)):
                o, c = o.clone(), c.clone()
                o[2, 1] = c[2, 1] = 0
                assert torch.equal(o, c)


def test_zero_vectors_and_lowest_values():
    """A vector of zeros: outputs 0, gradient dn w / sqrt(eps); one of the type's lowest
    value where its square still fits 32 bits, and tiny ones without eps."""
    print("[gpu] zeros and extremes", flush=True)
    pos, freq = torch.arange(3), ref.inv_freq(32)
    theta = ref.angles(pos, freq, (1, 3))
    where = (pos.to(DEV), freq.to(DEV))
    w = torch.linspace(0.5, 1.5, 64)
    for dtype, fill, eps in ((F32, 0.0, EPS), (BF16, 0.0, EPS), (F16, torch.finfo(F16).min, EPS),
                             (F32, 1e-21, 0.0), (F32, 1e17, EPS), (BF16, -3e17, EPS)):
        x = torch.full((1, 3, 2, 64), fill, dtype=dtype)
        dy = torch.randn(1, 3, 2, 64, generator=_gen(1)).to(dtype)
        y = qk_norm_rope_fwd(x.to(DEV), x.to(DEV), w.to(DEV), w.to(DEV), *where, eps)[0]
        want, bound = ref.forward(x, theta, "half", 1.0, w, eps)
        _held(y, want, bound, dtype, ("forward", fill))
        dx, dw, bx, bw = ref.backward(dy, x, theta, "half", 1.0, w, eps)
        if float(dx.abs().max()) < float(torch.finfo(dtype).max) / 4:
            got = qk_norm_rope_bwd(*[t.to(DEV) for t in (dy, dy, x, x, w, w)], *where, eps)
            _held(got[0], dx, bx, dtype, ("backward", fill))
            _held(got[2], dw, bw, F32, ("weights", fill))


def test_gradients_are_the_slopes():
    """Directional differences of the 64-bit forward against the kernel's gradients: the
    difference quotient is off by its second order, h^2 |f'''| / 6, and the gradient by the
    sum of its bounds."""
    print("[gpu] slopes", flush=True)
    g = _gen(21)
    x = torch.randn(1, 40, 3, 48, generator=g)
    w = 1 + 0.3 * torch.randn(48, generator=g)
    dy = torch.randn(1, 40, 3, 48, generator=g)
    pos, freq = torch.arange(40), ref.inv_freq(24)
    theta = ref.angles(pos, freq, (1, 40))
    got = qk_norm_rope_bwd(*[t.to(DEV) for t in (dy, dy, x, x, w, w, pos, freq)])
    _, _, bx, bw = ref.backward(dy, x, theta, "half", 1.0, w, EPS)

    def f(x, w):
        return float((ref.forward(x, theta, "half", 1.0, w, EPS)[0] * dy.double()).sum())

    h = 1e-5
    v = torch.randn(x.shape, generator=g).double()
    slope = (f(x.double() + h * v, w.double()) - f(x.double() - h * v, w.double())) / (2 * h)
    mine = float((got[1].cpu().double() * v).sum())
    assert abs(slope - mine) <= float((bx * v.abs()).sum()) + 1e-6
    u = torch.randn(48, generator=g).double()
    slope = (f(x.double(), w.double() + h * u) - f(x.double(), w.double() - h * u)) / (2 * h)
    assert abs(slope - float((got[3].cpu().double() * u).sum())) <= float((bw * u.abs()).sum()) + 1e-6


def _case(tokens=300, hq=8, hk=2, dim=128, dtype=BF16, seed=31, dev=DEV):
    g = _gen(seed)
    q, k, gq, gk = (torch.randn(tokens, h, dim, generator=g).to(dtype).to(dev)
                    for h in (hq, hk, hq, hk))
    w = [(1 + 0.2 * torch.randn(dim, generator=g)).to(dtype).to(dev) for _ in "qk"]
    pos = torch.randint(0, 9000, (tokens,), generator=g).to(dev)
    return q, k, gq, gk, w, pos, ref.inv_freq(dim // 2).to(dev)


def _all(q, k, gq, gk, w, pos, freq):
    return [*rope_fwd(q, k, pos, freq), *rope_bwd(gq, gk, pos, freq),
            *qk_norm_rope_fwd(q, k, *w, pos, freq), *qk_norm_rope_bwd(gq, gk, q, k, *w, pos, freq)]


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_same_call_gives_the_same_bits_on_any_stream():
    print("[gpu] determinism, streams", flush=True)
    case = _case(tokens=3001)
    want = _all(*case)
    inputs = [t.clone() for t in (*case[:4], *case[4], *case[5:])]
    for _ in range(3):
        assert _same(_all(*case), want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for s in streams * 2:  # several in flight at once
        with torch.cuda.stream(s):
            outs.append(_all(*case))
    torch.cuda.synchronize()
    assert all(_same(o, want) for o in outs)
    assert _same(inputs, (*case[:4], *case[4], *case[5:]))  # inputs are left as they were


def test_captured_calls_replay():
    """One graph of all four operators (a second one beside it, with workspaces of its own),
    replayed with new inputs between other work."""
    print("[gpu] graphs", flush=True)
    one, two = _case(seed=41), _case(tokens=517, hq=4, hk=4, dim=64, dtype=F16, seed=42)
    _all(*one), _all(*two)
    graphs, outs = [], []
    for case in (one, two):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_all(*case))
        graphs.append(gr)
    for i in range(4):
        for case, seed in ((one, 50 + i), (two, 60 + i)):
            fresh = _case(*((300, 8, 2, 128, BF16) if case is one else (517, 4, 4, 64, F16)), seed)
            for a, b in zip((*case[:4], *case[4], case[5]), (*fresh[:4], *fresh[4], fresh[5])):
                a.copy_(b)
        for gr in graphs:
            gr.replay()
        eager = [_all(*one), _all(*two)]
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            assert _same(got, want), i


@pytest.mark.parametrize("dim,dtype", [(128, BF16), (33, F32), (80, F16)])
def test_memory_around_the_outputs_is_left_alone(dim, dtype):
    """Outputs, weights' gradients and the workspace inside larger buffers: what lies around
    keeps its values."""
    print(f"[gpu] guards {dim} {dtype}", flush=True)
    q, k, gq, gk, w, pos, freq = _case(tokens=67, hq=5, hk=3, dim=dim, dtype=dtype)
    want = qk_norm_rope_bwd(gq, gk, q, k, *w, pos, freq)
    _, desc, _, _, _, _, ws_bytes, _kept = _rope.make_plan(
        "qk_norm_rope_bwd", q, k, pos, freq, None, "blocks", "half", 1.0, EPS, tuple(w), (gq, gk))
    bufs = []

    def guarded(n, dt):
        b = torch.full((n + 256,), 7.0, dtype=dt, device=DEV)
        bufs.append((b, n))
        return b[128:].data_ptr()

    ptrs = [guarded(t.numel(), t.dtype) for t in want]
    ws = guarded(ws_bytes // 4, F32)
    _lib.call("vbh_qk_norm_rope_bwd", desc, gq.data_ptr(), gk.data_ptr(), q.data_ptr(),
              k.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), pos.data_ptr(), freq.data_ptr(),
              *ptrs, ws, ws_bytes, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for (b, n), t in zip(bufs, want):
        assert torch.equal(b[128:128 + n], t.reshape(-1))
    for b, n in bufs:
        assert bool((b[:128] == 7).all()) and bool((b[128 + n:] == 7).all())


def test_a_non_contiguous_pass_off_the_vector_boundary():
    """Operands that start and step off 16-byte boundaries give the same values."""
    print("[gpu] misaligned operands", flush=True)
    q, k, gq, gk, w, pos, freq = _case(tokens=45)
    want = _all(q, k, gq, gk, w, pos, freq)

    def shifted(t):
        flat = torch.zeros(t.numel() + 8, dtype=t.dtype, device=DEV)
        flat[1:1 + t.numel()] = t.reshape(-1)
        return flat[1:1 + t.numel()].view(t.shape)

    got = _all(*[shifted(t) for t in (q, k, gq, gk)], [shifted(t) for t in w], shifted(pos),
               shifted(freq))
    assert _same(got, want)


def test_long_operands_pass_32_bit_offsets():
    """Tokens whose element offsets pass 2^32, through strides (few vectors are stored)."""
    print("[gpu] long strides", flush=True)
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 18 GB of device memory")
    stride = (1 << 31) + 128
    flat = torch.zeros(4 * stride + 4096, dtype=BF16, device=DEV)
    x = flat.as_strided((5, 2, 128), (stride, 128, 1))
    src = torch.randn(5, 2, 128, generator=_gen(2)).bfloat16().to(DEV)
    x.copy_(src)
    pos, freq = torch.arange(5, device=DEV) * 700, ref.inv_freq(64).to(DEV)
    w = torch.ones(128, dtype=BF16, device=DEV)
    assert _same(_all(x, x, x, x, [w, w], pos, freq), _all(src, src, src, src, [w, w], pos, freq))


def test_attention_block_forward_and_backward():
    """The operators as a model runs them: rms_norm, a projection, per-head norm and rotation
    of its slices, softmax over the scores; then back to the projection's gradient and the
    norms' weights, against automatic differentiation in 64 bits."""
    print("[gpu] attention block", flush=True)
    g = _gen(77)
    b, s, hq, hk, d, width = 2, 24, 4, 2, 32, 96
    x = torch.randn(b * s, width, generator=g)
    proj = torch.randn(width, (hq + 2 * hk) * d, generator=g) / width ** 0.5
    nw, qw, kw = (1 + 0.2 * torch.randn(n, generator=g) for n in (width, d, d))
    pos = torch.stack([torch.arange(s), torch.arange(s) // 4, torch.arange(s) % 4])
    freq = ref.inv_freq(16)
    how = dict(sections=(6, 5, 5), section_order="cycle", pairing="adjacent")
    dout = torch.randn(b, hq, s, d, generator=g)

    def attend(q, k, v, soft):  # [b, h, s, d]
        k, v = (t.repeat_interleave(hq // hk, 1) for t in (k, v))
        return soft(q @ k.transpose(-1, -2).contiguous() / d ** 0.5), v

    xd, pd, nd, qd, kd, posd, fd = (t.to(DEV) for t in (x, proj, nw, qw, kw, pos, freq))
    qkv = (rms_norm(xd, (width,), nd, 1e-6) @ pd).view(b, s, hq + 2 * hk, d)
    q, k, v = qkv.split([hq, hk, hk], 2)
    qr, kr = qk_norm_rope_fwd(q, k, qd, kd, posd, fd, 1e-6, **how)
    qh, kh, vh = (t.transpose(1, 2).contiguous() for t in (qr, kr, v))
    p, vr = attend(qh, kh, vh, softmax)
    out = p @ vr
    # back through the attention, by its formulas
    do = dout.to(DEV)
    dp = do @ vr.transpose(-1, -2).contiguous()
    ds = p * (dp - (dp * p).sum(-1, keepdim=True)) / d ** 0.5
    dqh = ds @ kh.repeat_interleave(hq // hk, 1)
    dkh = (ds.transpose(-1, -2).contiguous() @ qh).view(b, hk, hq // hk, s, d).sum(2)
    dq, dk, dqw, dkw = qk_norm_rope_bwd(dqh.transpose(1, 2), dkh.transpose(1, 2), q, k, qd, kd,
                                        posd, fd, 1e-6, **how)

    qkv64 = (ref.rms(x.double(), 1e-6) * x.double() * nw.double()) @ proj.double()
    qkv64 = qkv64.view(b, s, hq + 2 * hk, d).requires_grad_()
    w64 = [t.double().requires_grad_() for t in (qw, kw)]
    theta = ref.angles(pos, freq, (b, s), how["sections"], "cycle")
    q64, k64, v64 = qkv64.split([hq, hk, hk], 2)
    q64, k64 = (ref.forward(t, theta, "adjacent", 1.0, w, 1e-6)[0].transpose(1, 2)
                for t, w in zip((q64, k64), w64))
    p64, v64 = attend(q64, k64, v64.transpose(1, 2), lambda t: torch.softmax(t, -1))
    want = p64 @ v64
    grads = torch.autograd.grad((want * dout.double()).sum(), [qkv64, *w64])
    # 32-bit chains of 96 + 32 + 24 products, each within 2^-24 of values up to a few units
    # (relative to each result's largest): 300 steps hold them
    tol = 300 * 2.0 ** -24
    for got, ref64 in ((out, want), (dq, grads[0][:, :, :hq]), (dk, grads[0][:, :, hq:hq + hk]),
                       (dqw, grads[1]), (dkw, grads[2])):
        ref64 = ref64.detach()
        off = (got.cpu().double() - ref64).abs().max() / ref64.abs().max()
        assert float(off) <= tol, float(off)


def test_descriptor_calls_need_no_python_plan():
    """The C entry point with a descriptor of the caller's own."""
    print("[gpu] C entry point", flush=True)
    q, k, _, _, _, pos, freq = _case(tokens=21, hq=3, hk=1, dim=64, dtype=F32)
    d = _lib.RopeDesc()
    d.batch, d.seq, d.q_heads, d.k_heads, d.head_dim, d.n_freq = 1, 21, 3, 1, 64, 32
    d.q_stride[:], d.k_stride[:], d.pos_stride[:] = (0, 192, 64), (0, 64, 64), (0, 0, 1)
    d.sections[0], d.axes, d.pos_dtype, d.scale = 32, 1, _lib.I64, 1.0
    outs = torch.empty_like(q), torch.empty_like(k)
    _lib.call("vbh_rope_fwd", ctypes.addressof(d), q.data_ptr(), k.data_ptr(), pos.data_ptr(),
              freq.data_ptr(), *(o.data_ptr() for o in outs),
              torch.cuda.current_stream().cuda_stream)
    assert _same(outs, rope_fwd(q, k, pos, freq))
