"""The query / key operators on the CPU: the oracle against other ways to the same values,
and every call they refuse, in Python and at the C entry points (nothing is launched).
"""
import ctypes

import pytest
import torch

from dslperfgap_amd import _lib, _rope
from dslperfgap_amd.viperbench.qk_norm_rope.hip_impl import qk_norm_rope_bwd, qk_norm_rope_fwd
from dslperfgap_amd.viperbench.rope.hip_impl import rope_bwd, rope_fwd
from oracle import rope as ref

D, N = 16, 8
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("dim,n", [(8, 4), (10, 3), (9, 4)])
def test_oracle_turns_as_complex_numbers_do(pairing, dim, n):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 5, 3, dim, generator=g, dtype=torch.float64)
    theta = 3 * torch.randn(2, 5, n, generator=g, dtype=torch.float64)
    got = ref.turn(x, theta, pairing, 0.7)
    first, second = ref.pairs(n, pairing)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(
        torch.full_like(theta, 0.7), theta)[:, :, None]
    assert torch.allclose(got[..., first], z.real, atol=1e-14)
    assert torch.allclose(got[..., second], z.imag, atol=1e-14)
    assert torch.equal(got[..., 2 * n:], x[..., 2 * n:])
    back = ref.turn(got / 0.49, theta, pairing, 0.7, back=True)
    assert torch.allclose(back[..., :2 * n], x[..., :2 * n], atol=1e-14)


def test_oracle_axes():
    assert ref.axis_of((2, 3, 1), "blocks") == [0, 0, 1, 1, 1, 2]
    assert ref.axis_of((4, 2, 2), "cycle") == [0, 1, 2, 0, 1, 2, 0, 0]
    assert ref.axis_of((3, 3), "cycle") == [0, 1, 0, 1, 0, 1]
    pos = torch.tensor([[[1, 2]], [[10, 20]]])
    got = ref.angles(pos, torch.tensor([1.0, 0.5]), (1, 2), (1, 1))
    assert got.tolist() == [[[1.0, 5.0], [2.0, 10.0]]]


@pytest.mark.parametrize("weighted", [True, False])
def test_oracle_gradients_are_autograds_and_the_differences(weighted):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, 6, 2, D, generator=g, dtype=torch.float64, requires_grad=True)
    w = (1 + 0.2 * torch.randn(D, generator=g, dtype=torch.float64)).requires_grad_()
    theta = torch.randn(1, 6, 6, generator=g, dtype=torch.float64)
    dy = torch.randn(1, 6, 2, D, generator=g, dtype=torch.float64)
    ww = w if weighted else None

    def f(x, w):
        return (ref.forward(x, theta, "half", 1.3, w, 1e-6)[0] * dy).sum()

    dx, dw, *_ = ref.backward(dy, x.detach(), theta, "half", 1.3,
                              None if ww is None else w.detach(), 1e-6)
    want = torch.autograd.grad(f(x, ww), [x, w] if weighted else [x])
    assert torch.allclose(dx, want[0], atol=1e-12)
    if weighted:
        assert torch.allclose(dw, want[1], atol=1e-12)
    v = torch.randn(x.shape, generator=g, dtype=torch.float64)
    with torch.no_grad():
        slope = (f(x + 1e-6 * v, ww) - f(x - 1e-6 * v, ww)) / 2e-6
    assert abs(float(slope - (dx * v).sum())) < 1e-7


# ---------------------------------------------------------------------------
# refusals in Python: tensors on the CPU reach the device check only when every
# argument is right
# ---------------------------------------------------------------------------
def _args(lead=(2, 5), hq=4, hk=2, dim=D, n=N, dtype=F32, pos=None):
    q, k = torch.randn(*lead, hq, dim).to(dtype), torch.randn(*lead, hk, dim).to(dtype)
    pos = torch.arange(lead[-1]) if pos is None else pos
    return q, k, pos, ref.inv_freq(n)


def _calls(q, k, pos, freq, **how):
    w = torch.ones(q.shape[-1]) if q.dim() else torch.ones(1)
    return [lambda: rope_fwd(q, k, pos, freq, **how), lambda: rope_bwd(q, k, pos, freq, **how),
            lambda: qk_norm_rope_fwd(q, k, w, w, pos, freq, **how),
            lambda: qk_norm_rope_bwd(q, k, q, k, w, w, pos, freq, **how)]


def _refused(error, match, *args, **how):
    for call in _calls(*args, **how):
        with pytest.raises(error, match=match):
            call()


@pytest.mark.parametrize("args,how", [
    (_args(), {}), (_args(lead=(5,)), {}), (_args(dtype=BF16), {"pairing": "adjacent"}),
    (_args(pos=torch.zeros(2, 5, dtype=torch.int32)), {}),
    (_args(pos=torch.zeros(3, 2, 5)), {"sections": (4, 2, 2), "section_order": "cycle"}),
    (_args(pos=torch.zeros(2, 5, dtype=torch.int64)), {"sections": [8]}),
    (_args(pos=torch.zeros(2, 5, dtype=torch.int64)), {"sections": [5, 3]}),
    (_args(lead=(2, 0)), {}), (_args(hk=0), {}), (_args(dim=17), {}),
])
def test_right_arguments_reach_the_device_check(args, how):
    _refused(ValueError, "GPU tensors", *args, **how)


def test_shapes_are_refused():
    q, k, pos, f = _args()
    _refused(ValueError, "same tokens", q, k[:1], pos, f)
    _refused(ValueError, "same tokens", q, k[..., :8].contiguous(), pos, f)
    _refused(ValueError, "same tokens", q, k[0], pos, f)
    _refused(ValueError, "positions must have shape", q, k, pos[:4], f)
    _refused(ValueError, "positions must have shape", q, k, torch.zeros(5, 2, dtype=torch.int64), f)
    _refused(ValueError, "positions of 2 axes", q, k, pos, f, sections=(4, 4))
    _refused(ValueError, "positions must have shape", q, k, torch.zeros(2, 4), f, sections=(4, 4))
    _refused(ValueError, "inv_freq must be a contiguous vector", q, k, pos, f[None])
    _refused(ValueError, "inv_freq must be a contiguous vector", q, k, pos, f.repeat(2)[::2])
    _refused(ValueError, "inv_freq of 9", q, k, pos, ref.inv_freq(9))
    _refused(ValueError, "inv_freq of 0", q, k, pos, f[:0])
    _refused(ValueError, "head_dim must be", *_args(dim=1026))
    _refused(ValueError, r"must be \[tokens, heads", torch.randn(4, D).T, k, pos, f)
    with pytest.raises(ValueError, match="same tokens|must be"):
        rope_fwd(torch.randn(4, D), torch.randn(4, D), pos, f)
    with pytest.raises(ValueError, match="must be"):
        rope_fwd(torch.tensor(1.0), k, pos, f)


def test_types_are_refused():
    q, k, pos, f = _args()
    _refused(TypeError, "dtypes differ", q, k.half(), pos, f)
    _refused(TypeError, "not supported", q.double(), k.double(), pos, f)
    _refused(TypeError, "positions must be", q, k, pos.to(torch.int16), f)
    _refused(TypeError, "positions must be", q, k, pos.double(), f)
    _refused(TypeError, "inv_freq must be", q, k, pos, f.half())


def test_options_are_refused():
    q, k, pos, f = _args()
    pos3 = torch.zeros(3, 5, dtype=torch.int64)
    _refused(ValueError, "section_order must be", q, k, pos, f, section_order="rows")
    _refused(ValueError, "pairing must be", q, k, pos, f, pairing="pairs")
    _refused(ValueError, "add up", q, k, pos3, f, sections=(4, 2, 1))
    _refused(ValueError, "add up", q, k, pos3, f, sections=(10, -1, -1))
    _refused(ValueError, "1..4 axes", q, k, pos3, f, sections=())
    _refused(ValueError, "1..4 axes", q, k, pos3, f, sections=(4, 1, 1, 1, 1))
    _refused(ValueError, "in turn", q, k, pos3, f, sections=(2, 3, 3), section_order="cycle")
    for bad in (float("nan"), float("inf")):
        _refused(ValueError, "scale must be finite", q, k, pos, f, scale=bad)
    w = torch.ones(D)
    for bad in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps must be"):
            qk_norm_rope_fwd(q, k, w, w, pos, f, eps=bad)


def test_weights_and_gradients_are_refused():
    q, k, pos, f = _args(dtype=BF16)
    w = torch.ones(D)
    for bad, error, match in ((torch.ones(8), ValueError, r"shape \[16\]"),
                              (torch.ones(4, D), ValueError, r"shape \[16\]"),
                              (torch.ones(D, dtype=torch.int32), TypeError, "floating")):
        for qw, kw in ((bad, w), (w, bad)):
            with pytest.raises(error, match=match):
                qk_norm_rope_fwd(q, k, qw, kw, pos, f)
            with pytest.raises(error, match=match):
                qk_norm_rope_bwd(q, k, q, k, qw, kw, pos, f)
    with pytest.raises(TypeError, match="dq_out must be"):
        qk_norm_rope_bwd(q.float(), k.float(), q, k, w, w, pos, f)
    with pytest.raises(TypeError, match="dtypes differ"):
        qk_norm_rope_bwd(q.float(), k, q, k, w, w, pos, f)
    with pytest.raises(ValueError, match="dq_out must have shape"):
        qk_norm_rope_bwd(q[:, :4], k[:, :4], q, k, w, w, pos, f)
    with pytest.raises(ValueError, match="same tokens"):
        qk_norm_rope_bwd(q[:1], k, q, k, w, w, pos, f)
    for qw, kw in ((None, None), (w, None), (None, w.bfloat16()), (w, w.bfloat16()),
                   (w.double(), w.half())):
        with pytest.raises(ValueError, match="GPU tensors"):
            qk_norm_rope_bwd(q, k, q, k, qw, kw, pos, f)


def test_plans_hold_the_strides_and_are_kept():
    whole = torch.randn(2, 5, 8, D)
    q, k = whole[:, :, :4], whole[:, :, 4:6]
    pos = torch.zeros(5, dtype=torch.int32)
    freq = ref.inv_freq(N, dtype=torch.float64)
    def plan():
        with pytest.raises(ValueError, match="GPU tensors"):
            rope_fwd(q, k, pos, freq)
        return list(_rope._PLANS.values())[-1]

    _rope._PLANS.cache_clear()
    p = plan()
    _, address, q_shape, q_strides, k_shape, k_strides, ws_bytes, d = p
    assert plan() is p and len(_rope._PLANS) == 1 and address == ctypes.addressof(d)
    assert [d.batch, d.seq, d.q_heads, d.k_heads, d.head_dim, d.n_freq] == [2, 5, 4, 2, D, N]
    assert list(d.q_stride) == [5 * 8 * D, 8 * D, D] == list(d.k_stride)
    assert list(d.pos_stride) == [0, 0, 1] and d.pos_dtype == _lib.I32 and d.f64_freq == 1
    assert q_shape == (2, 5, 4, D) and q_strides == (5 * 4 * D, 4 * D, D, 1)
    assert k_shape == (2, 5, 2, D) and ws_bytes == 0
    q = k = torch.randn(2, 4, 5, D).transpose(1, 2)
    assert list(plan()[-1].q_stride) == [20 * D, D, 5 * D]
    q = k = torch.randn(2, 5, 4, D, 2)[..., 0]  # copied: the plan is that of the copy
    assert list(plan()[-1].q_stride) == [20 * D, 4 * D, D]


# ---------------------------------------------------------------------------
# the C entry points
# ---------------------------------------------------------------------------
def _desc(**over):
    d = _lib.RopeDesc()
    d.batch, d.seq, d.q_heads, d.k_heads, d.head_dim, d.n_freq = 2, 5, 4, 2, D, N
    d.q_stride[:] = (5 * 4 * D, 4 * D, D)
    d.k_stride[:] = (5 * 2 * D, 2 * D, D)
    d.dq_stride[:], d.dk_stride[:] = d.q_stride, d.k_stride
    d.pos_stride[:] = (0, 5, 1)
    d.sections[0] = N
    d.axes, d.pos_dtype, d.scale, d.eps = 1, _lib.I64, 1.0, 1e-6
    for name, v in over.items():
        if isinstance(v, (tuple, list)):
            getattr(d, name)[:len(v)] = v
        else:
            setattr(d, name, v)
    return d


_KEPT = []  # descriptors whose addresses are in use


def _entries(d, p=16, ws=16, ws_bytes=1 << 30):
    _KEPT.append(d)
    a = ctypes.addressof(d) if d is not None else None
    return [("vbh_rope_fwd", (a, p, p, p, p, p, p, None)),
            ("vbh_rope_bwd", (a, p, p, p, p, p, p, None)),
            ("vbh_qk_norm_rope_fwd", (a, p, p, p, p, p, p, p, p, None)),
            ("vbh_qk_norm_rope_bwd", (a, *[p] * 12, ws, ws_bytes, None))]


@pytest.mark.parametrize("over,code", [
    ({"dtype": 3}, _lib.E_DTYPE), ({"pos_dtype": _lib.F16}, _lib.E_DTYPE),
    ({"batch": -1}, _lib.E_INVALID), ({"seq": -5}, _lib.E_INVALID),
    ({"q_heads": -1}, _lib.E_INVALID), ({"k_heads": 1 << 20}, _lib.E_RANGE),
    ({"head_dim": 0}, _lib.E_RANGE), ({"head_dim": 1025}, _lib.E_RANGE),
    ({"n_freq": 0}, _lib.E_INVALID), ({"n_freq": 9}, _lib.E_INVALID),
    ({"n_freq": -(1 << 62)}, _lib.E_INVALID),
    ({"batch": 1 << 40, "seq": 1 << 40}, _lib.E_RANGE), ({"seq": 1 << 31}, _lib.E_RANGE),
    ({"axes": 0}, _lib.E_INVALID), ({"axes": 5}, _lib.E_INVALID),
    ({"section_order": 2}, _lib.E_INVALID), ({"pairing": -1}, _lib.E_INVALID),
    ({"sections": [7]}, _lib.E_INVALID), ({"sections": [1 << 62]}, _lib.E_INVALID),
    ({"axes": 2, "sections": [9, -1]}, _lib.E_INVALID),
    ({"axes": 2, "sections": [3, 5], "section_order": 1}, _lib.E_INVALID),
    ({"q_stride": (-1, 0, 0)}, _lib.E_RANGE), ({"k_stride": (0, 1 << 61, 0)}, _lib.E_RANGE),
    ({"pos_stride": (0, 1 << 60, 1 << 60)}, _lib.E_RANGE),
    ({"scale": float("inf")}, _lib.E_INVALID),
    # more values than any memory holds
    ({"batch": 1, "seq": (1 << 31) - 1, "q_heads": 1 << 16, "q_stride": (0, 0, 0),
      "k_stride": (0, 0, 0), "pos_stride": (0, 0, 0), "dq_stride": (0, 0, 0),
      "dk_stride": (0, 0, 0)}, _lib.E_RANGE),
])
def test_entry_points_refuse(over, code):
    for name, args in _entries(_desc(**over)):
        with pytest.raises(_lib.VbhError) as e:
            _lib.call(name, *args)
        assert e.value.code == code, (name, e.value)
    assert _lib.lib().vbh_qk_norm_rope_workspace_bytes(_desc(**over)) == 0


def test_entry_points_refuse_null_pointers_and_small_workspaces():
    for name, args in _entries(None):
        with pytest.raises(_lib.VbhError, match="null descriptor"):
            _lib.call(name, *args)
    for name, args in _entries(_desc()):
        optional = {"vbh_qk_norm_rope_fwd": (3, 4),
                    "vbh_qk_norm_rope_bwd": (5, 6, 11, 12)}.get(name, ())
        for i in range(1, len(args) - 1):
            if args[i] != 16 or i in optional:
                continue
            with pytest.raises(_lib.VbhError, match="null pointer|workspace"):
                _lib.call(name, *args[:i], None, *args[i + 1:])
    for name, args in _entries(_desc()):
        outs = (5, 6) if name.startswith("vbh_rope") else (7, 8) if "fwd" in name else (9, 10)
        for i in outs:
            with pytest.raises(_lib.VbhError, match="16-byte aligned"):
                _lib.call(name, *args[:i], 24, *args[i + 1:])
    d = _desc()
    need = _lib.lib().vbh_qk_norm_rope_workspace_bytes(d)
    assert need > 0 and need % (4 * D) == 0
    for ws, n in ((16, need - 1), (24, need), (16, -1)):
        name, args = _entries(d, ws=ws, ws_bytes=n)[3]
        with pytest.raises(_lib.VbhError, match="workspace"):
            _lib.call(name, *args)
    for over in ({"w_dtype": _lib.F16}, {"eps": -1.0}, {"eps": float("nan")}):
        for name, args in _entries(_desc(**over))[2:]:
            with pytest.raises(_lib.VbhError):
                _lib.call(name, *args)


def test_empty_launches_are_noops():
    for over in ({"seq": 0}, {"batch": 0}, {"q_heads": 0, "k_heads": 0}):
        d = _desc(**over)
        assert _lib.lib().vbh_qk_norm_rope_workspace_bytes(d) == 0
        for name, args in _entries(d, p=None, ws=None, ws_bytes=0):
            _lib.call(name, *args)


def test_workspaces_stay_small():
    """One row of sums for each of at most 1024 workgroups or so, whatever the tokens."""
    for tokens in (1, 7, 333, 8192, 1 << 20):
        for hq, hk, dim in ((32, 8, 128), (1, 1, 64), (64, 64, 256), (3, 5, 33), (1024, 1, 64)):
            d = _desc(batch=1, seq=tokens, q_heads=hq, k_heads=hk, head_dim=dim, n_freq=8,
                      q_stride=(0, hq * dim, dim), k_stride=(0, hk * dim, dim),
                      dq_stride=(0, hq * dim, dim), dk_stride=(0, hk * dim, dim))
            n = _lib.lib().vbh_qk_norm_rope_workspace_bytes(d)
            assert 0 < n <= 4 * dim * 2 * 1400, (tokens, hq, hk, dim, n)
