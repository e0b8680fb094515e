"""The norms around a block against their definition in 64 bits, forward and backward.

In fp32 a row's sum of squares has some 40 roundings on the way of any one term (16 in a lane, 6 in a wave, 16 over waves), so 1 / rms is off by a
relative 2^-19 at most, and every stored value by 2^-18 of the magnitudes it is made from, before its own rounding."""
import pytest
import torch

import layers8_reference as ref
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
types = pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
FP32 = 2.0 ** -18
# every shape of the row's group of lanes, whole and ragged
SIZES = [(1, 1), (1, 7), (3, 64), (5, 511), (4, 512), (6, 513), (2, 1000), (3, 1025), (2, 2048), (6, 2049), (3, 4096), (2, 4097), (2, 8000), (2, 8193), (1, 16384)]


def _rand(shape, seed, scale=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    return torch.randn(shape, generator=g) * scale


def _inputs(M, D, G, dtype, seed, gate_dtype=None):
    x, y = _rand((M, D), seed).to(dtype), _rand((M, D), seed + 1, 30.0).to(dtype)
    if M > 2:
        x[1], y[1] = 0, 0
        y[2] = 0
    gate = _rand((G, D), seed + 2).to(gate_dtype or dtype) if G else None
    return x, y, gate, _rand((D,), seed + 3).abs() + 0.5, _rand((D,), seed + 4).abs() + 0.5


def _d(t):
    return None if t is None else t.cuda()


def _within(got, want, magnitudes, what):
    bound_type = got.dtype
    bound = FP32 * magnitudes + ref.UNIT[bound_type] * (1 + 2.0 ** -8) * want.abs() + ref.TINY[bound_type]
    assert got.shape == want.shape, what
    got = got.cpu().double()
    if bound_type == torch.float16:  # beyond the type's range a value is an infinity
        beyond = want.abs() - FP32 * magnitudes > 65520
        assert (got[beyond] == torch.copysign(torch.tensor(float("inf"), dtype=torch.float64), want[beyond])).all(), what
        inside = want.abs() + bound < 65504
        got, want, bound = got[inside], want[inside], bound[inside]
    off = (got - want).abs()
    assert (off <= bound).all(), (what, float((off / bound).max()))


def _magnitudes(x, y, gate, w_post, w_pre, alpha):
    """Those that R and H are made from: |alpha x| + |gate z|, and the same times w_pre / rms(R), once more for 1 / rms."""
    M = x.shape[0]
    none = torch.zeros_like(x, dtype=torch.float64)
    rows = ref.gate_rows(gate, M)
    z, _ = ref.norm(none, y, rows, w_post, None, 0.0, ref.EPS)
    r, h = ref.norm(x, y, rows, w_post, w_pre, alpha, ref.EPS)
    mag_r = (alpha * x.double()).abs() + z.abs()
    s = 1 / torch.sqrt((r * r).mean(dim=1, keepdim=True) + ref.EPS)
    w = 1 if w_pre is None else w_pre.double().abs()
    # an error of R moves the row's rms too: by the mean of |R| times it
    return r, h, mag_r, w * s * (mag_r + r.abs()) + h.abs() * s * s * (r.abs() * mag_r).mean(dim=1, keepdim=True)


@types
@pytest.mark.parametrize("M,D", SIZES)
def test_norm_residual(M, D, dtype):
    for G, post, pre in ((1, True, True), (M, True, False), (0, False, True)):
        x, y, gate, w_post, w_pre = _inputs(M, D, G, dtype, 7 * D + M)
        w_post, w_pre = w_post if post else None, w_pre if pre else None
        r, h, mag_r, mag_h = _magnitudes(x, y, gate, w_post, w_pre, 0.75)
        R, H = tab_amd.NormResidual(x.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 0.75, ref.EPS, M, D)
        assert R.dtype == H.dtype == dtype
        _within(R, r, mag_r, "R")
        _within(H, h, mag_h, "H")
        only, = tab_amd.NormResidual(x.cuda(), y.cuda(), _d(gate), _d(w_post), None, 0.75, ref.EPS, M, D, tab_amd.NORM_NONE)
        assert torch.equal(only, R)
        first, = tab_amd.Norm(x.cuda(), _d(w_pre), ref.EPS, M, D)
        want = ref.norm(x, None, None, None, w_pre, 1.0, ref.EPS)[1]
        _within(first, want, want.abs(), "first norm")


@types
@pytest.mark.parametrize("M,D", SIZES)
def test_packed_output(M, D, dtype):
    """The packed H is the quantizer's of some H within the fp32 bound: its values are within half an 8-bit unit of H and that bound."""
    x, y, gate, w_post, w_pre = _inputs(M, D, 1, dtype, 3 * D + M)
    r, h, mag_r, mag_h = _magnitudes(x, y, gate, w_post, w_pre, 1.5)
    R, QH, SH = tab_amd.NormResidual(x.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 1.5, ref.EPS, M, D, tab_amd.NORM_8BIT)
    _within(R, r, mag_r, "R")
    got = ref.unpack(QH, SH, 1)
    assert (got[:, D:] == 0).all()
    scale = torch.repeat_interleave(ref.two_to(SH.cpu().view(torch.uint8).long() - 127).t(), 128, dim=1)[:, :D]
    unit = torch.maximum(h.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    assert ((got[:, :D] - h).abs() <= unit + 1.1 * FP32 * mag_h).all()
    # and the scales are those of the packed values: none could be halved
    q = QH.cpu().float().abs().view(M, -1, 128).amax(dim=2).t()
    assert ((q >= 224) | (SH.cpu().view(torch.uint8) == 1)).all()
    if dtype == torch.float32:  # the plain output is what was packed
        H, = tab_amd.NormResidual(x.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 1.5, ref.EPS, M, D)[1:]
        Q, S = tab_amd.Quantize8(H, M, D)
        assert torch.equal(Q.view(torch.uint8), QH.view(torch.uint8)) and torch.equal(S.view(torch.uint8), SH.view(torch.uint8))
    Q1, S1 = tab_amd.Norm(x.cuda(), _d(w_pre), ref.EPS, M, D, tab_amd.NORM_8BIT)
    assert Q1.shape == QH.shape and S1.shape == SH.shape


@pytest.mark.parametrize("M,G", [(12, 3), (12, 4), (7, 7), (9, 1), (5000, 5), (5000, 2500), (3000, 3000), (4099, 1)])
def test_gates_of_one_channel_sequence_or_token(M, G):
    D = 70
    for gate_dtype in (torch.float32, torch.bfloat16):
        x, y, gate, w_post, w_pre = _inputs(M, D, G, torch.bfloat16, 40, gate_dtype)
        r, h, mag_r, mag_h = _magnitudes(x, y, gate, w_post, w_pre, 1.0)
        R, H = tab_amd.NormResidual(x.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 1.0, ref.EPS, M, D)
        _within(R, r, mag_r, "R")
        _within(H, h, mag_h, "H")


@types
@pytest.mark.parametrize("D", [100, 1031, 2500])
def test_rows_of_wider_matrices(D, dtype):
    x, y, gate, w_post, w_pre = _inputs(5, D + 40, 1, dtype, 50)
    a, b = x.cuda()[:, 3:3 + D], y.cuda()[:, 11:11 + D]
    rest = (_d(gate[:, :D].contiguous()), _d(w_post[:D]), _d(w_pre[:D]), 1.0, ref.EPS, 5, D)
    for got, want in zip(tab_amd.NormResidual(a, b, *rest), tab_amd.NormResidual(a.contiguous(), b.contiguous(), *rest)):
        assert torch.equal(got, want)


def test_not_a_number_stays_in_its_row():
    x, y, gate, w_post, w_pre = _inputs(4, 600, 1, torch.float32, 60)
    clean = tab_amd.NormResidual(x.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 1.0, ref.EPS, 4, 600)
    y[2, 17], x[0, 599] = float("nan"), float("inf")
    got = tab_amd.NormResidual(x.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 1.0, ref.EPS, 4, 600)
    for a, b in zip(got, clean):
        assert torch.equal(a[[1, 3]], b[[1, 3]])
        assert torch.isnan(a[2]).all()
    assert torch.isinf(got[0][0, 599]) and torch.isnan(got[1][0, 599])


# ---- gradients --------------------------------------------------------------------------------------------------------


def _formula(dr, dh, r, y, gate, w_post, w_pre, alpha):
    """The gradients and the magnitudes they are made from, by the formulas in 64 bits; `gate` as rows of M."""
    r, one = r.double(), 1.0
    g = one if gate is None else gate.double()
    p = 1 / torch.sqrt((r * r).mean(dim=1, keepdim=True) + ref.EPS)
    t, mag = torch.zeros_like(r), torch.zeros_like(r)
    out, mags = {}, {}
    if dr is not None:
        t, mag = t + dr.double(), mag + dr.double().abs()
    if dh is not None:
        a = dh.double() * (one if w_pre is None else w_pre.double())
        t = t + p * a - r * p ** 3 * (r * a).mean(dim=1, keepdim=True)
        mag = mag + p * a.abs() + r.abs() * p ** 3 * (r * a).abs().mean(dim=1, keepdim=True)
        out["dw_pre"], mags["dw_pre"] = (dh.double() * r * p).sum(dim=0), (dh.double() * r * p).abs().sum(dim=0)
    out["dx"], mags["dx"] = alpha * t, abs(alpha) * mag
    if y is not None:
        y = y.double()
        w = one if w_post is None else w_post.double()
        q = 1 / torch.sqrt((y * y).mean(dim=1, keepdim=True) + ref.EPS)
        b, mag_b = t * g * w, mag * abs(g) * w
        out["dy"] = q * b - y * q ** 3 * (y * b).mean(dim=1, keepdim=True)
        mags["dy"] = 2 * (q * mag_b + y.abs() * q ** 3 * (y.abs() * mag_b).mean(dim=1, keepdim=True))
        out["dw_post"], mags["dw_post"] = (t * g * y * q).sum(dim=0), 2 * (mag * abs(g) * (y * q).abs()).sum(dim=0)
        out["dgate"], mags["dgate"] = t * y * q * w, 2 * mag * (y * q * w).abs()
    return out, mags


def _check_gradients(M, D, G, dtype, gate_dtype=None, with_dr=True, with_dh=True, weights=True, seed=70):
    r, y, gate, w_post, w_pre = _inputs(M, D, G, dtype, seed, gate_dtype)
    if not weights:
        w_post = w_pre = None
    dr = _rand((M, D), seed + 5, 0.1).to(dtype) if with_dr else None
    dh = _rand((M, D), seed + 6, 0.1).to(dtype) if with_dh else None
    got = tab_amd.NormResidualBackward(_d(dr), _d(dh), r.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 0.75, ref.EPS, M, D)
    want, mags = _formula(dr, dh, r, y, ref.gate_rows(gate, M), w_post, w_pre, 0.75)
    dx, dy, dgate, dw_post, dw_pre = got
    _within(dx, want["dx"], mags["dx"], "dx")
    _within(dy, want["dy"], mags["dy"], "dy")
    sums = 1 + M * 2.0 ** -24 / FP32  # the sums over rows add up to M roundings more
    if gate is None:
        assert dgate is None
    else:
        assert dgate.dtype == gate.dtype and dgate.shape == gate.shape
        each = M // G
        _within(dgate, want["dgate"].view(G, each, D).sum(dim=1), sums * mags["dgate"].view(G, each, D).sum(dim=1), "dgate")
    if weights:
        _within(dw_post, want["dw_post"], sums * mags["dw_post"], "dw_post")
        if with_dh:
            _within(dw_pre, want["dw_pre"], sums * mags["dw_pre"], "dw_pre")
        else:
            assert (dw_pre == 0).all()
    else:
        assert dw_post is None and dw_pre is None


@types
@pytest.mark.parametrize("M,D", SIZES)
def test_gradients(M, D, dtype):
    _check_gradients(M, D, 1, dtype)


# gates of few rows (whole gates in a group of rows), of one row, and of many (a gate in several groups)
@pytest.mark.parametrize("M,G", [(12, 3), (12, 4), (7, 7), (9, 1), (5000, 5), (5000, 2500), (6000, 6000), (4099, 1), (6006, 6), (6006, 1001)])
@pytest.mark.parametrize("gate_dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_gradients_of_gates(M, G, gate_dtype):
    _check_gradients(M, 70, G, torch.bfloat16, gate_dtype)


@pytest.mark.parametrize("with_dr,with_dh", [(True, False), (False, True)])
@pytest.mark.parametrize("M,D", [(6, 300), (40, 3000)])
def test_gradients_of_one_output(M, D, with_dr, with_dh):
    _check_gradients(M, D, 2, torch.float32, with_dr=with_dr, with_dh=with_dh)
    _check_gradients(M, D, 0, torch.bfloat16, with_dr=with_dr, with_dh=with_dh, weights=False)


@types
@pytest.mark.parametrize("M,D", [(1, 5), (7, 600), (300, 1500), (20, 9000)])
def test_gradients_of_the_first_norm(M, D, dtype):
    x, _, _, _, w = _inputs(M, D, 0, dtype, 80)
    dh = _rand((M, D), 81, 0.1).to(dtype)
    dx, dw = tab_amd.NormBackward(dh.cuda(), x.cuda(), w.cuda(), ref.EPS, M, D)
    want, mags = _formula(None, dh, x, None, None, None, w, 1.0)
    _within(dx, want["dx"], mags["dx"], "dx")
    _within(dw, want["dw_pre"], (1 + M * 2.0 ** -24 / FP32) * mags["dw_pre"], "dw")


def test_gradients_are_differences():
    """Central differences of the 64-bit definition, (f(v + d) - f(v - d)) / 2 |d|: off by d^2 / 6 of the third derivative, here below 1e-6 of
    the gradients' size, so that 1e-4 of it leaves room for fp32."""
    M, D, G, alpha = 6, 40, 3, 0.9
    x, y, gate, w_post, w_pre = _inputs(M, D, G, torch.float32, 90)
    dr, dh = _rand((M, D), 91), _rand((M, D), 92)
    tensors = {"x": x, "y": y, "gate": gate, "w_post": w_post, "w_pre": w_pre}

    def f(**changed):
        t = {k: v.double() for k, v in {**tensors, **changed}.items()}
        r, h = ref.norm(t["x"], t["y"], ref.gate_rows(t["gate"], M), t["w_post"], t["w_pre"], alpha, ref.EPS)
        return float((r * dr.double()).sum() + (h * dh.double()).sum())

    leaves = {k: v.cuda().requires_grad_() for k, v in tensors.items()}
    R, H = tab_nn.norm_residual(leaves["x"], leaves["y"], leaves["gate"], leaves["w_post"], leaves["w_pre"], alpha, ref.EPS)
    got = torch.autograd.grad((R, H), list(leaves.values()), (dr.cuda(), dh.cuda()))
    for (name, v), grad in zip(tensors.items(), got):
        for seed in range(3):
            direction = _rand(tuple(v.shape), 100 + seed).double()
            if name in ("x", "y"):  # rows of zeros have a derivative of 1 / sqrt(eps): steps far below sqrt(eps) would be needed
                direction[1:3] = 0
            step = 1e-4
            want = (f(**{name: v.double() + step * direction}) - f(**{name: v.double() - step * direction})) / (2 * step)
            size = float((grad.cpu().double().abs() * direction.abs()).sum())
            assert abs(float((grad.cpu().double() * direction).sum()) - want) <= 1e-4 * size, name


def test_same_call_same_bits():
    r, y, gate, w_post, w_pre = _inputs(3000, 600, 3, torch.bfloat16, 110)
    dr, dh = _rand((3000, 600), 111).bfloat16(), _rand((3000, 600), 112).bfloat16()
    args = (dr.cuda(), dh.cuda(), r.cuda(), y.cuda(), _d(gate), _d(w_post), _d(w_pre), 1.0, ref.EPS, 3000, 600)
    first = tab_amd.NormResidualBackward(*args)
    for _ in range(5):
        for a, b in zip(first, tab_amd.NormResidualBackward(*args)):
            assert torch.equal(a, b)
