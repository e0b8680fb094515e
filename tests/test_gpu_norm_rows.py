"""Norms of more rows than the chip holds at once, so that a group of lanes works through several: loads ahead, gates that change inside a group, sums
over its rows, against the definition in 64 bits."""
import pytest
import torch

import layers8_reference as ref
import tab_amd
from test_gpu_norm_residual import FP32, _d, _formula, _inputs, _magnitudes

pytestmark = pytest.mark.gpu

# (M, D): three rows and more a group for each shape of a row's lanes; M a multiple of 21
ROWS = [(25011, 70), (13020, 521), (6237, 1500), (3129, 4096), (1575, 4100), (1071, 8200), (1071, 16384)]
per_gate = pytest.mark.parametrize("rows_per_gate", [0, 1, 3, 7, 1000000], ids=["none", "token", "three", "seven", "one"])
rows = pytest.mark.parametrize("M,D", ROWS)
two_types = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


def _gates(M, rows_per_gate):
    return 0 if rows_per_gate == 0 else M // min(M, rows_per_gate)


def _cuda(*tensors):
    return [_d(t) for t in tensors]


def _within(got, want, magnitudes, what):
    """The bound of the smaller norms' tests, on the GPU."""
    bound = FP32 * magnitudes + ref.UNIT[got.dtype] * (1 + 2.0 ** -8) * want.abs() + ref.TINY[got.dtype]
    off = (got.double() - want).abs()
    assert off.shape == bound.shape and bool((off <= bound).all()), (what, float((off / bound).max()))


def _packed_within(QH, SH, h, mag_h, M, D):
    """Half an 8-bit unit and the fp32 bound, and no scale that could be halved."""
    scale = torch.repeat_interleave(((SH.view(torch.uint8).long() + 1023 - 127) << 52).view(torch.float64).t(), 128, dim=1)
    got = QH.float().double() * scale
    assert bool((got[:, D:] == 0).all())
    unit = torch.maximum(h.abs() * 2.0 ** -4, scale[:, :D] * 2.0 ** -10)
    assert bool(((got[:, :D] - h).abs() <= unit + 1.1 * FP32 * mag_h).all())
    q = QH.float().abs().view(M, -1, 128).amax(dim=2).t()
    assert bool(((q >= 224) | (SH.view(torch.uint8) == 1)).all())


@two_types
@per_gate
@rows
def test_forward(M, D, rows_per_gate, dtype):
    x, y, gate, w_post, w_pre = _cuda(*_inputs(M, D, _gates(M, rows_per_gate), dtype, 7 * D + M))
    r, h, mag_r, mag_h = _magnitudes(x, y, gate, w_post, w_pre, 0.75)
    R, H = tab_amd.NormResidual(x, y, gate, w_post, w_pre, 0.75, ref.EPS, M, D)
    _within(R, r, mag_r, "R")
    _within(H, h, mag_h, "H")
    only, = tab_amd.NormResidual(x, y, gate, w_post, None, 0.75, ref.EPS, M, D, tab_amd.NORM_NONE)
    assert torch.equal(only, R)
    R8, QH, SH = tab_amd.NormResidual(x, y, gate, w_post, w_pre, 0.75, ref.EPS, M, D, tab_amd.NORM_8BIT)
    assert torch.equal(R8, R)
    _packed_within(QH, SH, h, mag_h, M, D)


@two_types
@pytest.mark.parametrize("M,D", [(1, 1), (3, 100), (5, 511), (2, 1000), (3, 1025), (3, 4096), (2, 8000), (2, 16384)] + ROWS)
def test_first_norm(M, D, dtype):
    x, _, _, _, w = _cuda(*_inputs(M, D, 0, dtype, 5 * D + M))
    want = ref.norm(x, None, None, None, w, 1.0, ref.EPS)[1]
    H, = tab_amd.Norm(x, w, ref.EPS, M, D)
    _within(H, want, want.abs(), "H")
    QH, SH = tab_amd.Norm(x, w, ref.EPS, M, D, tab_amd.NORM_8BIT)
    _packed_within(QH, SH, want, want.abs(), M, D)
    if dtype == torch.float32:  # the plain output is what was packed
        Q, S = tab_amd.Quantize8(H, M, D)
        assert torch.equal(Q.view(torch.uint8), QH.view(torch.uint8)) and torch.equal(S.view(torch.uint8), SH.view(torch.uint8))


def test_stack_whose_first_block_takes_the_packed_norm():
    from tab_amd import nn as tab_nn
    D, M = 200, 40
    x, _, _, _, _ = _cuda(*_inputs(M, D, 0, torch.float32, 60))
    w, head = (torch.randn((n, D), generator=torch.Generator("cpu").manual_seed(s)) * D ** -0.5 for n, s in ((D, 61), (30, 62)))
    stack = tab_nn.ResidualStack([tab_nn.Linear8.from_float(w)], D, head=tab_nn.Linear8.from_float(head)).cuda()
    with torch.no_grad():
        got = stack(x)
        h, = tab_amd.Norm(x, stack.w_pre[0], ref.EPS, M, D)
        y = tab_amd.Linear8Packed(*tab_amd.Quantize8(h, M, D), stack.blocks[0].QW, stack.blocks[0].SW, M, D, D)
        _, h = tab_amd.NormResidual(x, y, stack.gate[0], stack.w_post[0], stack.w_pre[1], 1.0, ref.EPS, M, D)
        want = tab_amd.Linear8Packed(*tab_amd.Quantize8(h, M, D), stack.head.QW, stack.head.SW, M, 30, D)
    assert torch.equal(got, want)


@two_types
@per_gate
@rows
def test_gradients(M, D, rows_per_gate, dtype):
    G = _gates(M, rows_per_gate)
    r, y, gate, w_post, w_pre = _cuda(*_inputs(M, D, G, dtype, 9 * D + M))
    g = torch.Generator("cuda").manual_seed(D)
    dr, dh = ((torch.randn((M, D), generator=g, device="cuda") * 0.1).to(dtype) for _ in range(2))
    dx, dy, dgate, dw_post, dw_pre = tab_amd.NormResidualBackward(dr, dh, r, y, gate, w_post, w_pre, 0.75, ref.EPS, M, D)
    want, mags = _formula(dr, dh, r, y, ref.gate_rows(gate, M), w_post, w_pre, 0.75)
    _within(dx, want["dx"], mags["dx"], "dx")
    _within(dy, want["dy"], mags["dy"], "dy")
    sums = 1 + M * 2.0 ** -24 / FP32  # the sums over rows add up to M roundings more
    _within(dw_post, want["dw_post"], sums * mags["dw_post"], "dw_post")
    _within(dw_pre, want["dw_pre"], sums * mags["dw_pre"], "dw_pre")
    if G:
        _within(dgate, want["dgate"].view(G, M // G, D).sum(dim=1), sums * mags["dgate"].view(G, M // G, D).sum(dim=1), "dgate")
