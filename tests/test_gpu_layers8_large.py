"""8-bit products by every tile and with every cut of K, against their definitions in 64 bits, and operands whose offsets pass 2^31."""
import pytest
import torch

import layers8_reference as ref
import tab_amd
from test_gpu_layers8 import _rand
from test_layers8_host import WAYS

pytestmark = pytest.mark.gpu


def _check(y, a, b):
    """As the smaller products' check, with the sums in 64 bits on the GPU."""
    a, b = a.cuda(), b.cuda()
    want, magnitudes = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    bound = (a.shape[1] * 2.0 ** -24 + (0 if y.dtype == torch.float32 else 2.0 ** -10)) * magnitudes + ref.UNIT[y.dtype] * (1 + 2.0 ** -10) * want.abs() + ref.TINY[y.dtype]
    off = (y.double() - want).abs()
    assert off.shape == bound.shape and bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("format", [0, 1])
@pytest.mark.parametrize("out,M,N,K,way", WAYS)
def test_every_tile_and_cut(out, M, N, K, way, format):
    dtype = [torch.float32, torch.bfloat16][out]
    x, w = _rand((M, K), M + K).to(torch.bfloat16), _rand((N, K), N, K ** -0.5)
    block_rows = 128 if (M + format) % 2 else 1
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K, 1, format)
    QW, SW = tab_amd.Quantize8(w.cuda(), N, K, block_rows)
    a, b = ref.unpack(QX, SX, 1), ref.unpack(QW, SW, block_rows)
    y = tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K, dtype)
    _check(y, a, b)
    if out == 1:
        _check(tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K, torch.float16), a, b)
    assert torch.equal(y, tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K, dtype))


def test_packed_rows_past_two_gigabytes():
    """Rows repeat after 64: so do the numbers of both layouts, and the product's rows."""
    M, N, K = 32832, 40, 65700  # 2.16e9 numbers
    some = _rand((64, K), 1).to(torch.bfloat16)
    x = some.cuda().repeat(M // 64, 1)
    QX, SX, QT, ST = tab_amd.Quantize8Both(x, M, K)
    q, s = tab_amd.Quantize8(some.cuda(), 64, K)
    assert torch.equal(QX.view(torch.uint8).view(M // 64, 64, -1), q.view(torch.uint8).expand(M // 64, -1, -1))
    assert torch.equal(SX.view(torch.uint8).view(-1, M // 64, 64), s.view(torch.uint8)[:, None, :].expand(-1, M // 64, -1))
    qt, st = tab_amd.Quantize8Transposed(some.cuda().repeat(2, 1), 128, K)
    full = M // 128 * 128
    assert torch.equal(QT.view(torch.uint8)[:, :full].view(K, -1, 128), qt.view(torch.uint8)[:, None, :].expand(-1, full // 128, -1))
    assert torch.equal(ST.view(torch.uint8)[:full // 128], st.view(torch.uint8).expand(full // 128, -1))
    del QT, ST, x
    w = _rand((N, K), 2, K ** -0.5)
    QW, SW = tab_amd.Quantize8(w.cuda(), N, K, 128)
    y = tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K, torch.bfloat16)
    _check(y[-64:], ref.unpack(q, s, 1), ref.unpack(QW, SW, 128))
    assert torch.equal(y.view(M // 64, 64, N), y[-64:].expand(M // 64, -1, -1))
    # the weights past two gigabytes
    y = tab_amd.Linear8Packed(*tab_amd.Quantize8(w.cuda(), N, K), QX, SX, N, M, K, torch.bfloat16)
    assert torch.equal(y.view(N, M // 64, 64), y[:, None, -64:].expand(-1, M // 64, -1))


def test_output_past_two_gigabytes():
    M, N, K = 40000, 54400, 100  # 2.18e9 numbers
    some, w = _rand((64, K), 3).to(torch.bfloat16), _rand((64, K), 4)
    QX, SX = tab_amd.Quantize8(some.cuda().repeat(M // 64, 1), M, K)
    QW, SW = tab_amd.Quantize8(w.cuda().repeat(N // 64, 1), N, K)
    y = tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K, torch.bfloat16)
    _check(y[-64:, -64:], ref.unpack(*tab_amd.Quantize8(some.cuda(), 64, K), 1), ref.unpack(*tab_amd.Quantize8(w.cuda(), 64, K), 1))
    last = y[-64:, -64:].repeat(1, N // 64)
    assert all(torch.equal(y[m:m + 64], last) for m in range(0, M, 64))


@pytest.mark.parametrize("gates", [0, 5])
def test_norm_past_two_gigabytes(gates):
    """2.16e9 numbers; rows repeat after 64 (and under the gates, of which each repeats too)."""
    M, D = 132480, 16300
    x, y = (_rand((64, D), s).to(torch.bfloat16).cuda() for s in (5, 6))
    g = torch.full((1, D), 0.5, dtype=torch.bfloat16, device="cuda")
    wp, wq = (torch.rand(D, device="cuda") + 0.5 for _ in range(2))
    big = lambda t: t.repeat(M // 64, 1)  # noqa: E731
    gate = g.repeat(gates, 1) if gates else None
    R, H = tab_amd.NormResidual(big(x), big(y), gate, wp, wq, 0.5, ref.EPS, M, D)
    r, h = tab_amd.NormResidual(x, y, g if gates else None, wp, wq, 0.5, ref.EPS, 64, D)
    assert torch.equal(R.view(-1, 64, D), r.expand(M // 64, -1, -1)) and torch.equal(H.view(-1, 64, D), h.expand(M // 64, -1, -1))
    big_grad = tab_amd.NormResidualBackward(H, big(x), R, big(y), gate, wp, wq, 0.5, ref.EPS, M, D)
    grad = tab_amd.NormResidualBackward(h, x, r, y, g if gates else None, wp, wq, 0.5, ref.EPS, 64, D)
    for a, b in zip(big_grad[:2], grad[:2]):
        assert torch.equal(a.view(-1, 64, D), b.expand(M // 64, -1, -1))
