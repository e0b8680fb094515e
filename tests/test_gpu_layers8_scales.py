"""8-bit products of operands that were packed elsewhere: scale bytes that the quantizer does not give, and long sums, in which one product more or
less has to show."""
import pytest
import torch

import layers8_reference as ref
import tab_amd
from test_gpu_layers8 import _rand

pytestmark = pytest.mark.gpu

# few rows, tiles of 64 x 64 whole and in parts, 64 x 128, 128 x 128, 256 x 256 (16-bit outputs)
SIZES = [(1, 40, 300), (20, 40, 300), (70, 72, 300), (100, 72, 8192), (70, 8299, 130), (2970, 643, 130), (1425, 8304, 130)]
outputs = pytest.mark.parametrize("out", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


def _packed(R, K, seed, byte, block_rows=1):
    """Numbers of 4 to 448 under one scale byte."""
    x = _rand((R, K), seed)
    x = torch.sign(x) * (x.abs() * 40).clamp(4, 448)
    q = torch.zeros(R, ref.blocks(K) * 128)
    q[:, :K] = ref.nearest8(x.double(), 0).float()
    s = torch.full((ref.blocks(K), -(-R // block_rows)), byte, dtype=torch.uint8)
    return q.to(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu)


def _product(QX, SX, QW, SW, M, N, K, out):
    return tab_amd.Linear8Packed(QX.cuda(), SX.cuda(), QW.cuda(), SW.cuda(), M, N, K, out)


@outputs
@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("x_byte,w_byte", [(0, 254), (254, 0), (0, 127), (127, 0), (1, 253), (240, 10)])
def test_extreme_scales(x_byte, w_byte, M, N, K, out):
    """2^(byte - 127) for every byte below 255.  Numbers from 4 on: none below 2^-126 after its scale; those under 253 and 254 below 1, none above
    fp32's largest."""
    QX, SX = _packed(M, K, 1, x_byte)
    QW, SW = _packed(N, K, 2, w_byte, 128)
    if x_byte >= 253:
        QX = (QX.float() / 512).to(torch.float8_e4m3fn)
    if w_byte >= 253:
        QW = (QW.float() / 512).to(torch.float8_e4m3fn)
    y = _product(QX, SX, QW, SW, M, N, K, out)
    a, b = (ref.unpack(*t) for t in ((QX, SX, 1), (QW, SW, 128)))
    want, magnitudes = (a.cuda() @ b.cuda().t().contiguous()), (a.abs().cuda() @ b.abs().cuda().t().contiguous())
    bound = (a.shape[1] * 2.0 ** -24 + (0 if out == torch.float32 else 2.0 ** -10)) * magnitudes + ref.UNIT[out] * (1 + 2.0 ** -10) * want.abs() + ref.TINY[out]
    off = (y.double() - want).abs()
    assert off.shape == bound.shape and bool((off <= bound).all()), float((off / bound).max())


@outputs
@pytest.mark.parametrize("M,N,K", SIZES)
def test_scale_that_is_no_number(M, N, K, out):
    """Byte 255 is NaN: so are the rows and columns whose sums have a product under it, and no others."""
    QX, SX = _packed(M, K, 3, 127)
    QW, SW = _packed(N, K, 4, 127)
    last = ref.blocks(K) - 1
    SX.view(torch.uint8)[last, M // 2] = 255
    SW.view(torch.uint8)[0, N // 3] = 255
    y = _product(QX, SX, QW, SW, M, N, K, out)
    want = torch.zeros((M, N), dtype=torch.bool, device="cuda")
    want[M // 2], want[:, N // 3] = True, True
    assert torch.equal(torch.isnan(y), want)


def _groups_lose(products):
    """At most what the products of groups of eight neighbours lose when 13 bits below the largest are kept: a unit of the last bit each, nothing where a
    product is a whole number of units."""
    p = products.view(*products.shape[:-1], -1, 8)
    _, e = torch.frexp(p.abs().amax(dim=-1, keepdim=True))
    unit = ((e.long() - 1 - 13 + 1023) << 52).view(torch.float64)  # 2^(e - 1 - 13)
    return torch.where(torch.remainder(p, unit) == 0, torch.zeros_like(p), unit.expand_as(p)).sum(dim=(-1, -2))


# few rows, 64 x 64 in parts, 256 x 256 (64 x 128 in fp32) in parts and whole
@pytest.mark.parametrize("M,N,K", [(4, 300, 10855), (64, 300, 10855), (2214, 2718, 10855), (1283, 9011, 2007)])
def test_mean_error_of_long_sums(M, N, K):
    """A sum of many products may be off by more than one of them.  The mean of all errors may not: it is at most what the groups lose, K roundings of fp32 (of
    partial sums: each is the difference of two from the start) and half of the output's largest rounding, since that is anywhere within half a unit.  Taken over
    a part of the output, where every product is known; a product lost or counted twice in each sum is more."""
    x, w = _rand((M, K), 5).to(torch.bfloat16), _rand((N, K), 6, K ** -0.5)
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K)
    QW, SW = tab_amd.Quantize8(w.cuda(), N, K, 128)
    rows, columns = torch.arange(0, M, max(1, M // 12)), torch.arange(0, N, N // 12)
    a, b = ref.unpack(QX, SX, 1)[rows].cuda(), ref.unpack(QW, SW, 128)[columns].cuda()
    products = a[:, None, :] * b[None, :, :]
    want, mean_product = products.sum(dim=-1), float(products.abs().sum(dim=-1).mean()) / K
    partial, lose = products.cumsum(dim=-1).abs().amax(dim=-1), _groups_lose(products)
    for out in (torch.float32, torch.float16):
        y = tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K, out)[rows.cuda()][:, columns.cuda()].double()
        bound = K * 2.0 ** -24 * 2 * partial + (0 if out == torch.float32 else lose) + ref.UNIT[out] / 2 * want.abs() + ref.TINY[out]
        mean, allowed = float((y - want).abs().mean()), float(bound.mean())
        assert allowed < mean_product and mean <= allowed, (out, mean, allowed, mean_product)
