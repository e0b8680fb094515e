"""4-bit weights against their definition in 64 bits: packed numbers and scales equal, products within what fp32 sums and one rounding allow."""
import copy

import pytest
import torch

import experts_reference as ref
import layers8_reference as ref8
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
types = pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])


def _rand(shape, seed, scale=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    return torch.randn(shape, generator=g) * torch.exp(torch.randn((shape[0], 1), generator=g)) * scale


def _same_packed(Q, S, x):
    q, e = ref.quantize4(x)
    exponents = S.cpu().view(torch.uint8).long() - 127
    assert Q.dtype == torch.float4_e2m1fn_x2 and S.dtype == torch.float8_e8m0fnu
    assert exponents.shape == e.shape and torch.equal(exponents, e)
    assert torch.equal(ref.numbers4(Q), q)


@types
@pytest.mark.parametrize("M,K", [(1, 1), (1, 32), (3, 33), (5, 127), (31, 128), (33, 129), (131, 300), (32, 1000), (257, 64), (500, 7)])
def test_quantize4(M, K, dtype):
    x = _rand((M, K), M * 1000 + K).to(dtype)
    _same_packed(*tab_amd.Quantize4(x.cuda(), M, K), x)


@types
def test_quantize4_rows_of_a_wider_matrix(dtype):
    x = _rand((37, 300), 5).to(dtype)
    xd = x.cuda()[:, 13:13 + 261]
    assert not xd.is_contiguous()
    _same_packed(*tab_amd.Quantize4(xd, 37, 261), x[:, 13:13 + 261])


@types
def test_quantize4_special_values(dtype):
    """Groups of zeros, magnitudes at and beside the bound of a scale, subnormals, the type's extremes, ties between two numbers, infinities and NaN."""
    big = torch.finfo(dtype).max
    smallest = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    one = 1 + torch.finfo(dtype).eps
    groups = [[0.0], [-0.0, 0.0], [6.0, 1.0, -3.0], [6.0 * one, 1.0], [1.5, 1.5 * one, -1.5], [smallest, -smallest, 3 * smallest], [big, -big, 1.0],
              [6.0, 0.25, -0.25, 0.75, 1.25, 1.75, 2.5, -3.5, 5.0, -5.0, 0.25 * one, 0.75 / one, 2.5 * one, 3.5 / one, 5.0 * one], [float("inf"), 2.0, -1.0],
              [float("-inf"), float("nan"), 0.5], [float("nan")], [1e-3, 60000.0, -2e-5]]
    x = torch.zeros((len(groups), 130))
    for i, g in enumerate(groups):
        x[i, 32:32 + len(g)] = torch.tensor(g)
        x[i, 128] = g[0]
    x = x.to(dtype)
    _same_packed(*tab_amd.Quantize4(x.cuda(), x.shape[0], x.shape[1]), x)


def test_quantize4_takes_no_scale_below_the_smallest():
    x = torch.full((2, 128), 2.0 ** -140)
    Q, S = tab_amd.Quantize4(x.cuda(), 2, 128)
    assert (S.view(torch.uint8) == 1).all()
    _same_packed(Q, S, x)


# every way the product is computed: rows (whole, cut up among workgroups), tiles of 64 with K in parts and whole, of 128, of 256
SIZES = [(1, 1, 1), (1, 16, 128), (1, 1000, 2050), (2, 17, 129), (15, 40, 1024), (15, 33, 4096), (16, 33, 4096), (17, 20, 4096), (16, 100, 640), (16, 8300, 130), (17, 33, 300),
         (31, 64, 128), (32, 130, 2000), (33, 5, 77), (40, 1003, 640), (64, 64, 128), (65, 65, 1153), (100, 72, 8192), (3, 50, 30000), (129, 300, 257), (300, 129, 4000), (500, 777, 520),
         (33, 4096, 300), (96, 1003, 2050), (68, 1000, 4096), (69, 1000, 4096), (256, 64, 1024), (512, 16, 640), (513, 16, 640), (130, 2048, 1100), (70, 4100, 520)]


@types
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear4(M, N, K, dtype):
    x = _rand((M, K), M + N + K).to(dtype)
    w = _rand((N, K), M + 2 * N, K ** -0.5)
    if M > 3:
        x[2] = 0
    QW, SW = tab_amd.Quantize4(w.cuda(), N, K)
    want, mag = ref.product(ref8.value(*ref8.quantize(x, 1, 0), 1), ref.unpack4(QW, SW))
    ref.check(tab_amd.Linear4(x.cuda(), QW, SW, M, N, K), want, mag, K, dtype != torch.float32, "Linear4")
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K)
    for out in TYPES:
        y = tab_amd.Linear4Packed(QX, SX, QW, SW, M, N, K, out)
        assert y.dtype == out
        ref.check(y, want, mag, K, out != torch.float32, f"Linear4Packed to {out}")


@pytest.mark.parametrize("M,N,K", [(1024, 4096, 256), (2100, 4000, 130), (4096, 4100, 384), (4099, 4097, 128)])
def test_large_tiles(M, N, K):
    x, w = _rand((M, K), 3).to(torch.bfloat16), _rand((N, K), 4, 0.1)
    QW, SW = tab_amd.Quantize4(w.cuda(), N, K)
    a, b = (t.cuda() for t in (ref8.value(*ref8.quantize(x, 1, 0), 1), ref.unpack4(QW, SW)))
    want, mag = ref.product(a, b.contiguous())
    for out in (torch.bfloat16, torch.float32):
        y = tab_amd.Linear4Packed(*tab_amd.Quantize8(x.cuda(), M, K), QW, SW, M, N, K, out)
        ref.check(y, want.cpu(), mag.cpu(), K, out != torch.float32, "tiles")


@types
@pytest.mark.parametrize("M", [1, 20, 70, 300])
def test_not_a_number_stays_in_its_row_and_column(M, dtype):
    N, K = 80, 400
    x, w = _rand((M, K), 5).to(dtype), _rand((N, K), 6)
    x[0, 200], w[7, 130], w[40, 390] = float("inf"), float("nan"), float("-inf")
    QW, SW = tab_amd.Quantize4(w.cuda(), N, K)
    y = tab_amd.Linear4(x.cuda(), QW, SW, M, N, K).cpu()
    want = torch.zeros((M, N), dtype=torch.bool)
    want[0], want[:, 7], want[:, 40] = True, True, True
    assert torch.equal(torch.isnan(y), want)
    x[0, 200], w[7, 130], w[40, 390] = 0.0, 0.0, 0.0
    clean = ~want
    exact, mag = ref.product(ref8.value(*ref8.quantize(x, 1, 0), 1), ref.value4(*ref.quantize4(w)))
    ref.check(y[clean], exact[clean], mag[clean], K, dtype != torch.float32, "beside NaN")


def test_every_scale_byte_of_a_weight():
    """Scales of all sizes, as a weight from elsewhere may have them; products of whole numbers that fp32 holds."""
    K = 128
    for dtype in (torch.float32, torch.bfloat16):
        S = torch.arange(1, 255, dtype=torch.uint8)[None, :, None].expand(1, -1, 4).contiguous()  # 2^-126 .. 2^127
        Q = torch.full((254, 64), 0x22, dtype=torch.uint8)                                        # ones
        x = torch.zeros((40, K))
        x[:, 0], x[:, 127] = 1.0, 0.5
        for M in (3, 40):
            y = tab_amd.Linear4(x[:M].to(dtype).cuda(), Q.view(torch.float4_e2m1fn_x2).cuda(), S.view(torch.float8_e8m0fnu).cuda(), M, 254, K).cpu().double()
            want = 1.5 * ref8.two_to(torch.arange(1, 255) - 127)
            assert ((y - want).abs() <= 2.0 ** -8 * want).all()


@types
def test_linear4_rows_of_a_wider_matrix(dtype):
    for M in (3, 50):
        x = _rand((M, 400), 8).to(dtype)
        QW, SW = tab_amd.Quantize4(_rand((40, 300), 9).cuda(), 40, 300)
        y = tab_amd.Linear4(x.cuda()[:, 33:333], QW, SW, M, 40, 300)
        assert torch.equal(y, tab_amd.Linear4(x[:, 33:333].contiguous().cuda(), QW, SW, M, 40, 300))


def test_same_call_same_bits():
    x = _rand((70, 8192), 10).cuda()
    QW, SW = tab_amd.Quantize4(_rand((100, 8192), 11).cuda(), 100, 8192)
    first = tab_amd.Linear4(x, QW, SW, 70, 100, 8192)
    for _ in range(5):
        assert torch.equal(first, tab_amd.Linear4(x, QW, SW, 70, 100, 8192))


def test_whole_numbers_are_exact():
    """Products of small whole numbers, in every type and every way."""
    g = torch.Generator("cpu").manual_seed(12)
    w = torch.tensor([0.0, 1, 2, 3, 4, 6, -1, -2, -3, -4, -6])[torch.randint(0, 11, (70, 140), generator=g)]
    w[:, ::32] = 6  # so that every group's scale is one
    w[:, 139] = 6
    for M in (1, 20, 100):
        x = torch.randint(-1, 2, (M, 140), generator=g).float()
        x[:, 0] = 1
        y = x @ w.t()
        keep = y.abs() <= 256  # what bf16 holds
        for dtype in TYPES:
            got = tab_amd.Linear4(x.to(dtype).cuda(), *tab_amd.Quantize4(w.to(dtype).cuda(), 70, 140), M, 70, 140).float().cpu()
            assert torch.equal(got[keep], y[keep])


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.double(), lambda m: m.cpu().cuda(), lambda m: m.to("cuda", torch.bfloat16), copy.deepcopy],
                         ids=["half", "double", "cpu_and_back", "to", "copy"])
def test_layer_keeps_its_weight(convert):
    layer = tab_nn.Linear4.from_float(_rand((30, 300), 34, 1e-6))
    x = _rand((10, 300), 35).view(2, 5, 300).cuda()
    want, qw, sw = layer(x), layer.QW.view(torch.uint8).clone(), layer.SW.view(torch.uint8).clone()
    assert want.shape == (2, 5, 30)
    layer = convert(layer)
    assert layer.QW.dtype == torch.float4_e2m1fn_x2 and layer.SW.dtype == torch.float8_e8m0fnu
    assert torch.equal(layer.QW.view(torch.uint8), qw) and torch.equal(layer.SW.view(torch.uint8), sw)
    assert torch.equal(layer(x), want)
    with pytest.raises(RuntimeError, match="inference"):
        layer(x.requires_grad_())


@pytest.mark.parametrize("M", [2, 300])
def test_weight_past_32_bits(M):
    """A weight of more than 4 GiB, its scales and its outputs far behind its beginning: few rows, and tiles."""
    N, K = 1100003, 8192
    g = torch.Generator("cuda").manual_seed(1)
    QW = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device="cuda").view(torch.float4_e2m1fn_x2)
    SW = torch.randint(120, 128, (K // 128, N, 4), generator=g, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    x = _rand((M, K), 2).to(torch.bfloat16)
    y = tab_amd.Linear4(x.cuda(), QW, SW, M, N, K)
    a = ref8.value(*ref8.quantize(x, 1, 0), 1)
    for n in (slice(0, 200), slice(N - 300, N)):
        want, mag = ref.product(a, ref.unpack4(QW[n], SW[:, n]))
        ref.check(y[:, n], want, mag, K, True, f"columns from {n.start}")
