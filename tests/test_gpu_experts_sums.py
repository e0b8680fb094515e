"""Sums of the 4-bit layers, of products over experts and of their gradients as a whole: the mean of all errors, and rows that do not depend on the batch that they
are in."""
import pytest
import torch

import experts_reference as ref
import layers8_reference as ref8
import tab_amd
from tab_amd import nn as tab_nn
from test_gpu_layers8_scales import _groups_lose

pytestmark = pytest.mark.gpu

OUT = (torch.float32, torch.bfloat16, torch.float16)


def _rand(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)) * scale


def bounds(a, b):
    """Of operands (.., K) whose products are summed: the sums, what the mean of all errors may be for each type of output, and the mean product.  As for the 8-bit
    layers: each product may lose what a group of eight keeps below its largest (towards 16 bits), K roundings of fp32, of partial sums that are
    differences of two from the start, and half of the output's largest rounding, since that is anywhere within half a unit."""
    products = a * b
    K = products.shape[-1]
    want, partial, lose = products.sum(dim=-1), products.cumsum(dim=-1).abs().amax(dim=-1), _groups_lose(products)
    allowed = {out: float((K * 2.0 ** -24 * 2 * partial + (0 if out == torch.float32 else lose) + ref.UNIT[out] / 2 * want.abs() + ref.TINY[out]).mean()) for out in OUT}
    return want, allowed, float(products.abs().mean())


def check_mean(y, want, allowed, mean_product, what):
    """The mean error is within its bound, and that is below one product lost or counted twice in each sum."""
    mean = float((y.double() - want.to(y.device)).abs().mean())
    assert allowed[y.dtype] < mean_product and mean <= allowed[y.dtype], (what, y.dtype, mean, allowed[y.dtype], mean_product)


def _some(n, most=12):
    return torch.arange(0, n, max(1, n // most))


def linear4_problem(M, N, K):
    x, w = _rand((M, K), 5).to(torch.bfloat16), _rand((N, K), 6, K ** -0.5)
    m, n = _some(M), _some(N, 40)
    a, b = ref8.value(*ref8.quantize(x[m], 1, 0), 1), ref.value4(*ref.quantize4(w[n]))
    return x, w, m, n, bounds(a[:, None, :], b[None, :, :])


# one row, few rows cut up among workgroups, tiles whole and in parts of K, 256 x 256
LINEAR4 = [(1, 300, 2007), (24, 1003, 2050), (64, 300, 4000), (700, 512, 2007), (2214, 2718, 2007)]


@pytest.mark.parametrize("M,N,K", LINEAR4)
def test_mean_error_of_4_bit_layers(M, N, K):
    x, w, m, n, expected = linear4_problem(M, N, K)
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K)
    QW, SW = tab_amd.Quantize4(w.cuda(), N, K)
    for out in OUT:
        check_mean(tab_amd.Linear4Packed(QX, SX, QW, SW, M, N, K, out).cpu()[m][:, n], *expected, "packed")
    check_mean(tab_amd.Linear4(x.cuda(), QW, SW, M, N, K).cpu()[m][:, n], *expected, "x quantized on the way")


def experts_problem(R, E, N, K, bits):
    M = (R + 1) // 2
    x, w = _rand((M, K), 7).to(torch.bfloat16), _rand((E, N, K), 8, K ** -0.5)
    g = torch.Generator("cpu").manual_seed(R + E)
    offsets = torch.tensor([0] + torch.sort(torch.randint(0, R + 1, (E - 1,), generator=g)).values.tolist() + [R], dtype=torch.int32)
    rows = torch.randint(0, M, (R,), generator=g, dtype=torch.int32)
    r, n = _some(R), _some(N, 40)
    expert = torch.searchsorted(offsets.long(), r, right=True) - 1
    a = ref8.value(*ref8.quantize(x[rows[r].long()], 1, 0), 1)
    if bits == 4:
        b = torch.stack([ref.value4(*ref.quantize4(w[e][n])) for e in expert])
    else:
        b = torch.stack([ref8.value(*ref8.quantize(w[e], 128, 0), 128)[n] for e in expert])
    return x, w, rows, offsets, r, n, M, bounds(a[:, None, :], b)


# few rows to an expert, tiles of every size, K whole and in parts
EXPERTS = [(60, 24, 1003, 776), (40, 5, 300, 4000), (1500, 8, 512, 2007), (564, 57, 98, 2007), (9000, 6, 1088, 1003)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("R,E,N,K", EXPERTS)
def test_mean_error_of_products_by_expert(R, E, N, K, bits):
    x, w, rows, offsets, r, n, M, expected = experts_problem(R, E, N, K, bits)
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K)
    QW, SW = tab_amd.QuantizeExperts(w.cuda(), E, N, K, bits)
    for out in OUT:
        y = tab_amd.ExpertsLinearPacked(QX, SX, rows.cuda(), offsets.cuda(), QW, SW, M, R, E, N, K, out)
        check_mean(y.cpu()[r][:, n], *expected, "packed")
    check_mean(tab_amd.ExpertsLinear(x.cuda(), rows.cuda(), offsets.cuda(), QW, SW, M, R, E, N, K).cpu()[r][:, n], *expected, "x quantized on the way")


def gradient_problem(R, E, N, K):
    dy, x = _rand((R, N), 9).to(torch.bfloat16), _rand((R, K), 10, R ** -0.5).to(torch.bfloat16)
    offsets = torch.tensor([R * e // E - (e % 2) * (R // (5 * E)) for e in range(E)] + [R], dtype=torch.int32)
    n, k = _some(N), _some(K)
    expected = []
    for e, first, end in ref.runs(offsets):
        a, b = (ref8.value(*ref8.quantize(t[first:end][:, c].t(), 1, 0), 1) for t, c in ((dy, n), (x, k)))
        expected.append((e, bounds(a[:, None, :], b[None, :, :])))
    return dy, x, offsets, n, k, expected


GRADIENTS = [(3000, 4, 600, 700), (900, 8, 70, 1000), (9000, 6, 1100, 1500)]


@pytest.mark.parametrize("R,E,N,K", GRADIENTS)
def test_mean_error_of_the_weights_gradients(R, E, N, K):
    dy, x, offsets, n, k, expected = gradient_problem(R, E, N, K)
    qd, qx = (tab_amd.Quantize8ByExpert(t.cuda(), None, offsets.cuda(), R, R, E, c) for t, c in ((dy, N), (x, K)))
    for out in OUT:
        dw = tab_amd.ExpertsGradWeight(*qd, *qx, offsets.cuda(), R, E, N, K, out).cpu()
        for e, each in expected:
            check_mean(dw[e][n][:, k], *each, f"expert {e}")


class _Whole(torch.nn.Module):
    """Logits that are whole numbers, whatever the order of the sums."""

    def __init__(self, E, D, seed):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.randint(-2, 3, (E, D), generator=torch.Generator("cpu").manual_seed(seed)).float())

    def forward(self, x):
        return (x.float() @ self.weight.t().contiguous())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rows", [16, 300, 3000])
def test_a_token_does_not_depend_on_its_batch(rows, bits, dtype):
    """Whole numbers: every sum is exact, in any order and cut, by any tile.  The first product's sums stay below 2^11; in 8 bits they are whole numbers of
    four significant bits, so the second's are whole numbers below 2^21, and the products of a group of eight are whole numbers below 2^13, of which nothing is
    lost 13 bits below the largest."""
    D, H, E, k = 200, 140, 12, 3
    g = torch.Generator("cpu").manual_seed(rows)
    up, down = torch.randint(-3, 4, (E, H, D), generator=g).float(), torch.randint(-3, 4, (E, D, H), generator=g).float()
    block = tab_nn.MixtureOfExperts(_Whole(E, D, 3), tab_nn.Experts8(up), tab_nn.Experts8(down), k, activation=torch.nn.ReLU()).cuda().packed(bits)
    x = torch.randint(-2, 3, (rows, D), generator=g).to(dtype).cuda()
    with torch.no_grad():
        got = block(x)
        for t in (0, 1, rows // 2, rows - 1):
            assert torch.equal(block(x[t:t + 1])[0], got[t]), t
        some = torch.arange(0, rows, 3, device="cuda")
        assert torch.equal(block(x[some]), got[some])


# ---- operands that were packed elsewhere: scale bytes that the quantizers do not give -----------------------------------------------------


def _packed8(R, K, seed, byte, block_rows=1):
    """Numbers of 4 to 448 (of 2^-7 to 7/8 under bytes from 253 on) under one scale byte."""
    x = _rand((R, K), seed)
    x = torch.sign(x) * (x.abs() * 40).clamp(4, 448)
    q = torch.zeros(R, ref8.blocks(K) * 128)
    q[:, :K] = ref8.nearest8(x.double(), 0).float() / (512 if byte >= 253 else 1)
    s = torch.full((ref8.blocks(K), -(-R // block_rows)), byte, dtype=torch.uint8)
    return q.to(torch.float8_e4m3fn), s.view(torch.float8_e8m0fnu)


def _packed4(R, K, seed, byte):
    """Numbers 4 and 6 (1/2 under bytes from 253 on) of either sign under one scale byte."""
    g = torch.Generator("cpu").manual_seed(seed)
    code = torch.randint(6, 8, (R, K), generator=g) if byte < 253 else torch.ones((R, K), dtype=torch.int64)
    code = code + 8 * torch.randint(0, 2, (R, K), generator=g)
    c = torch.zeros((R, ref8.blocks(K) * 128), dtype=torch.int64)
    c[:, :K] = code
    q = (c[:, 0::2] | c[:, 1::2] << 4).to(torch.uint8).view(torch.float4_e2m1fn_x2)
    return q, torch.full((ref8.blocks(K), R, 4), byte, dtype=torch.uint8).view(torch.float8_e8m0fnu)


SCALES = [(0, 254), (254, 0), (0, 127), (127, 0), (1, 253), (240, 10)]
outputs = pytest.mark.parametrize("out", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


def _check_scales(y, a, b, out):
    """As for other products; a sum below 2^-126 may count as zero."""
    want, magnitudes = a @ b.t().contiguous(), a.abs() @ b.abs().t().contiguous()
    bound = (a.shape[1] * 2.0 ** -24 + (0 if out == torch.float32 else 2.0 ** -10)) * magnitudes + ref.UNIT[out] * (1 + 2.0 ** -10) * want.abs() + 2.0 ** -126
    off = (y.cpu().double() - want).abs()
    assert off.shape == bound.shape and bool((off <= bound).all()), float((off / bound).max())


@outputs
@pytest.mark.parametrize("M,N,K", [(1, 40, 300), (20, 40, 300), (600, 72, 300), (700, 8299, 130), (2970, 643, 130)])
@pytest.mark.parametrize("x_byte,w_byte", SCALES)
def test_extreme_scales_of_4_bit_weights(x_byte, w_byte, M, N, K, out):
    """2^(byte - 127) for every byte below 255, also 2^-127.  No number is below 2^-126 after its scale, and none above fp32's largest."""
    QX, SX = _packed8(M, K, 1, x_byte)
    QW, SW = _packed4(N, K, 2, w_byte)
    y = tab_amd.Linear4Packed(QX.cuda(), SX.cuda(), QW.cuda(), SW.cuda(), M, N, K, out)
    _check_scales(y, ref8.unpack(QX, SX, 1), ref.unpack4(QW, SW), out)


@outputs
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("R,E,N,K", [(12, 3, 40, 300), (600, 2, 300, 300), (3000, 2, 643, 130)])
@pytest.mark.parametrize("x_byte,w_byte", SCALES + [(127, 255), (255, 127)])
def test_extreme_scales_by_expert(x_byte, w_byte, R, E, N, K, bits, out):
    """The same, and byte 255, which is NaN: one expert's weight has it, or one row of x."""
    x_nan, w_nan = x_byte == 255, w_byte == 255
    QX, SX = _packed8(R, K, 3, 127 if x_nan else x_byte)
    packed = [_packed4(N, K, 4 + e, 127 if w_nan else w_byte) if bits == 4 else _packed8(N, K, 4 + e, 127 if w_nan else w_byte, 128) for e in range(E)]
    b = [ref.unpack4(*p) if bits == 4 else ref8.unpack(*p, 128) for p in packed]
    QW, SW = (torch.stack([p[i].view(torch.uint8) for p in packed]).view(packed[0][i].dtype) for i in (0, 1))
    a = ref8.unpack(QX, SX, 1)
    if x_nan:
        SX.view(torch.uint8)[0, R // 2] = 255
    if w_nan:
        SW.view(torch.uint8)[E - 1] = 255
    offsets = torch.tensor([0] + [R * (e + 1) // E for e in range(E)], dtype=torch.int32)
    y = tab_amd.ExpertsLinearPacked(QX.cuda(), SX.cuda(), None, offsets.cuda(), QW.cuda(), SW.cuda(), R, R, E, N, K, out).cpu()
    nan = torch.zeros((R, N), dtype=torch.bool)
    if x_nan:
        nan[R // 2] = True
    if w_nan:
        nan[int(offsets[E - 1]):] = True
    assert torch.equal(torch.isnan(y), nan)
    for e, first, end in ref.runs(offsets):
        rows = [r for r in range(first, end) if not nan[r].any()]
        if rows:
            _check_scales(y[rows], a[rows], b[e], out)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,E", [(1, 1), (5, 4), (700, 3), (200, 128)])
def test_a_batch_of_padding_alone(rows, E, dtype, normalize):
    """Every expert closed to every token: no rows, zeros out, and zeros for all gradients."""
    N, K, k = 140, 300, min(E, 2)
    x, w = _rand((rows, K), 1).to(dtype).cuda().requires_grad_(), _rand((E, N, K), 2).to(dtype).cuda().requires_grad_()
    logits = torch.full((rows, E), -float("inf"), device="cuda", dtype=dtype, requires_grad=True)
    routing = tab_nn.route(logits, k, normalize)
    assert not routing.offsets.any() and (routing.rows == -1).all() and not routing.weights.any()
    y = tab_nn.experts_linear8(x, w, routing)
    out = tab_nn.combine(y, routing)
    assert y.shape == (rows * k, N) and not y.any() and not out.any()
    for g in torch.autograd.grad(out, (x, w, logits), torch.ones_like(out)):
        assert not g.any()
    with torch.no_grad():
        for bits in (8, 4):
            layer = tab_nn.PackedExperts.from_float(w, bits)
            assert not layer(x.detach(), routing).any() and not layer(_rand((rows * k, K), 3).to(dtype).cuda(), routing, gather=False).any()
