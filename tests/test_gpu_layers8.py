"""8-bit quantizers and products against their definitions in 64 bits: packed numbers and scales equal, products within what fp32 sums and
one rounding allow."""
import pytest
import torch

import layers8_reference as ref
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
types = pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])


def _rand(shape, seed, scale=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    return torch.randn(shape, generator=g) * torch.exp(torch.randn((shape[0], 1), generator=g)) * scale


def _same_packed(Q, S, x, block_rows, format):
    q, e = ref.quantize(x, block_rows, format)
    got, exponents = Q.cpu().to(torch.float32).double(), S.cpu().view(torch.uint8).long() - 127
    assert got.shape == q.shape and exponents.shape == e.shape
    assert torch.equal(exponents, e)
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(q, nan=1e9))


def _check_quantize(x, xd, block_rows, format):
    M, K = x.shape
    Q, S = tab_amd.Quantize8(xd, M, K, block_rows, format)
    _same_packed(Q, S, x, block_rows, format)
    QT, ST = tab_amd.Quantize8Transposed(xd, M, K, block_rows, format)
    _same_packed(QT, ST, x.t(), block_rows, format)
    both = tab_amd.Quantize8Both(xd, M, K, block_rows, format)
    for a, b in zip(both, (Q, S, QT, ST)):
        assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@types
@pytest.mark.parametrize("format", [0, 1])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (128, 129), (131, 300), (33, 1000), (257, 64), (500, 8)])
def test_quantize(M, K, block_rows, format, dtype):
    x = _rand((M, K), M * 1000 + K).to(dtype)
    _check_quantize(x, x.cuda(), block_rows, format)


@types
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("wide,at", [(1, 0), (8, 8), (27, 13)])
def test_quantize_rows_of_a_wider_matrix(wide, at, block_rows, dtype):
    x = _rand((37, 261 + wide), 5).to(dtype)
    xd = x.cuda()[:, at:at + 261]
    assert not xd.is_contiguous()
    _check_quantize(x[:, at:at + 261], xd, block_rows, 0)


@types
@pytest.mark.parametrize("format", [0, 1])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_special_values(block_rows, format, dtype):
    """Blocks of zeros, magnitudes at and beside the bound of a scale, subnormals, the type's extremes, infinities and NaN beside finite
    values, ties between two 8-bit numbers."""
    big = torch.finfo(dtype).max
    smallest = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    one = 1 + torch.finfo(dtype).eps
    rows = [[0.0], [-0.0, 0.0], [448.0, 1.0, -3.0], [448.0 * one, 1.0], [1.75, 1.75 * one, -1.75], [57344.0, 1.0, -2.0 ** -14],
            [smallest, -smallest, 3 * smallest], [big, -big, 1.0], [float("inf"), 2.0, -1.0], [float("-inf"), float("nan"), 0.5], [float("nan")],
            [float("inf"), float("-inf")], [17.0, 19.0, 21.0, -17.0, 448.0, 2.0 ** -9 * 0.5, 2.0 ** -9 * 1.5], [1e-3, 60000.0, -2e-5]]
    x = torch.zeros((len(rows), 130))
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
        x[i, 128] = r[0]
    x = x.to(dtype)
    _check_quantize(x, x.cuda(), block_rows, format)


def test_quantize_takes_no_scale_below_the_smallest():
    x = torch.full((2, 128), 2.0 ** -140)
    Q, S = tab_amd.Quantize8(x.cuda(), 2, 128)
    assert (S.view(torch.uint8) == 1).all()
    _same_packed(Q, S, x, 1, 0)


def _check_product(y, a, b, what):
    """a (M, K), b (N, K) fp64, what the operands stand for.  fp32 output: products of 4-bit mantissas are exact in fp32; the sums have at most
    K - 1 roundings of partial sums, each bounded by the sum of magnitudes.  16-bit output: besides, each product of a group of eight in K
    loses at most 2^-13 of the group's largest, which is at most the group's sum of magnitudes: 2^-10 of the sum of magnitudes over all
    groups.  Then one rounding to the output's type."""
    want, magnitudes = a @ b.t(), a.abs() @ b.abs().t()
    bound = (a.shape[1] * 2.0 ** -24 + (0 if y.dtype == torch.float32 else 2.0 ** -10)) * magnitudes + ref.UNIT[y.dtype] * (1 + 2.0 ** -10) * want.abs() + ref.TINY[y.dtype]
    got = y.cpu().double()
    assert got.shape == want.shape, what
    if y.dtype == torch.float16:  # beyond the type's range it is an infinity
        inside = want.abs() < 65000
        got, want, bound = got[inside], want[inside], bound[inside]
    off = (got - want).abs()
    assert (off <= bound).all(), (what, float((off / bound).max()))


# every way the product is computed: rows (1 .. 32), tiles of 64 with K in parts and whole, of 128, of 256
SIZES = [(1, 1, 1), (1, 16, 128), (1, 1000, 2050), (2, 17, 129), (15, 40, 1024), (15, 33, 4096), (16, 33, 4096), (17, 20, 4096), (16, 100, 640), (16, 8300, 130), (17, 33, 300), (31, 64, 128), (32, 130, 2000), (33, 5, 77),
         (40, 1003, 640), (64, 64, 128), (65, 65, 1153), (100, 72, 8192), (3, 50, 30000), (129, 300, 257), (300, 129, 4000), (500, 777, 520)]


@types
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_linear8(M, N, K, block_rows, dtype):
    x = _rand((M, K), M + N + K).to(dtype)
    w = _rand((N, K), M + 2 * N, K ** -0.5)
    if M > 3:
        x[2] = 0
    QW, SW = tab_amd.Quantize8(w.cuda(), N, K, block_rows)
    a = ref.value(*ref.quantize(x, 1, 0), 1)
    b = ref.unpack(QW, SW, block_rows)
    _check_product(tab_amd.Linear8(x.cuda(), QW, SW, M, N, K), a, b, "Linear8")
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K)
    for out in TYPES:
        y = tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K, out)
        assert y.dtype == out
        _check_product(y, a, b, f"Linear8Packed to {out}")


@pytest.mark.parametrize("M,N,K", [(1, 50, 300), (20, 70, 500), (70, 200, 700), (200, 90, 5000)])
def test_wide_format_operand(M, N, K):
    x, w = _rand((M, K), 1, 1e-3), _rand((N, K), 2)
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K, 1, tab_amd.E5M2)
    QW, SW = tab_amd.Quantize8(w.cuda(), N, K, 128)
    assert QX.dtype == torch.float8_e5m2
    _check_product(tab_amd.Linear8Packed(QX, SX, QW, SW, M, N, K), ref.value(*ref.quantize(x, 1, 1), 1), ref.unpack(QW, SW, 128), "E5M2")


@pytest.mark.parametrize("M,N,K", [(1024, 4096, 256), (2100, 4000, 130), (4096, 4100, 384), (4099, 4097, 128)])
def test_large_tiles(M, N, K):
    """Outputs of many tiles: enough for those of 128 and of 256; ragged edges."""
    x, w = _rand((M, K), 3).to(torch.bfloat16), _rand((N, K), 4, 0.1)
    QW, SW = tab_amd.Quantize8(w.cuda(), N, K, 128)
    y = tab_amd.Linear8(x.cuda(), QW, SW, M, N, K)
    _check_product(y, ref.value(*ref.quantize(x, 1, 0), 1), ref.unpack(QW, SW, 128), "tiles")


@pytest.mark.parametrize("M", [1, 20, 70])
def test_not_a_number_stays_in_its_row_and_column(M):
    N, K = 80, 400
    x, w = _rand((M, K), 5), _rand((N, K), 6)
    x[0, 200], w[7, 130] = float("inf"), float("nan")
    QW, SW = tab_amd.Quantize8(w.cuda(), N, K, 128)
    y = tab_amd.Linear8(x.cuda(), QW, SW, M, N, K).cpu()
    want = torch.zeros((M, N), dtype=torch.bool)
    want[0], want[:, 7] = True, True
    assert torch.equal(torch.isnan(y), want)
    x[0, 200], w[7, 130] = 0.0, 0.0
    clean = torch.isfinite(y)
    a, b = ref.value(*ref.quantize(x, 1, 0), 1), ref.value(*ref.quantize(w, 128, 0), 128)
    want = a @ b.t()
    assert ((y.double() - want).abs()[clean] <= (K * 2.0 ** -24 * (a.abs() @ b.abs().t()) + 2.0 ** -24 * want.abs())[clean]).all()


@types
def test_linear8_rows_of_a_wider_matrix(dtype):
    for M in (3, 50):
        x = _rand((M, 400), 8).to(dtype)
        w = _rand((40, 300), 9)
        QW, SW = tab_amd.Quantize8(w.cuda(), 40, 300, 128)
        part = x[:, 33:333]
        y = tab_amd.Linear8(x.cuda()[:, 33:333], QW, SW, M, 40, 300)
        assert torch.equal(y, tab_amd.Linear8(part.contiguous().cuda(), QW, SW, M, 40, 300))
        _check_product(y, ref.value(*ref.quantize(part, 1, 0), 1), ref.unpack(QW, SW, 128), "wide")


def test_same_call_same_bits():
    x, w = _rand((70, 8192), 10).cuda(), _rand((100, 8192), 11).cuda()
    QW, SW = tab_amd.Quantize8(w, 100, 8192, 128)
    first = tab_amd.Linear8(x, QW, SW, 70, 100, 8192)
    for _ in range(5):
        assert torch.equal(first, tab_amd.Linear8(x, QW, SW, 70, 100, 8192))


# ---- training ---------------------------------------------------------------------------------------------------------


@types
@pytest.mark.parametrize("format", [0, 1])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 130, 70), (130, 72, 300), (300, 260, 129)])
def test_gradients_are_products_of_packed_operands(M, N, K, format, dtype):
    x, w, dy = _rand((M, K), 12).to(dtype), _rand((N, K), 13, 0.2).to(dtype), _rand((M, N), 14, 1e-2).to(dtype)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = tab_nn.linear8(xd, wd, grad_format=format)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == dtype
    qx, qw = ref.value(*ref.quantize(x, 1, 0), 1)[:, :K], ref.value(*ref.quantize(w, 128, 0), 128)[:, :K]
    _check_product(y.detach(), qx, qw, "y")
    _check_product(dx, ref.value(*ref.quantize(dy, 1, format), 1)[:, :N], qw.t(), "dx")
    _check_product(dw, ref.value(*ref.quantize(dy.t(), 1, format), 1)[:, :M], ref.value(*ref.quantize(x.t(), 1, 0), 1)[:, :M], "dw")


def test_gradients_are_differences():
    """Small whole numbers are 8-bit numbers whatever their block's scale, so y is x w^T exactly and its differences are its derivatives."""
    g = torch.Generator("cpu").manual_seed(15)
    M, N, K = 6, 5, 140
    x, w, dy = (torch.randint(-3, 4, s, generator=g).float() for s in ((M, K), (N, K), (M, N)))
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = tab_nn.linear8(xd, wd)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    f = lambda a, b: float((tab_nn.linear8(a.cuda(), b.cuda()).cpu() * dy).sum())  # noqa: E731
    for m, k in ((0, 0), (3, 77), (5, 139)):
        d = torch.zeros_like(x)
        d[m, k] = 1
        assert f(x + d, w) - f(x - d, w) == 2 * float(dx[m, k])
    for n, k in ((0, 0), (2, 128), (4, 139)):
        d = torch.zeros_like(w)
        d[n, k] = 1
        assert f(x, w + d) - f(x, w - d) == 2 * float(dw[n, k])


def test_gradients_of_expanded_and_partial_inputs():
    """A gradient of ones that was never written out, an input with more dimensions, one operand without a gradient."""
    x, w = _rand((6, 200), 16).cuda(), _rand((30, 200), 17).cuda()
    a = x.view(2, 3, 200).detach().requires_grad_()
    y = tab_nn.linear8(a, w)
    assert y.shape == (2, 3, 30)
    y.sum().backward()
    ones = ref.value(*ref.quantize(torch.ones(6, 30), 1, 0), 1)[:, :30]
    _check_product(a.grad.view(6, 200), ones, ref.value(*ref.quantize(w.cpu(), 128, 0), 128)[:, :200].t(), "dx")
    b = w.detach().requires_grad_()
    tab_nn.linear8(x, b).sum().backward()
    _check_product(b.grad, ones.t(), ref.value(*ref.quantize(x.cpu().t(), 1, 0), 1)[:, :6], "dw")
    y = tab_nn.linear8(a, b)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y.sum(), a, create_graph=True)
    with torch.no_grad():
        assert not tab_nn.linear8(a, b).requires_grad
