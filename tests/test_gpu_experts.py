"""Products over experts and their gradients against their definitions in 64 bits."""
import pytest
import torch

import experts_reference as ref
import layers8_reference as ref8
import tab_amd
from tab_amd import _capi
from tab_amd import nn as tab_nn
from test_experts_host import GRAD_WAYS, WAYS

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
types = pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])


def _rand(shape, seed, scale=1.0):
    g = torch.Generator("cpu").manual_seed(seed)
    return torch.randn(shape, generator=g) * torch.exp(torch.randn((shape[0], *[1] * (len(shape) - 1)), generator=g)) * scale


def _pack(w, bits, block_rows=128):
    """Packed weights of E experts and what they stand for."""
    E, N, K = w.shape
    if bits == 8 and block_rows == 1:
        packed = [tab_amd.Quantize8(w[e].cuda(), N, K) for e in range(E)]
        QW = torch.stack([p[0].view(torch.uint8) for p in packed]).view(torch.float8_e4m3fn)
        SW = torch.stack([p[1].view(torch.uint8) for p in packed]).view(torch.float8_e8m0fnu)
    else:
        QW, SW = tab_amd.QuantizeExperts(w.cuda(), E, N, K, bits)
    values = [ref.unpack4(QW[e], SW[e]) if bits == 4 else ref8.unpack(QW[e], SW[e], block_rows) for e in range(E)]
    return QW, SW, values


def _cuda(plan):
    return [t.cuda() for t in plan]


@types
@pytest.mark.parametrize("E,N,K", [(1, 1, 1), (3, 130, 70), (2, 128, 300), (5, 7, 129)])
def test_weights_are_packed_one_by_one(E, N, K, dtype):
    w = _rand((E, N, K), E + N).to(dtype)
    Q, S, QT, ST = tab_amd.QuantizeExperts(w.cuda(), E, N, K, 8, True)
    Q4, S4 = tab_amd.QuantizeExperts(w.cuda(), E, N, K, 4)
    alone = tab_amd.QuantizeExperts(w.cuda(), E, N, K)
    assert torch.equal(alone[0].view(torch.uint8), Q.view(torch.uint8)) and torch.equal(alone[1].view(torch.uint8), S.view(torch.uint8))
    for e in range(E):
        for got, want in zip((Q[e], S[e], QT[e], ST[e]), tab_amd.Quantize8Both(w[e].cuda(), N, K, 128)):
            assert got.shape == want.shape and torch.equal(got.view(torch.uint8), want.view(torch.uint8))
        for got, want in zip((Q4[e], S4[e]), tab_amd.Quantize4(w[e].cuda(), N, K)):
            assert got.shape == want.shape and torch.equal(got.view(torch.uint8), want.view(torch.uint8))


# tokens, choices, experts, N, K: few rows in one launch (one token, odd sizes, an expert with more rows than a workgroup holds), tiles with K whole and in parts,
# experts without rows, more than 64 experts
SIZES = [(1, 1, 1, 1, 1), (1, 3, 5, 40, 300), (2, 2, 2, 17, 129), (16, 4, 64, 96, 1024), (20, 3, 24, 1003, 776), (9, 1, 3, 33, 4096), (30, 2, 90, 50, 260), (40, 2, 4, 65, 129),
         (100, 3, 7, 130, 520), (300, 2, 5, 200, 257), (64, 1, 1, 64, 2000), (129, 4, 130, 70, 300), (700, 2, 3, 140, 640)]


@types
@pytest.mark.parametrize("bits,block_rows", [(8, 128), (8, 1), (4, 1)], ids=["8", "8rows", "4"])
@pytest.mark.parametrize("M,k,E,N,K", SIZES)
def test_rows_of_tokens(M, k, E, N, K, bits, block_rows, dtype):
    x = _rand((M, K), M + K).to(dtype)
    QW, SW, w = _pack(_rand((E, N, K), N, K ** -0.5), bits, block_rows)
    _, _, rows, _, offsets = ref.plan(M, E, k, M + E, closed=M // 9, shy=[E // 2] if E > 4 else [])
    R = M * k
    want, mag = ref.by_expert(ref8.value(*ref8.quantize(x, 1, 0), 1), w, rows, offsets, N)
    y = tab_amd.ExpertsLinear(x.cuda(), rows.cuda(), offsets.cuda(), QW, SW, M, R, E, N, K)
    assert y.shape == (R, N) and not y[int(offsets[-1]):].any()
    ref.check(y, want, mag, K, dtype != torch.float32, "rows of tokens")
    QX, SX = tab_amd.Quantize8(x.cuda(), M, K)
    for out in TYPES:
        y = tab_amd.ExpertsLinearPacked(QX, SX, rows.cuda(), offsets.cuda(), QW, SW, M, R, E, N, K, out)
        assert y.dtype == out and not y[int(offsets[-1]):].any()
        ref.check(y, want, mag, K, out != torch.float32, f"packed to {out}")
    # the same rows, sorted by the caller
    sorted_x = x[rows.clamp(min=0).long()]
    z = tab_amd.ExpertsLinear(sorted_x.cuda(), None, offsets.cuda(), QW, SW, R, R, E, N, K)
    assert torch.equal(z, tab_amd.ExpertsLinear(x.cuda(), rows.cuda(), offsets.cuda(), QW, SW, M, R, E, N, K))
    y = tab_amd.ExpertsLinearPacked(*tab_amd.Quantize8(sorted_x.cuda(), R, K), None, offsets.cuda(), QW, SW, R, R, E, N, K, dtype)
    ref.check(y, want, mag, K, dtype != torch.float32, "sorted rows")


# output type, R, E, N, K: every tile, K whole and in parts
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("out,R,E,N,K,way", WAYS)
def test_every_tile_and_cut(out, R, E, N, K, way, bits):
    """Rows repeat after 64, experts after two: what they stand for is made on the GPU."""
    dtype = [torch.float32, torch.bfloat16][out]
    some, w = _rand((64, K), R).to(torch.bfloat16), _rand((2, N, K), N, K ** -0.5)
    g = torch.Generator("cpu").manual_seed(R + N)
    cuts = torch.sort(torch.randint(0, R + 1, (E,), generator=g)).values.tolist()  # (the last rows are no expert's)
    offsets = torch.tensor([0] + cuts, dtype=torch.int32)
    rows = torch.randint(0, 64, (R,), generator=g, dtype=torch.int32)
    QW, SW, values = _pack(w, bits)
    repeat = [(t.view(torch.uint8).repeat((E + 1) // 2, *[1] * (t.dim() - 1))[:E].contiguous()).view(t.dtype) for t in (QW, SW)]
    QX, SX = tab_amd.Quantize8(some.cuda(), 64, K)
    y = tab_amd.ExpertsLinearPacked(QX, SX, rows.cuda(), offsets.cuda(), *repeat, 64, R, E, N, K, dtype)
    a = ref8.unpack(QX, SX, 1).cuda()
    pairs = [ref.product(a, v.cuda().contiguous()) for v in values]
    want, mag = torch.zeros((R, N), dtype=torch.float64, device="cuda"), torch.zeros((R, N), dtype=torch.float64, device="cuda")
    for e, first, end in ref.runs(offsets):
        at = rows[first:end].long().cuda()
        want[first:end], mag[first:end] = pairs[e % 2][0][at], pairs[e % 2][1][at]
    ref.check(y, want.cpu(), mag.cpu(), K, out != 0, "tiles")
    assert not y[int(offsets[-1]):].any()
    assert torch.equal(y, tab_amd.ExpertsLinearPacked(QX, SX, rows.cuda(), offsets.cuda(), *repeat, 64, R, E, N, K, dtype))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("M", [3, 100])
def test_not_a_number_stays_in_its_rows(M, bits):
    k, E, N, K = 2, 3, 70, 300
    x, w = _rand((M, K), 1), _rand((E, N, K), 2)
    x[1, 299], w[2, 5, 40] = float("nan"), float("inf")
    QW, SW, _ = _pack(w, bits)
    _, experts, rows, places, offsets = ref.plan(M, E, k, 3, closed=1)
    y = tab_amd.ExpertsLinear(x.cuda(), rows.cuda(), offsets.cuda(), QW, SW, M, M * k, E, N, K).cpu()
    want = torch.zeros((M * k, N), dtype=torch.bool)
    for p in places[1].tolist():
        if p >= 0:
            want[p] = True
    want[int(offsets[2]):int(offsets[3]), 5] = True
    assert torch.equal(torch.isnan(y), want)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("M", [4, 90])
def test_rows_and_offsets_that_are_not_right(M, bits):
    """A row outside X counts as zeros, offsets out of order or range are cut: nothing else is read, and the other rows are as they are."""
    E, N, K = 4, 40, 200
    x = _rand((M, K), 1).to(torch.bfloat16)
    QW, SW, w = _pack(_rand((E, N, K), 2, 0.1), bits)
    rows = torch.arange(M, dtype=torch.int32)
    rows[1], rows[3] = 1 << 30, -7
    offsets = torch.tensor([-5, M // 2, M // 4, M // 2, 9 * M], dtype=torch.int32)
    cut = torch.tensor([0, M // 2, M // 2, M // 2, M], dtype=torch.int32)
    a = ref8.value(*ref8.quantize(x, 1, 0), 1)
    a[1], a[3] = 0, 0
    want, mag = ref.by_expert(a, w, torch.arange(M, dtype=torch.int32), cut, N)
    # expert 2's run is M/4 .. M/2 as its own offsets say; each row is then one of two experts', whichever wrote it last: those rows are left out
    keep = torch.ones(M, dtype=torch.bool)
    keep[M // 4:M // 2] = False
    y = tab_amd.ExpertsLinear(x.cuda(), rows.cuda(), offsets.cuda(), QW, SW, M, M, E, N, K)
    ref.check(y.cpu()[keep], want[keep], mag[keep], K, True, "cut")
    sx = tab_amd.Quantize8ByExpert(x.cuda(), rows.cuda(), offsets.cuda(), M, M, E, K)
    dw = tab_amd.ExpertsGradWeight(*sx, *sx, offsets.cuda(), M, E, K, K)
    assert dw.shape == (E, K, K)


@types
def test_columns_of_a_wider_matrix(dtype):
    for M in (3, 80):
        wide = _rand((M, 400), 8).to(dtype).cuda()
        part = wide[:, 33:333]
        QW, SW, _ = _pack(_rand((3, 40, 300), 9), 8)
        _, _, rows, _, offsets = _cuda(ref.plan(M, 3, 2, 4))
        a, b = (tab_amd.ExpertsLinear(v, rows, offsets, QW, SW, M, 2 * M, 3, 40, 300) for v in (part, part.contiguous()))
        assert torch.equal(a, b)


# ---- training ---------------------------------------------------------------------------------------------------------


def _transposed(x, offsets, E, format):
    """The packed transposed rows, expert by expert, as their tensors' used columns and scales."""
    out = []
    for e, a, b in ref.runs(offsets):
        out.append((e, *ref8.quantize(x[a:b].t(), 1, format)))
    return out


@types
@pytest.mark.parametrize("format", [0, 1])
@pytest.mark.parametrize("M,k,E,K", [(1, 1, 1, 1), (5, 2, 3, 130), (200, 3, 4, 70), (300, 2, 70, 7), (400, 1, 2, 300)])
def test_rows_packed_for_the_gradients(M, k, E, K, format, dtype):
    x = _rand((M, K), M + K).to(dtype)
    if K > 100:
        x[1, 3], x[0, 100] = float("inf"), float("nan")
    _, _, rows, _, offsets = ref.plan(M, E, k, M, closed=M // 9)
    R = M * k
    for sort in (False, True):
        xs = x[rows.clamp(min=0).long()]
        if sort:
            Q, S, QT, ST = tab_amd.Quantize8ByExpert(xs.cuda(), None, offsets.cuda(), R, R, E, K, format, True)
            n = int(offsets[-1])
            q, e = ref8.quantize(xs[:n], 1, format)
            assert torch.equal(torch.nan_to_num(Q[:n].cpu().float().double(), nan=1e9), torch.nan_to_num(q, nan=1e9))
            assert torch.equal(S.cpu().view(torch.uint8).long()[:, :n] - 127, e)
        else:
            QT, ST = tab_amd.Quantize8ByExpert(x.cuda(), rows.cuda(), offsets.cuda(), M, R, E, K, format)
        assert QT.shape == (K, 128 * tab_amd.run_blocks(R, E)) and ST.shape == (tab_amd.run_blocks(R, E), K)
        block = 0
        for _, q, e in _transposed(xs, offsets, E, format):
            got = QT.cpu()[:, 128 * block:128 * block + q.shape[1]].float().double()
            assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(q, nan=1e9))
            assert torch.equal(ST.cpu().view(torch.uint8).long()[block:block + e.shape[0]] - 127, e)
            block += e.shape[0]


TRAIN = [(1, 1, 1, 1, 1), (5, 2, 3, 130, 70), (33, 3, 7, 39, 52), (130, 2, 4, 72, 300), (300, 4, 5, 260, 129), (200, 1, 1, 64, 128), (90, 2, 70, 20, 33)]


@types
@pytest.mark.parametrize("format", [0, 1])
@pytest.mark.parametrize("gather", [True, False], ids=["tokens", "sorted"])
@pytest.mark.parametrize("M,k,E,N,K", TRAIN)
def test_gradients_are_products_of_packed_operands(M, k, E, N, K, gather, format, dtype):
    R = M * k
    plan = ref.plan(M, E, k, M + N, closed=M // 9, shy=[1] if E > 4 else [])
    _, _, rows, places, offsets = plan
    x, w, dy = _rand((M if gather else R, K), 12).to(dtype), _rand((E, N, K), 13, 0.2).to(dtype), _rand((R, N), 14, 1e-2).to(dtype)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = tab_nn.experts_linear8(xd, wd, tab_nn.Routing(*_cuda(plan)), gather, format)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.cuda())
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == dtype and dx.shape == x.shape and dw.shape == w.shape
    qw = [ref.rounded(w[e], 128, 0) for e in range(E)]
    sixteen = dtype != torch.float32
    ref.check(y, *ref.by_expert(ref.rounded(x, 1, 0), qw, rows if gather else None, offsets, N), K, sixteen, "y")
    want, mag = ref.by_expert(ref.rounded(dy, 1, format), [v.t() for v in qw], None, offsets, K)
    if gather:  # the sum over a token's rows: k more roundings
        at, chosen = places.clamp(min=0).long(), (places >= 0)[..., None]
        want, mag = ((chosen * v[at]).sum(dim=1) for v in (want, mag))
    ref.check(dx, want, mag, N + k, sixteen, "dx")
    want, mag = (torch.zeros((E, N, K), dtype=torch.float64) for _ in range(2))
    for e, a, b in ref.runs(offsets):
        xe = x[rows[a:b].long()] if gather else x[a:b]
        want[e], mag[e] = ref.product(ref.rounded(dy[a:b].t(), 1, format), ref.rounded(xe.t(), 1, 0))
    ref.check(dw, want, mag, R, sixteen, "dw")


@pytest.mark.parametrize("out,R,E,N,K,way", GRAD_WAYS)
def test_gradients_of_weights_by_every_tile(out, R, E, N, K, way):
    dtype = [torch.float32, torch.bfloat16][out]
    g = torch.Generator("cpu").manual_seed(R)
    offsets = torch.tensor([0] + torch.sort(torch.randint(0, R + 1, (E,), generator=g)).values.tolist(), dtype=torch.int32)
    x, dy = _rand((R, K), 1).to(torch.bfloat16), _rand((R, N), 2).to(torch.bfloat16)
    qx, qd = (tab_amd.Quantize8ByExpert(t.cuda(), None, offsets.cuda(), R, R, E, n) for t, n in ((x, K), (dy, N)))
    dw = tab_amd.ExpertsGradWeight(*qd, *qx, offsets.cuda(), R, E, N, K, dtype)
    block = 0
    for e in range(E):
        a, b = int(offsets[e]), int(offsets[e + 1])
        n = -(-(b - a) // 128)
        if n == 0:
            assert not dw[e].any()
            continue
        d, v = (ref8.unpack(q[:, 128 * block:128 * (block + n)], s[block:block + n], 1).cuda() for q, s in (qd, qx))
        want, mag = ref.product(d, v.contiguous())
        ref.check(dw[e], want.cpu(), mag.cpu(), b - a, out != 0, f"expert {e}")
        block += n
    assert torch.equal(dw, tab_amd.ExpertsGradWeight(*qd, *qx, offsets.cuda(), R, E, N, K, dtype))


def test_gradients_are_differences():
    """Small whole numbers are 8-bit numbers whatever their block's scale, so y is exact and its differences are its derivatives."""
    g = torch.Generator("cpu").manual_seed(15)
    M, k, E, N, K = 6, 2, 3, 5, 140
    plan = ref.plan(M, E, k, 3, closed=1)
    routing = tab_nn.Routing(*_cuda(plan))
    x, w, dy = (torch.randint(-3, 4, s, generator=g).float() for s in ((M, K), (E, N, K), (M * k, N)))
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    dx, dw = torch.autograd.grad(tab_nn.experts_linear8(xd, wd, routing), (xd, wd), dy.cuda())
    f = lambda a, b: float((tab_nn.experts_linear8(a.cuda(), b.cuda(), routing).cpu() * dy).sum())  # noqa: E731
    for at in ((0, 0), (3, 77), (5, 139)):
        d = torch.zeros_like(x)
        d[at] = 1
        assert f(x + d, w) - f(x - d, w) == 2 * float(dx[at])
    for at in ((0, 0, 0), (1, 2, 128), (2, 4, 139)):
        d = torch.zeros_like(w)
        d[at] = 1
        assert f(x, w + d) - f(x, w - d) == 2 * float(dw[at])


def test_partial_and_expanded_gradients():
    M, k, E, N, K = 40, 2, 3, 30, 200
    plan = ref.plan(M, E, k, 5)
    routing = tab_nn.Routing(*_cuda(plan))
    x, w = _rand((M, K), 16).cuda(), _rand((E, N, K), 17).cuda()
    both = [t.detach().requires_grad_() for t in (x, w)]
    y = tab_nn.experts_linear8(*both, routing)
    dx, dw = torch.autograd.grad(y.sum(), both)
    a = x.view(2, 20, K).detach().requires_grad_()
    tab_nn.experts_linear8(a, w, routing).sum().backward()
    assert a.grad.shape == a.shape and torch.equal(a.grad.view(M, K), dx)
    b = w.detach().requires_grad_()
    tab_nn.experts_linear8(x, b, routing).sum().backward()
    assert torch.equal(b.grad, dw)
    wide = torch.stack((w, w), dim=1).detach()[:, 0].requires_grad_()  # not contiguous
    assert not wide.is_contiguous()
    tab_nn.experts_linear8(x, wide, routing).sum().backward()
    assert torch.equal(wide.grad, dw)
    y = tab_nn.experts_linear8(*both, routing)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(y.sum(), both, create_graph=True)
    y = tab_nn.experts_linear8(*both, routing)
    y *= 2  # no view
    with torch.no_grad():
        assert torch.equal(tab_nn.experts_linear8(*both, routing) * 2, y)


def test_activations_of_16_bits_and_weights_of_32():
    """Weights that are bf16 numbers, held in fp32: the same y and dx, and dw in the weights' type."""
    M, k, E, N, K = 90, 2, 4, 70, 260
    routing = tab_nn.Routing(*_cuda(ref.plan(M, E, k, 6)))
    x, w = _rand((M, K), 20).to(torch.bfloat16).cuda().requires_grad_(), _rand((E, N, K), 21).to(torch.bfloat16).cuda().requires_grad_()
    wide = w.detach().float().requires_grad_()
    dy = _rand((M * k, N), 22).to(torch.bfloat16).cuda()
    y, z = tab_nn.experts_linear8(x, w, routing), tab_nn.experts_linear8(x, wide, routing)
    assert z.dtype == torch.bfloat16 and torch.equal(y, z)
    (dx, dw), (dx2, dw2) = torch.autograd.grad(y, (x, w), dy), torch.autograd.grad(z, (x, wide), dy)
    assert torch.equal(dx, dx2) and dw2.dtype == torch.float32
    # both are sums of the same products: one bound for each
    d, v = dy.double().cpu(), x.detach().double().cpu()
    rows, offsets = routing.rows.cpu(), routing.offsets.cpu()
    for e, first, end in ref.runs(offsets):
        want, mag = ref.product(ref.rounded(d[first:end].t(), 1, 0), ref.rounded(v[rows[first:end].long()].t(), 1, 0))
        ref.check(dw[e], want, mag, end - first, True, "16 bits")
        ref.check(dw2[e], want, mag, end - first, False, "32 bits")


@pytest.mark.parametrize("R", [30, 9000])
@pytest.mark.parametrize("bits", [8, 4])
def test_fp32_outputs_with_the_sums_of_16_bits(bits, R):
    """full_sums 0 through the C ABI: within its bound; with weights of 4 bits there is no such form, the sums are the full ones."""
    E, N, K = 8, 1024, 300
    x, w = _rand((R, K), 30).to(torch.bfloat16), _rand((E, N, K), 31, 0.1)
    QW, SW, values = _pack(w, bits)
    QX, SX = tab_amd.Quantize8(x.cuda(), R, K)
    g = torch.Generator("cpu").manual_seed(32)
    offsets = torch.sort(torch.randint(0, R + 1, (E + 1,), generator=g)).values.int()
    offsets[0] = 0
    lib, on = _capi.load(), offsets.cuda()
    y = [torch.full((R, N), float("nan"), device="cuda") for _ in range(2)]
    for full in (0, 1):
        size = lib.tab_experts_linear_packed_workspace_bytes(0, full, bits, R, E, N, K)
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        status = lib.tab_experts_linear_packed(QX.data_ptr(), 0, SX.data_ptr(), R, None, on.data_ptr(), QW.data_ptr(), SW.data_ptr(), bits, 128, R, E, N, K, y[full].data_ptr(),
                                               0, full, ws.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
        assert status == 0, lib.tab_last_error().decode()
    a = ref8.unpack(QX, SX, 1)
    want, mag = torch.zeros((R, N), dtype=torch.float64), torch.zeros((R, N), dtype=torch.float64)
    for e, first, end in ref.runs(offsets):
        want[first:end], mag[first:end] = ref.product(a[first:end], values[e])
    ref.check(y[1], want, mag, K, False, "full sums")
    ref.check(y[0], want, mag, K, bits == 8, "sums of 16 bits")
    if bits == 4:
        assert torch.equal(y[0], y[1])


def _random_weights(E, N, K, bits, seed):
    """Packed weights by bytes: finite numbers of any size, scales from 2^-7 to 1."""
    g = torch.Generator("cuda").manual_seed(seed)
    KB = -(-K // 128)
    if bits == 8:
        q = torch.randint(0, 256, (E, N, KB * 128), generator=g, dtype=torch.uint8, device="cuda").bitwise_and_(0xB7).view(torch.float8_e4m3fn)
        s = torch.randint(120, 128, (E, KB, -(-N // 128)), generator=g, dtype=torch.uint8, device="cuda")
    else:
        q = torch.randint(0, 256, (E, N, KB * 64), generator=g, dtype=torch.uint8, device="cuda").view(torch.float4_e2m1fn_x2)
        s = torch.randint(120, 128, (E, KB, N, 4), generator=g, dtype=torch.uint8, device="cuda")
    return q, s.view(torch.float8_e8m0fnu)


@pytest.mark.parametrize("R", [70, 9000])
@pytest.mark.parametrize("bits,E", [(8, 70), (4, 140)])
def test_weights_past_32_bits(bits, E, R):
    """Experts whose weights begin past 4 GiB: few rows to an expert, and tiles.  (K is a whole number of blocks: what is behind K would not be zeros.)"""
    N, K = 7683, 8192  # N - 387 is a whole number of blocks
    QW, SW = _random_weights(E, N, K, bits, 1)
    assert E * N * K * bits // 8 > 1 << 32
    x = _rand((50, K), 2).to(torch.bfloat16)
    g = torch.Generator("cpu").manual_seed(3)
    rows = torch.randint(0, 50, (R,), generator=g, dtype=torch.int32)
    offsets = torch.sort(torch.randint(0, R + 1, (E + 1,), generator=g)).values.int()
    offsets = offsets.clamp(max=R - R // 9)  # the last expert has rows
    offsets[0], offsets[E] = 0, R
    y = tab_amd.ExpertsLinear(x.cuda(), rows.cuda(), offsets.cuda(), QW, SW, 50, R, E, N, K)
    a = ref8.value(*ref8.quantize(x, 1, 0), 1)
    for e in (0, E // 2, E - 1):
        first, end = int(offsets[e]), min(int(offsets[e + 1]), int(offsets[e]) + 40)
        n = slice(N - 300, N)
        if bits == 8:
            w = ref8.unpack(QW[e, N - 387:], SW[e][:, (N - 387) // 128:], 128)[-300:]
        else:
            w = ref.unpack4(QW[e, n], SW[e][:, n])
        want, mag = ref.product(a[rows[first:end].long()], w)
        ref.check(y[first:end, n], want, mag, K, True, f"expert {e}")


def test_outputs_past_32_bits():
    """Rows of Y, and gradients of weights, that begin past 4 GiB (and past 2^31 elements)."""
    R, E, N, K = 600000, 3, 4000, 64
    x = _rand((77, K), 4).to(torch.bfloat16)
    QW, SW, w = _pack(_rand((E, N, K), 5, K ** -0.5), 8)
    rows = torch.arange(R, dtype=torch.int32) % 77
    offsets = torch.tensor([0, 1000, 1001, R - 5], dtype=torch.int32)
    y = tab_amd.ExpertsLinear(x.cuda(), rows.cuda(), offsets.cuda(), QW, SW, 77, R, E, N, K)
    assert y.numel() > 1 << 31
    a = ref8.value(*ref8.quantize(x, 1, 0), 1)
    for e, first, end in ((0, 0, 200), (2, 1001, 1300), (2, R - 300, R - 5)):
        want, mag = ref.product(a[rows[first:end].long()], w[e])
        ref.check(y[first:end], want, mag, K, True, f"rows {first}")
    assert not y[R - 5:].any()
    # back to the tokens: k = 2
    places = torch.arange(R, dtype=torch.int32).view(-1, 2)
    out = tab_amd.Combine(y, places.cuda(), None, R // 2, 2, R, N)
    last = y[R - 40:].double().cpu()
    ref.check(out[R // 2 - 20:], last[0::2] + last[1::2], last[0::2].abs() + last[1::2].abs(), 2, False, "combine")
    del out
    dout = torch.randn((R // 2, N), device="cuda", dtype=torch.bfloat16)
    dy, dweights = tab_amd.CombineBackward(dout, y, places.cuda(), torch.ones((R // 2, 2), device="cuda"), None, R // 2, 2, R, N)
    assert torch.equal(dy[0::2], dout) and torch.equal(dy[1::2], dout)
    d = dout[R // 2 - 20:].double().cpu()
    for j in (0, 1):
        ref.check(dweights[R // 2 - 20:, j], (d * last[j::2]).sum(1), (d * last[j::2]).abs().sum(1), N, False, "dweights")


def test_gradients_past_32_bits():
    R, E, N, K = 3000, 33, 8192, 8200
    g = torch.Generator("cpu").manual_seed(6)
    offsets = torch.sort(torch.randint(0, R - 99, (E + 1,), generator=g)).values.int()
    offsets[0], offsets[E] = 0, R
    x, dy = _rand((R, K), 7).to(torch.bfloat16), _rand((R, N), 8).to(torch.bfloat16)
    qx, qd = (tab_amd.Quantize8ByExpert(t.cuda(), None, offsets.cuda(), R, R, E, n) for t, n in ((x, K), (dy, N)))
    dw = tab_amd.ExpertsGradWeight(*qd, *qx, offsets.cuda(), R, E, N, K, torch.bfloat16)
    assert dw.numel() > 1 << 31
    e, a = E - 1, int(offsets[E - 1])
    want, mag = ref.product(ref.rounded(dy[a:, N - 50:].t(), 1, 0), ref.rounded(x[a:, K - 70:].t(), 1, 0))
    ref.check(dw[e, N - 50:, K - 70:], want, mag, R - a, True, "the last expert")


@pytest.mark.parametrize("bits,dtype", [(8, torch.bfloat16), (4, torch.float32)])
def test_sorted_rows_past_32_bits(bits, dtype):
    """Rows that come sorted, past 4 GiB of packed numbers: each tile reads its own, so there is no bound on all of them as there is on listed ones."""
    R, E, N, K = 560000, 3, 40, 8192
    g = torch.Generator("cuda").manual_seed(11)
    x = torch.randint(-3, 4, (R, K), generator=g, dtype=torch.int8, device="cuda").to(dtype)
    w = torch.randint(-3, 4, (E, N, K), generator=torch.Generator("cpu").manual_seed(12)).float()  # (no number of 4 bits is 5)
    QW, SW = tab_amd.QuantizeExperts(w.cuda(), E, N, K, bits)
    offsets = torch.tensor([0, 1000, 300003, R - 77], dtype=torch.int32)
    y = tab_amd.ExpertsLinear(x, None, offsets.cuda(), QW, SW, R, R, E, N, K)
    assert not y[R - 77:].any()
    for e, first, end in ((0, 0, 1000), (1, 1000, 1300), (1, 299000, 300003), (2, 300003, 300300), (2, R - 700, R - 77)):
        want = x[first:end].double().cpu() @ w[e].double().t()  # whole numbers below 2^17: exact but for the output's rounding
        assert torch.equal(y[first:end].cpu(), want.to(dtype)), f"rows {first}"


def test_training_past_32_bits():
    """Gradients of more sorted rows than listed ones could be: what the forward pass takes, the backward pass takes."""
    M, k, E, N, K = 280000, 2, 3, 8192, 16
    R = M * k
    assert R * N > 1 << 32
    g = torch.Generator("cpu").manual_seed(13)
    x = torch.randint(-4, 5, (M, K), generator=g).to(torch.bfloat16)
    w = torch.randint(-3, 4, (E, N, K), generator=g).float()
    routing = tab_nn.route(torch.randn((M, E), generator=g).cuda(), k)
    rows, places, offsets = (t.cpu() for t in routing[2:])
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    y = tab_nn.experts_linear8(xd, wd, routing)
    dy = torch.randint(-1, 2, (R, N), generator=torch.Generator("cuda").manual_seed(14), dtype=torch.int8, device="cuda").to(torch.bfloat16)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy)
    x64, w64, at = x.double(), w.double(), offsets.tolist()
    for e in range(E):
        first, end = at[e], at[e + 1]
        assert torch.equal(y[end - 50:end].cpu().double(), x64[rows[end - 50:end].long()] @ w64[e].t()), f"expert {e}"  # whole numbers up to 192
        n = slice(N - 40, N)
        assert torch.equal(dw[e, n].cpu().double(), dy[first:end, n].double().cpu().t() @ x64[rows[first:end].long()]), f"gradient of weight {e}"  # below 2^24
    for t in (0, 1, M // 2, *range(M - 60, M)):
        want = 0
        for p in places[t].tolist():
            e = next(e for e in range(E) if at[e] <= p < at[e + 1])
            want = want + dy[p].double().cpu() @ w64[e]
        assert torch.equal(dx[t].cpu(), want.to(torch.bfloat16)), f"gradient of token {t}"


def test_training_is_refused_before_its_first_product():
    """More rows than the gradients of the weights may have: the forward pass says so where a gradient of them is wanted, and runs where none is."""
    M, E, N, K = 128 * 65535 + 1, 1, 8, 8
    x, w = torch.ones((M, K), device="cuda", dtype=torch.bfloat16), torch.ones((E, N, K), device="cuda", dtype=torch.bfloat16)
    routing = tab_nn.route(torch.zeros((M, E), device="cuda"), 1)
    with pytest.raises(tab_amd.TabError, match="blocks of rows"):
        tab_nn.experts_linear8(x, w.requires_grad_(), routing)
    y = tab_nn.experts_linear8(x.requires_grad_(), w.detach(), routing)
    assert (y == K).all()
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert (dx == N).all()
