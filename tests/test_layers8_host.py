"""Refusals of the 8-bit layers and the norms, through the C ABI and from Python: bad arguments are named before anything is launched (no GPU is
touched)."""
import ctypes

import pytest
import torch

import tab_amd
from tab_amd import _capi
from tab_amd import nn as tab_nn

P = 4096  # an aligned address that is never dereferenced: every call below fails its checks

# (0 fp32 or 1 16-bit output, M, N, K, half of the tile's rows + columns * 100 + parts of K): every tile, K whole and in parts, one step of K and
# many
WAYS = [(0, 34, 35, 60, 6401), (0, 33, 34, 940, 6408), (0, 65, 8299, 63, 9601), (0, 578, 1252, 6526, 9604), (0, 2970, 643, 60, 12801),
        (0, 2100, 4003, 500, 12801), (1, 34, 35, 60, 6401), (1, 37, 33, 2708, 6408), (1, 65, 8299, 63, 9601), (1, 2100, 2050, 1100, 9601),
        (1, 260, 771, 6986, 9604), (1, 2970, 643, 60, 12801), (1, 2322, 833, 903, 12801), (1, 1425, 8304, 61, 25601),
        (1, 3343, 3616, 252, 25601), (1, 1283, 9011, 2007, 25601), (1, 2214, 2718, 10855, 25602)]


def _refuses(status, message, code=-1):
    assert status == code, status
    assert message in _capi.load().tab_last_error().decode()


@pytest.mark.parametrize("out,M,N,K,way", WAYS)
def test_products_take_the_tiles_that_they_are_tested_for(out, M, N, K, way):
    assert ctypes.CDLL(_capi.LIB_PATH).tab_internal_linear8_way(out, M, N, K) == way
    if out == 1:
        assert ctypes.CDLL(_capi.LIB_PATH).tab_internal_linear8_way(2, M, N, K) == way
    assert ctypes.CDLL(_capi.LIB_PATH).tab_internal_linear8_way(out, 32, N, 1000) == 0


def test_sizes_of_packed_operands():
    lib = _capi.load()
    assert [lib.tab_blocks8(k) for k in (-1, 0, 1, 127, 128, 129, 2050)] == [0, 0, 1, 1, 1, 2, 17]
    assert tab_amd.blocks8(2050) == 17
    # up to 32 rows whose packed numbers and scales fit 72 KB are quantized and multiplied in one launch, others packed in the workspace
    # (numbers, then scales)
    for out in (0, 1, 2):
        assert lib.tab_linear8_workspace_bytes(out, 17, 1000, 4096) == 0 < lib.tab_linear8_workspace_bytes(out, 18, 1000, 4096)
        assert lib.tab_linear8_workspace_bytes(out, 32, 1000, 1000) == 0 < lib.tab_linear8_workspace_bytes(out, 33, 1000, 1000)
        assert lib.tab_linear8_packed_workspace_bytes(out, 17, 1000, 4096) == 0
        assert lib.tab_linear8_workspace_bytes(out, 1000, 4096, 300) >= 1000 * (384 + 3)
        assert lib.tab_linear8_workspace_bytes(out, 0, 1, 1) == lib.tab_linear8_packed_workspace_bytes(out, 1, -1, 1) == 0
    assert lib.tab_norm_residual_backward_workspace_bytes(10, 64, 3) == 0       # 10 rows have no 3 gates
    assert lib.tab_norm_residual_backward_workspace_bytes(10, 16385, 0) == 0
    assert lib.tab_norm_residual_backward_workspace_bytes(10, 64, 5) > 0


def test_quantize_refusals():
    q = lambda X=P, dtype=0, M=4, K=256, ld=256, rows=1, format=0, Q=P, S=P, QT=None, ST=None: _capi.load().tab_quantize8(  # noqa: E731
        X, dtype, M, K, ld, rows, format, Q, S, QT, ST, None)
    _refuses(q(dtype=3), "dtype")
    _refuses(q(dtype=-1), "dtype")
    _refuses(q(format=2), "format")
    _refuses(q(rows=64), "1 or 128 rows")
    _refuses(q(M=0), "positive")
    _refuses(q(K=-5), "positive")
    _refuses(q(X=None), "null device pointer: X")
    _refuses(q(X=P + 2), "aligned")
    _refuses(q(X=P + 1, dtype=1), "aligned")
    _refuses(q(ld=255), "row stride")
    _refuses(q(ld=1 << 31), "row stride")
    _refuses(q(Q=None, S=None), "null device pointer")
    _refuses(q(S=None), "null device pointer")
    _refuses(q(Q=P + 8), "16 bytes")
    _refuses(q(QT=P), "null device pointer: QT or ST")
    _refuses(q(QT=P + 4, ST=P), "16 bytes")
    _refuses(q(M=0x7fffffff - 600, K=128 * 64, ld=128 * 64), "one launch", -2)
    _refuses(q(M=0x7fffffff), "one launch", -2)


def test_product_refusals():
    lib = _capi.load()
    p = lambda QX=P, xf=0, SX=P, QW=P, SW=P, rows=128, M=64, N=64, K=256, Y=P, out=0, ws=P, bytes=1 << 30: lib.tab_linear8_packed(  # noqa: E731
        QX, xf, SX, QW, SW, rows, M, N, K, Y, out, ws, bytes, None)
    _refuses(p(xf=2), "format")
    _refuses(p(out=3), "out_dtype")
    _refuses(p(rows=2), "1 or 128 rows")
    for size in ("M", "N", "K"):
        _refuses(p(**{size: 0}), "positive")
    for name in ("QX", "SX", "QW", "SW", "Y"):
        _refuses(p(**{name: None}), "null device pointer")
    _refuses(p(QX=P + 8), "16 bytes")
    _refuses(p(QW=P + 1), "16 bytes")
    _refuses(p(Y=P + 2), "aligned")
    _refuses(p(K=128 * 65536), "too large", -2)
    _refuses(p(N=0x7fffffff), "too large", -2)
    _refuses(p(M=0x7ffffd00, N=0x7ffffd00), "too large", -2)
    need = lib.tab_linear8_packed_workspace_bytes(0, 64, 64, 8192)
    assert need > 0
    _refuses(p(K=8192, ws=None), "workspace", -3)
    _refuses(p(K=8192, bytes=need - 1), "workspace", -3)
    _refuses(p(K=8192, ws=P + 8), "workspace", -3)
    x = lambda X=P, dtype=1, ld=256, QW=P, SW=P, rows=128, M=64, N=64, K=256, Y=P, ws=P, bytes=1 << 30: lib.tab_linear8(  # noqa: E731
        X, dtype, ld, QW, SW, rows, M, N, K, Y, ws, bytes, None)
    _refuses(x(dtype=4), "dtype")
    _refuses(x(X=None), "null device pointer: X")
    _refuses(x(X=P + 1), "aligned")
    _refuses(x(ld=200), "row stride")
    _refuses(x(SW=None), "null device pointer")
    _refuses(x(ws=None), "workspace", -3)
    _refuses(x(M=1, Y=None), "null device pointer: Y")


def test_norm_refusals():
    lib = _capi.load()
    f = ctypes.c_float
    n = lambda X=P, ldx=64, Y=P, ldy=64, gate=P, gd=0, gates=2, post=P, pre=P, alpha=1.0, eps=1e-6, dtype=1, M=4, D=64, R=P, H=P, S=None: (  # noqa: E731
        lib.tab_norm_residual(X, ldx, Y, ldy, gate, gd, gates, post, pre, f(alpha), f(eps), dtype, M, D, R, H, S, None))
    _refuses(n(dtype=3), "dtype")
    _refuses(n(M=0), "positive")
    _refuses(n(D=16385, ldx=16385, ldy=16385), "16384", -2)
    _refuses(n(eps=-1.0), "eps")
    _refuses(n(eps=float("nan")), "eps")
    _refuses(n(gates=3), "multiple of gates")
    _refuses(n(gates=0), "multiple of gates")
    _refuses(n(gd=2), "gate_dtype")
    _refuses(n(X=None), "null device pointer: X")
    _refuses(n(R=None), "null device pointer: R")
    _refuses(n(ldx=63), "row stride of X")
    _refuses(n(ldy=63), "row stride of Y")
    _refuses(n(H=P + 1), "aligned")
    _refuses(n(H=None, S=P), "null device pointer: H or S")
    _refuses(n(H=P + 8, S=P), "16 bytes")
    _refuses(n(post=P + 2), "aligned")
    alone = dict(Y=None, gate=None, post=None, R=None)
    _refuses(n(**{**alone, "gate": P}), "belong to a block")
    _refuses(n(**{**alone, "post": P}), "belong to a block")
    _refuses(n(**alone, alpha=0.5), "belong to a block")
    _refuses(n(**{**alone, "R": P}), "R is X")
    _refuses(n(**alone, H=None), "null device pointer: H")
    b = lambda dR=P, dH=P, R=P, Y=P, gate=P, gd=0, gates=2, post=P, pre=P, dtype=0, M=4, D=64, dX=P, dY=P, dg=P, dpost=P, dpre=P, ws=P, bytes=1 << 30: (  # noqa: E731
        lib.tab_norm_residual_backward(dR, dH, R, Y, gate, gd, gates, post, pre, f(1.0), f(1e-6), dtype, M, D, dX, dY, dg, dpost, dpre, ws, bytes, None))
    _refuses(b(dR=None, dH=None), "dR and dH")
    _refuses(b(R=None), "null device pointer: R")
    _refuses(b(dX=None), "null device pointer: dX")
    _refuses(b(dY=None), "null device pointer: dY")
    _refuses(b(gate=None), "not there")
    _refuses(b(Y=None, gate=None, post=None, dg=None, dpost=None), "not there")
    _refuses(b(dR=P + 2), "aligned")
    _refuses(b(dpre=P + 1), "aligned")
    _refuses(b(ws=None), "workspace", -3)
    _refuses(b(bytes=8), "workspace", -3)


def test_python_refuses_what_is_no_tensor_or_not_on_the_gpu():
    x = torch.zeros(4, 128)
    for call in (tab_amd.Quantize8, tab_amd.Quantize8Transposed, tab_amd.Quantize8Both):
        with pytest.raises(TypeError, match="X must be a torch.Tensor"):
            call([1.0], 4, 128)
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call(x, 4, 128)
        with pytest.raises(RuntimeError, match="dtype"):
            call(x.double(), 4, 128)
        with pytest.raises(RuntimeError, match="block_rows"):
            call(x, 4, 128, 64)
        with pytest.raises(RuntimeError, match="positive"):
            call(x, 0, 128)
    with pytest.raises(TypeError, match="QW must be a torch.Tensor"):
        tab_amd.Linear8(x, None, x, 4, 4, 128)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        tab_amd.Linear8(x, x, x, 4, 4, 128)
    q, s = torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(TypeError, match="out_dtype"):
        tab_amd.Linear8Packed(q, s, q, s, 4, 4, 128, "bf16")
    with pytest.raises(RuntimeError, match="dtype"):
        tab_amd.Linear8Packed(q, s, q, s, 4, 4, 128, torch.float64)
    with pytest.raises(RuntimeError, match="QX must have dtype"):
        tab_amd.Linear8Packed(x, s, q, s, 4, 4, 128)
    with pytest.raises(TypeError, match="w must be a torch.Tensor or None"):
        tab_amd.Norm(x, 1.0, 1e-6, 4, 128)
    with pytest.raises(TypeError, match="Y must be a torch.Tensor"):
        tab_amd.NormResidual(x, None, None, None, None, 1.0, 1e-6, 4, 128)
    with pytest.raises(TypeError, match="gate must be a torch.Tensor or None"):
        tab_amd.NormResidual(x, x, 2, None, None, 1.0, 1e-6, 4, 128)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        tab_amd.NormResidual(x, x, None, None, None, 1.0, 1e-6, 4, 128)
    with pytest.raises(RuntimeError, match="output"):
        tab_amd.NormResidual(x, x, None, None, None, 1.0, 1e-6, 4, 128, 3)
    with pytest.raises(RuntimeError, match="output"):
        tab_amd.Norm(x, None, 1e-6, 4, 128, tab_amd.NORM_NONE)
    with pytest.raises(RuntimeError, match="dR or dH"):
        tab_amd.NormResidualBackward(None, None, x, x, None, None, None, 1.0, 1e-6, 4, 128)
    with pytest.raises(TypeError, match="dH must be a torch.Tensor"):
        tab_amd.NormBackward(None, x, None, 1e-6, 4, 128)


def test_layers_refuse_sizes_that_do_not_agree():
    with pytest.raises(RuntimeError, match="agree in K"):
        tab_nn.linear8(torch.zeros(4, 100), torch.zeros(8, 101))
    with pytest.raises(RuntimeError, match="not be empty"):
        tab_nn.linear8(torch.zeros(0, 100), torch.zeros(8, 100))
    with pytest.raises(RuntimeError, match="format"):
        tab_nn.linear8(torch.zeros(4, 100), torch.zeros(8, 100), grad_format=2)
    with pytest.raises(TypeError):
        tab_nn.linear8(None, torch.zeros(8, 100))
    with pytest.raises(RuntimeError, match="x's shape"):
        tab_nn.norm_residual(torch.zeros(4, 8), torch.zeros(5, 8))
    with pytest.raises(RuntimeError, match="nothing to do"):
        tab_nn.norm_residual(torch.zeros(4, 8), output=tab_amd.NORM_NONE)
    with pytest.raises(ValueError, match="at least one block"):
        tab_nn.ResidualStack([], 8)
    q, s = torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(RuntimeError, match="input must be"):
        tab_nn.Linear8(q, s, 128, 4)(torch.zeros(2, 100))
    with pytest.raises(RuntimeError, match="inference"):
        tab_nn.Linear8(q, s, 128, 4)(torch.zeros(2, 128, requires_grad=True))
