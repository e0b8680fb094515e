"""Refusals of the 4-bit layers and of the layers of experts, through the C ABI and from Python: bad arguments are named before anything is launched (no GPU
is touched)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import tab_amd
from tab_amd import _capi
from tab_amd import nn as tab_nn

P = 4096  # an aligned address that is never dereferenced: every call below fails its checks

# (0 fp32 or 1 16-bit output, rows, experts, N, K, half of the tile's rows + columns * 100 + parts of K): every tile, K whole and in parts
WAYS = [(0, 42, 1, 44, 66, 6401), (0, 46, 1, 32, 1600, 6404), (0, 54, 1, 50, 1989, 6416), (0, 5765, 59, 66, 66, 9601), (0, 542, 46, 515, 4787, 9602),
        (0, 846, 20, 1364, 67, 12801), (1, 44, 1, 35, 85, 6401), (1, 1796, 50, 40, 4648, 6402), (1, 49, 1, 45, 1926, 6416), (1, 64, 47, 3550, 74, 9601),
        (1, 564, 57, 98, 5479, 9604), (1, 1230, 37, 695, 69, 12801), (1, 3961, 51, 978, 87, 25601), (1, 10826, 24, 129, 8020, 25604),
        (1, 30000, 20, 1088, 100, 25601), (1, 30000, 20, 1003, 300, 25601), (1, 45000, 1000, 33, 140, 6401), (1, 30000, 129, 300, 300, 12801), (0, 9000, 200, 40, 70, 6401)]
# (output, rows, experts, N, K, half of the tile's rows + columns) of the gradients of the weights
GRAD_WAYS = [(1, 3000, 4, 1100, 1500, 128), (1, 2000, 2, 300, 520, 64), (1, 1059, 46, 67, 131, 96), (1, 1000, 30, 300, 90, 96), (1, 233, 41, 1171, 131, 256), (1, 2000, 41, 1171, 400, 256),
             (0, 3000, 4, 600, 700, 64), (0, 33, 45, 33, 358, 96), (0, 900, 8, 1000, 1400, 128),
             (1, 3000, 130, 67, 131, 64), (0, 900, 1000, 40, 50, 64), (1, 9000, 1024, 33, 20, 64)]


def _refuses(status, message, code=-1):
    assert status == code, status
    assert message in _capi.load().tab_last_error().decode()


@pytest.mark.parametrize("out,R,E,N,K,way", WAYS)
def test_products_take_the_tiles_that_they_are_tested_for(out, R, E, N, K, way):
    way_of = ctypes.CDLL(_capi.LIB_PATH).tab_internal_experts_way
    for bits in (8, 4):
        assert way_of(out, bits, R, E, N, K) == way
        if out == 1:
            assert way_of(2, bits, R, E, N, K) == way


@pytest.mark.parametrize("out,R,E,N,K,way", GRAD_WAYS)
def test_gradients_take_the_tiles_that_they_are_tested_for(out, R, E, N, K, way):
    assert ctypes.CDLL(_capi.LIB_PATH).tab_internal_experts_grad_way(out, R, E, N, K) == way


def test_sizes():
    lib = _capi.load()
    assert [lib.tab_run_blocks(r, e) for r, e in ((0, 1), (1, 0), (1, 1), (1, 9), (128, 1), (129, 1), (129, 2), (256, 300), (1000, 4))] == [0, 0, 1, 1, 1, 2, 2, 256, 11]
    assert tab_amd.run_blocks(1000, 4) == 11
    for out in (0, 1, 2):
        # one launch, its rows cut up among four workgroups (1000 columns) or whole (4096)
        assert lib.tab_linear4_workspace_bytes(out, 68, 1000, 4096) == 0 < lib.tab_linear4_workspace_bytes(out, 69, 1000, 4096)
        assert lib.tab_linear4_workspace_bytes(out, 17, 4096, 4096) == 0 < lib.tab_linear4_workspace_bytes(out, 18, 4096, 4096)
        assert lib.tab_linear4_packed_workspace_bytes(out, 68, 1000, 4096) == lib.tab_linear4_packed_workspace_bytes(out, 17, 4096, 4096) == 0
        assert lib.tab_experts_linear_workspace_bytes(out, 8, 16, 64, 24, 1003, 776) == 0
        assert lib.tab_experts_linear_workspace_bytes(out, 4, 4096, 8192, 8, 512, 300) >= 4096 * (384 + 3)
        assert lib.tab_experts_linear_workspace_bytes(out, 8, 0, 1, 1, 1, 1) == lib.tab_experts_linear_packed_workspace_bytes(out, 1, 8, 1, -1, 1, 1) == 0
    assert lib.tab_route_workspace_bytes(128, 64, 4) == 0 < lib.tab_route_workspace_bytes(129, 64, 4)
    assert lib.tab_route_workspace_bytes(129, 1025, 4) == lib.tab_route_workspace_bytes(0, 1, 1) == 0


def test_quantize4_refusals():
    lib = _capi.load()
    q = lambda W=P, dtype=0, E=1, M=4, K=256, ld=256, Q=P, S=P: lib.tab_quantize4(W, dtype, E, M, K, ld, Q, S, None)  # noqa: E731
    _refuses(q(dtype=3), "dtype")
    _refuses(q(E=0), "positive")
    _refuses(q(M=0), "positive")
    _refuses(q(K=-5), "positive")
    _refuses(q(W=None), "null device pointer: W")
    _refuses(q(W=P + 2), "aligned")
    _refuses(q(ld=255), "row stride")
    _refuses(q(Q=None), "null device pointer")
    _refuses(q(S=None), "null device pointer")
    _refuses(q(Q=P + 8), "16 bytes")
    _refuses(q(E=1 << 16, M=1 << 16), "one launch", -2)
    _refuses(q(M=0x7fffffff - 600, K=128 * 64, ld=128 * 64), "one launch", -2)
    e = lambda W=P, dtype=0, E=2, N=4, K=256, ld=256, Q=P, S=P, QT=None, ST=None: lib.tab_quantize8_experts(W, dtype, E, N, K, ld, Q, S, QT, ST, None)  # noqa: E731
    _refuses(e(dtype=-1), "dtype")
    _refuses(e(E=0), "positive")
    _refuses(e(E=1025), "experts")
    _refuses(e(W=None), "null device pointer: W")
    _refuses(e(ld=10), "row stride")
    _refuses(e(Q=None, S=None), "null device pointer")
    _refuses(e(QT=P), "null device pointer: QT or ST")
    _refuses(e(QT=P + 4, ST=P), "16 bytes")
    _refuses(e(E=1024, N=1 << 22), "one launch", -2)


def test_linear4_refusals():
    lib = _capi.load()
    p = lambda QX=P, SX=P, QW=P, SW=P, M=64, N=64, K=256, Y=P, out=0, ws=P, bytes=1 << 30: lib.tab_linear4_packed(QX, SX, QW, SW, M, N, K, Y, out, ws, bytes, None)  # noqa: E731
    _refuses(p(out=3), "out_dtype")
    _refuses(p(M=0), "positive")
    _refuses(p(QX=None), "null device pointer: QX or SX")
    _refuses(p(SW=None), "null device pointer: QW or SW")
    _refuses(p(QW=P + 8), "16 bytes")
    _refuses(p(SW=P + 2), "4 bytes")
    _refuses(p(Y=None), "null device pointer: Y")
    _refuses(p(M=0x7fffffff), "32-bit offsets", -2)
    _refuses(p(M=400, K=8192, ws=None), "workspace", -3)
    x = lambda X=P, dtype=0, ld=256, QW=P, SW=P, M=64, N=64, K=256, Y=P, ws=P, bytes=1 << 30: lib.tab_linear4(X, dtype, ld, QW, SW, M, N, K, Y, ws, bytes, None)  # noqa: E731
    _refuses(x(dtype=3), "dtype")
    _refuses(x(K=0), "positive")
    _refuses(x(X=None), "null device pointer: X")
    _refuses(x(ld=255), "row stride")
    _refuses(x(SW=P + 1), "4 bytes")
    _refuses(x(M=1000, bytes=16), "workspace", -3)
    _refuses(x(M=1000, ws=P + 8), "workspace", -3)


def test_route_refusals():
    lib = _capi.load()
    r = lambda L=P, dtype=0, ld=64, M=200, E=64, k=4, w=P, e=P, rows=P, places=P, offsets=P, ws=P, bytes=1 << 30: lib.tab_route(  # noqa: E731
        L, dtype, ld, M, E, k, 1, w, e, rows, places, offsets, ws, bytes, None)
    _refuses(r(dtype=3), "dtype")
    _refuses(r(M=0), "positive")
    _refuses(r(E=0), "experts")
    _refuses(r(E=1025, ld=1025), "experts")
    _refuses(r(k=0), "k must be")
    _refuses(r(k=65), "k must be")
    _refuses(r(k=33), "k must be")
    _refuses(r(M=1 << 30), "too many rows", -2)
    _refuses(r(L=None), "null device pointer: logits")
    _refuses(r(L=P + 1), "aligned")
    _refuses(r(ld=63), "row stride")
    for name in ("w", "e", "rows", "places", "offsets"):
        _refuses(r(**{name: None}), "null device pointer")
        _refuses(r(**{name: P + 2}), "aligned")
    _refuses(r(ws=None), "workspace", -3)
    _refuses(r(bytes=8), "workspace", -3)
    b = lambda g=P, w=P, e=P, L=P, dtype=0, ld=64, M=4, E=64, k=4, d=P: lib.tab_route_backward(g, w, e, L, dtype, ld, M, E, k, 1, d, None)  # noqa: E731
    for name in ("g", "w", "e", "L", "d"):
        _refuses(b(**{name: None}), "null device pointer")
    _refuses(b(k=65), "k must be")
    _refuses(b(dtype=9), "dtype")


def test_experts_refusals():
    lib = _capi.load()
    x = lambda X=P, dtype=1, ld=256, M=64, rows=P, offsets=P, QW=P, SW=P, bits=8, block=128, R=2048, E=8, N=64, K=256, Y=P, ws=P, bytes=1 << 30: lib.tab_experts_linear(  # noqa: E731
        X, dtype, ld, M, rows, offsets, QW, SW, bits, block, R, E, N, K, Y, ws, bytes, None)
    _refuses(x(dtype=3), "dtype")
    _refuses(x(bits=2), "4 or 8 bits")
    _refuses(x(block=64), "1 or 128 rows")
    _refuses(x(M=0), "positive")
    _refuses(x(R=0), "positive")
    _refuses(x(E=0), "experts")
    _refuses(x(E=1025), "experts")
    _refuses(x(N=0), "positive")
    _refuses(x(rows=P + 1), "aligned")
    _refuses(x(offsets=None), "null device pointer: offsets")
    _refuses(x(rows=None), "without rows")
    _refuses(x(X=None), "null device pointer: X")
    _refuses(x(ld=255), "row stride")
    _refuses(x(QW=None), "null device pointer: QW or SW")
    _refuses(x(bits=4, SW=P + 2), "4 bytes")
    _refuses(x(Y=None), "null device pointer: Y")
    _refuses(x(ws=None), "workspace", -3)
    _refuses(x(M=1 << 24), "3.5 GiB", -2)
    _refuses(x(R=0x7fffffff - 512, N=4096), "one launch", -2)
    p = lambda QX=P, xf=0, SX=P, M=64, rows=P, offsets=P, QW=P, SW=P, bits=8, block=128, R=2048, E=8, N=64, K=256, Y=P, out=0, ws=P, bytes=1 << 30: lib.tab_experts_linear_packed(  # noqa: E731
        QX, xf, SX, M, rows, offsets, QW, SW, bits, block, R, E, N, K, Y, out, 1, ws, bytes, None)
    _refuses(p(xf=2), "format")
    _refuses(p(xf=1, bits=4), "E4M3")
    _refuses(p(out=-1), "out_dtype")
    _refuses(p(QX=None), "null device pointer: QX or SX")
    _refuses(p(QX=P + 8), "16 bytes")
    _refuses(p(rows=None, M=5), "without rows")


def test_gradient_refusals():
    lib = _capi.load()
    q = lambda X=P, dtype=0, ld=64, M=64, rows=P, offsets=P, R=128, E=2, K=64, f=0, Q=None, S=None, QT=P, ST=P: lib.tab_quantize8_by_expert(  # noqa: E731
        X, dtype, ld, M, rows, offsets, R, E, K, f, Q, S, QT, ST, None)
    _refuses(q(dtype=3), "dtype")
    _refuses(q(f=2), "format")
    _refuses(q(rows=None), "without rows")
    _refuses(q(offsets=None), "offsets")
    _refuses(q(K=0), "positive")
    _refuses(q(X=None), "null device pointer: X")
    _refuses(q(QT=None), "null device pointer: QT or ST")
    _refuses(q(Q=P), "null device pointer: Q or S")
    _refuses(q(ld=3), "row stride")
    g = lambda QD=P, f=0, SD=P, QX=P, SX=P, offsets=P, R=128, E=2, N=64, K=64, W=P, out=0: lib.tab_experts_grad_weight(QD, f, SD, QX, SX, offsets, R, E, N, K, W, out, None)  # noqa: E731
    _refuses(g(f=3), "format")
    _refuses(g(out=3), "out_dtype")
    _refuses(g(offsets=None), "offsets")
    _refuses(g(N=0), "positive")
    _refuses(g(QD=None), "null device pointer: QD or SD")
    _refuses(g(SX=None), "null device pointer: QX or SX")
    _refuses(g(W=None), "null device pointer: dW")
    _refuses(g(R=128 * 65536), "32-bit offsets", -2)


def test_combine_refusals():
    lib = _capi.load()
    c = lambda Y=P, dtype=0, places=P, w=P, M=4, k=2, R=8, D=64, out=P, od=0: lib.tab_combine(Y, dtype, places, w, M, k, R, D, out, od, None)  # noqa: E731
    _refuses(c(dtype=3), "dtype")
    _refuses(c(dtype=1, od=2), "out_dtype must be dtype")
    _refuses(c(M=0), "positive")
    _refuses(c(D=0), "positive")
    _refuses(c(places=None), "null device pointer: places")
    _refuses(c(w=P + 2), "aligned")
    _refuses(c(Y=None), "null device pointer: Y")
    _refuses(c(out=None), "null device pointer: out")
    _refuses(c(M=1 << 20, D=1 << 16), "one launch", -2)
    b = lambda g=P, Y=P, dtype=0, places=P, w=P, used=P, M=4, k=2, R=8, D=64, dy=P, dw=P: lib.tab_combine_backward(g, Y, dtype, places, w, used, M, k, R, D, dy, dw, None)  # noqa: E731
    _refuses(b(g=None), "null device pointer: dout")
    _refuses(b(dy=None, dw=None), "dY and dweights")
    _refuses(b(Y=None), "null device pointer: Y")
    _refuses(b(used=P + 1), "aligned")
    _refuses(b(dw=P + 1), "aligned")


def test_python_refuses_what_is_no_tensor_of_the_right_kind():
    x, q4, q8 = torch.zeros(4, 128), torch.zeros(8, 64, dtype=torch.uint8).view(torch.float4_e2m1fn_x2), torch.zeros(8, 128).to(torch.float8_e4m3fn)
    s = torch.zeros(1, 8, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    i = torch.zeros(5, dtype=torch.int32)
    for call in (lambda: tab_amd.Quantize4([1.0], 1, 1), lambda: tab_amd.Linear4(x, None, s, 4, 8, 128), lambda: tab_amd.Linear4Packed(x, s, q4, s, 4, 8, 128, "fp32"),
                 lambda: tab_amd.Route("logits", 4, 8, 2), lambda: tab_amd.ExpertsLinear(x, 3, i, q8, s, 4, 4, 1, 8, 128), lambda: tab_amd.QuantizeExperts(None, 1, 1, 1),
                 lambda: tab_amd.ExpertsLinearPacked(x, s, None, i, q8, s, 4, 4, 1, 8, 128, 1), lambda: tab_amd.Quantize8ByExpert(x, i, None, 4, 4, 1, 128),
                 lambda: tab_amd.ExpertsGradWeight(x, s, x, None, i, 4, 1, 8, 128), lambda: tab_amd.Combine(x, None, None, 4, 1, 4, 128),
                 lambda: tab_amd.CombineBackward(x, x, i, 3, None, 4, 1, 4, 128)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: tab_amd.Quantize4(x, 4, 128), lambda: tab_amd.Linear4(x, q4, s, 4, 8, 128), lambda: tab_amd.Route(x, 4, 128, 2),
                 lambda: tab_amd.ExpertsLinear(x, None, i, q8, s, 4, 4, 4, 8, 128), lambda: tab_amd.Combine(x, i[:4].view(4, 1), None, 4, 1, 4, 128)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    for call, message in ((lambda: tab_amd.Quantize4(x.double(), 4, 128), "dtype"), (lambda: tab_amd.Route(x, 4, 128, 129), "k must be"), (lambda: tab_amd.Route(x, 0, 128, 1), "positive"),
                          (lambda: tab_amd.QuantizeExperts(x, 1, 4, 128, 2), "4 or 8"), (lambda: tab_amd.QuantizeExperts(x, 1, 4, 128, 4, True), "transposed"),
                          (lambda: tab_amd.ExpertsLinear(x, None, i, q8, s, 4, 5, 4, 8, 128), "without rows")):
        with pytest.raises(RuntimeError, match=message):
            call()


def test_layers_refuse():
    i = torch.zeros(8, dtype=torch.int32)
    routing = tab_nn.Routing(torch.zeros(4, 2), i.view(4, 2), i, i.view(4, 2), torch.zeros(4, dtype=torch.int32))
    x, w = torch.zeros(4, 128), torch.zeros(3, 8, 128)
    for a, b, gather, message in ((x, w[:, :, :5], True, "agree in K"), (x, w[0], True, "agree in K"), (x[:3], w, True, "4 tokens"), (x, w, False, "8 sorted rows"),
                                  (x, w[:2], True, "one of 3 experts"), (x.double(), w, True, "dtype"), (x, w.double(), True, "dtype"), (x[:0], w, True, "empty")):
        with pytest.raises(RuntimeError, match=message):
            tab_nn.experts_linear8(a, b, routing, gather)
    with pytest.raises(RuntimeError, match="format"):
        tab_nn.experts_linear8(x, w, routing, grad_format=2)
    for y, wt, message in ((x, routing.weights, "rows of y"), (torch.zeros(8, 3, 2), routing.weights, "must be"), (torch.zeros(8, 3), torch.zeros(4, 1), "weights must be")):
        with pytest.raises(RuntimeError, match=message):
            tab_nn.combine(y, routing._replace(weights=wt))
    with pytest.raises(RuntimeError, match="empty"):
        tab_nn.route(x[:0], 2)
    with pytest.raises(RuntimeError, match="k must be"):
        tab_nn.route(x, 129)


def test_tangents_are_refused_and_not_dropped():
    def dual(*shape):
        return forward_ad.make_dual(torch.ones(shape), torch.ones(shape))

    i = torch.zeros(8, dtype=torch.int32)
    routing = tab_nn.Routing(torch.zeros(4, 2), i.view(4, 2), i, i.view(4, 2), torch.zeros(4, dtype=torch.int32))
    q, s = torch.zeros(8, 64, dtype=torch.uint8).view(torch.float4_e2m1fn_x2), torch.zeros(1, 8, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with forward_ad.dual_level():
        for call in (lambda: tab_nn.route(dual(4, 3), 2), lambda: tab_nn.experts_linear8(dual(4, 128), torch.zeros(3, 8, 128), routing),
                     lambda: tab_nn.experts_linear8(torch.zeros(4, 128), dual(3, 8, 128), routing), lambda: tab_nn.combine(dual(8, 5), routing),
                     lambda: tab_nn.combine(torch.zeros(8, 5), routing._replace(weights=dual(4, 2))), lambda: tab_nn.Linear4(q, s, 128, 8)(dual(4, 128)),
                     lambda: tab_nn.PackedExperts(q, s, 3, 128, 8)(dual(4, 128), routing)):
            with pytest.raises(RuntimeError, match="forward mode"):
                call()


@pytest.mark.parametrize("N", [1 << 29, (1 << 29) + 16, 0x7fffffff - 512])
@pytest.mark.parametrize("M,K", [(1, 128), (1, 300), (700, 128)])
def test_weights_of_4_bits_whose_scales_32_bits_do_not_reach(M, K, N):
    """Four scale bytes a row: from 2^29 rows on the offset of a row's, and of the next block of K's, would come round to below zero."""
    lib, E, R, W = _capi.load(), 1, 1, 1 << 40
    for dtype in (0, 1, 2):
        _refuses(lib.tab_linear4(P, dtype, 1 << 10, P, P, M, N, K, P, P, W, None), "", -2)
        _refuses(lib.tab_linear4_packed(P, P, P, P, M, N, K, P, dtype, P, W, None), "", -2)
        _refuses(lib.tab_experts_linear(P, dtype, 1 << 10, M, P, P, P, P, 4, 1, R, E, N, K, P, P, W, None), "", -2)
        _refuses(lib.tab_experts_linear_packed(P, 0, P, M, P, P, P, P, 4, 1, R, E, N, K, P, dtype, 1, P, W, None), "", -2)
    if M == 1 and K == 128:
        _refuses(lib.tab_linear4(P, 1, 1 << 10, P, P, M, N, K, P, P, W, None), "weights of 4 bits", -2)


def test_sorted_rows_have_no_bound_that_listed_ones_have():
    """(Refused for their workspace, which is checked behind the sizes.)"""
    lib, R, N, K = _capi.load(), 1 << 24, 64, 256
    for bits in (8, 4):
        for rows, message, code in ((P, "3.5 GiB", -2), (None, "workspace", -3)):
            _refuses(lib.tab_experts_linear(P, 1, K, R, rows, P, P, P, bits, 128, R, 8, N, K, P, None, 0, None), message, code)
    _refuses(lib.tab_experts_linear_packed(P, 0, P, R, P, P, P, P, 8, 128, R, 8, N, K, None, 1, 0, None, 0, None), "3.5 GiB", -2)
    _refuses(lib.tab_experts_linear_packed(P, 0, P, R, None, P, P, P, 8, 128, R, 8, N, K, None, 1, 0, None, 0, None), "null device pointer: Y")


@pytest.mark.parametrize("dtype,w_dtype", [(0, 0), (1, 1), (2, 0), (1, 0)])
@pytest.mark.parametrize("M,k,E,N,K", [(100, 2, 4, 64, 64), (128 * 65536, 1, 1, 8, 8), (128 * 65535, 1, 1, 8, 8), (128 * 65535, 1, 2, 8, 8), (1 << 24, 1, 1, 8, 8), ((1 << 24) - 1, 1, 1, 8, 8),
                                       (1 << 23, 2, 3, 8, 8), (1 << 23, 0, 3, 8, 8), (1 << 20, 1, 3, 65536, 8), (1 << 20, 0, 3, 8, 65536), (1 << 14, 2, 1024, 1 << 15, 1 << 16),
                                       (1 << 22, 4, 7, 20000, 16), (500, 2, 3, 128 * 65536, 8), (1000, 8, 1024, 8192, 8192)])
def test_training_is_refused_where_its_gradients_would_be(M, k, E, N, K, dtype, w_dtype):
    """The check agrees with the calls that the backward pass makes (which refuse a null pointer once the sizes are accepted)."""
    lib, R = _capi.load(), M * max(k, 1)

    def taken(status):
        if status == -2:
            return False
        assert status == -1 and "null device pointer" in lib.tab_last_error().decode()
        return True

    by_expert = taken(lib.tab_quantize8_by_expert(None, dtype, N, R, None, P, R, E, N, 0, None, None, P, P, None))
    of_w = by_expert and taken(lib.tab_experts_grad_weight(None, 0, P, P, P, P, R, E, N, K, P, w_dtype, None))
    product = taken(lib.tab_experts_linear_packed(None, 0, P, R, None, P, P, P, 8, 128, R, E, K, N, P, 0 if k else dtype, dtype == 0, P, 1 << 60, None))
    product = product and (k == 0 or taken(lib.tab_combine(P, 0, None, None, M, k, R, K, P, dtype, None)))
    rows = taken(lib.tab_quantize8(None, dtype, R, N, N, 1, 0, P, P, None, None, None))
    for want_x, want_w, want in ((0, 0, True), (0, 1, of_w), (1, 0, rows and product), (1, 1, of_w and product)):
        status = lib.tab_experts_check_gradients(dtype, w_dtype, M, k, R, E, N, K, want_x, want_w)
        assert status == (0 if want else -2), (want_x, want_w)


def test_refusals_of_derivatives_name_no_other_layer():
    """A router or a 4-bit layer that refuses a tangent does not speak of 8-bit layers or norms."""
    i = torch.zeros(8, dtype=torch.int32)
    routing = tab_nn.Routing(torch.zeros(4, 2), i.view(4, 2), i, i.view(4, 2), torch.zeros(4, dtype=torch.int32))
    with forward_ad.dual_level():
        dual = lambda *shape: forward_ad.make_dual(torch.ones(shape), torch.ones(shape))  # noqa: E731
        for call in (lambda: tab_nn.route(dual(4, 3), 2), lambda: tab_nn.combine(dual(8, 5), routing)):
            with pytest.raises(RuntimeError) as error:
                call()
            assert "forward mode" in str(error.value) and "8-bit" not in str(error.value) and "norms" not in str(error.value)
