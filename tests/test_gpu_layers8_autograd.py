"""The differentiable 8-bit layers and norms as parts of a user's program: outputs changed in place, weights of other shapes and types, blocks
without a gradient, layers moved and converted."""
import copy

import pytest
import torch
from torch.autograd import forward_ad

import layers8_reference as ref
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu


def _rand(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)) * scale


def _leaves(*tensors):
    return [t.detach().cuda().requires_grad_() for t in tensors]


@pytest.mark.parametrize("shape", [(6, 200), (2, 3, 200)])
def test_linear8_output_changed_in_place(shape):
    """As after torch's own linear: a bias added and an activation applied in place, and the gradients of the same out of place."""
    x, w, b = _rand(shape, 1), _rand((30, 200), 2, 0.1), _rand((30,), 3)
    dy = _rand((*shape[:-1], 30), 4).cuda()
    a = _leaves(x, w, b)
    y = tab_nn.linear8(a[0], a[1])
    y += a[2]
    torch.relu_(y)
    c = _leaves(x, w, b)
    want = torch.relu(tab_nn.linear8(c[0], c[1]) + c[2])
    assert torch.equal(y, want)
    for got, expected in zip(torch.autograd.grad(y, a, dy), torch.autograd.grad(want, c, dy)):
        assert torch.equal(got, expected)


@pytest.mark.parametrize("shape", [(6, 200), (2, 3, 200)])
def test_norm_outputs_changed_in_place(shape):
    """H is nobody's but the caller's.  R is what the backward pass reads: once changed, it says so."""
    x, y, gate, w = _rand(shape, 5), _rand(shape, 6, 9.0), _rand((2, 200), 7), _rand((200,), 8)
    dh = _rand(shape, 9).cuda()
    for block in (True, False):
        def norm(leaves):
            return tab_nn.norm_residual(leaves[0], leaves[1], leaves[2], leaves[3], leaves[3], 0.9) if block else tab_nn.norm_residual(leaves[0], w_pre=leaves[3])
        a, c = _leaves(x, y, gate, w), _leaves(x, y, gate, w)
        h, want = norm(a)[-1], norm(c)[-1] * 3.0
        h *= 3.0
        assert torch.equal(h, want)
        wanted = (0, 1, 2, 3) if block else (0, 3)
        for got, expected in zip(torch.autograd.grad(h, [a[i] for i in wanted], dh), torch.autograd.grad(want, [c[i] for i in wanted], dh)):
            assert torch.equal(got, expected)
    a = _leaves(x, y, gate, w)
    r, h = tab_nn.norm_residual(*a, a[3], 0.9)
    r += 1.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, a, dh)


def test_tangent_of_a_gradient_is_refused():
    x, w = _leaves(_rand((6, 200), 10), _rand((30, 200), 11))
    y = tab_nn.linear8(x, w)
    h, = tab_nn.norm_residual(x)
    with forward_ad.dual_level():
        for out in (y, h):
            dy = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward mode"):
                torch.autograd.grad(out, x, dy, retain_graph=True)
    torch.autograd.grad(y, x, torch.ones_like(y))


def test_weights_of_one_row():
    M, D = 5, 300
    x, y, gate, w_post, w_pre = _rand((M, D), 12), _rand((M, D), 13), _rand((1, D), 14), _rand((D,), 15), _rand((D,), 16)
    dr, dh = _rand((M, D), 17).cuda(), _rand((M, D), 18).cuda()
    a, c = _leaves(x, y, gate, w_post, w_pre), _leaves(x, y, gate, w_post[None], w_pre[None, None])
    want = torch.autograd.grad(tab_nn.norm_residual(*a), a, (dr, dh))
    got = torch.autograd.grad(tab_nn.norm_residual(*c), c, (dr, dh))
    for g, e, leaf in zip(got, want, c):
        assert g.shape == leaf.shape and torch.equal(g.view(e.shape), e)
    w = _rand((1, D), 19).cuda().requires_grad_()
    h, = tab_nn.norm_residual(x.cuda(), w_pre=w)
    h.backward(dh)
    assert w.grad.shape == (1, D)


@pytest.mark.parametrize("nested", [False, True])
def test_stack_does_not_cut_a_gradient_in_silence(nested):
    """A ternary layer has no backward pass: the stack's outputs are as without gradients, and a gradient that would have to pass it is an error."""
    D, x = 64, _rand((10, 64), 20).cuda()
    layer = tab_nn.TABLinear.from_float(_rand((D, D), 21), tab_amd.TNN)
    stack = tab_nn.ResidualStack([torch.nn.Sequential(layer) if nested else layer], D).cuda()
    with torch.no_grad():
        want = stack(x)
    out = stack(x)
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="no gradient"):
        out.sum().backward()
    stack.w_pre[0].requires_grad_(False)  # nothing before the block wants one
    out = stack(x)
    assert torch.equal(out, want)
    out.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in (stack.gate[0], stack.w_post[0], stack.w_pre[1]))
    with pytest.raises(RuntimeError, match="no gradient"):
        stack(x.clone().requires_grad_()).sum().backward()


def test_stack_leaves_a_gradient_that_a_block_stops_on_purpose():
    D, x = 64, _rand((10, 64), 22).cuda()

    class Stop(torch.nn.Module):
        def forward(self, h):
            return h.detach() * 2

    stack = tab_nn.ResidualStack([Stop()], D).cuda()
    stack(x).sum().backward()
    assert torch.isfinite(stack.gate[0].grad).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_weights_of_16_bits(dtype):
    """They are the fp32 weights of the same values; their gradients are rounded to their type."""
    M, D = 7, 300
    x, y, gate = (t.to(dtype) for t in (_rand((M, D), 23), _rand((M, D), 24), _rand((1, D), 25)))
    w_post, w_pre = (_rand((D,), s).to(dtype) for s in (26, 27))
    dr, dh = _rand((M, D), 28).to(dtype).cuda(), _rand((M, D), 29).to(dtype).cuda()
    a, c = _leaves(x, y, gate, w_post, w_pre), _leaves(x, y, gate, w_post.float(), w_pre.float())
    got, want = tab_nn.norm_residual(*a), tab_nn.norm_residual(*c)
    for g, e in zip(got, want):
        assert torch.equal(g, e)
    for g, e, leaf in zip(torch.autograd.grad(got, a, (dr, dh)), torch.autograd.grad(want, c, (dr, dh)), a):
        assert g.dtype == leaf.dtype and torch.equal(g, e.to(dtype))
    with torch.no_grad():
        for output in (tab_amd.NORM_PLAIN, tab_amd.NORM_8BIT):
            for g, e in zip(tab_nn.norm_residual(*a, output=output), tab_nn.norm_residual(*c, output=output)):
                assert torch.equal(g.view(torch.uint8), e.view(torch.uint8))


@pytest.mark.parametrize("ternary_head", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_stack_converted_to_16_bits(dtype, ternary_head):
    D, w = 128, _rand((10, 128), 32, 128 ** -0.5)
    head = tab_nn.TABLinear.from_float(w, tab_amd.TNN) if ternary_head else tab_nn.Linear8.from_float(w)
    blocks = [tab_nn.Linear8.from_float(_rand((D, D), 30, D ** -0.5)), tab_nn.TABLinear.from_float(_rand((D, D), 31), tab_amd.TBN)]
    stack = tab_nn.ResidualStack(blocks, D, alpha=0.5, head=head).cuda()
    x = _rand((9, D), 33).to(dtype).cuda()
    half = copy.deepcopy(stack).to(dtype)
    with torch.no_grad():  # its parameters are ones, the same in every type
        out = half(x)
        assert torch.equal(out, stack(x))
    assert torch.isfinite(out).all() and float(out.abs().max()) > 0


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.double(), lambda m: m.float(), lambda m: m.cpu().cuda(),
                                     lambda m: m.to("cuda", torch.bfloat16), lambda m: m.type(torch.float16), copy.deepcopy],
                         ids=["half", "bfloat16", "double", "float", "cpu_and_back", "to", "type", "copy"])
def test_packed_weight_survives_conversions(convert):
    layer = tab_nn.Linear8.from_float(_rand((30, 300), 34, 1e-6))  # scales that 16 bits do not hold
    x = _rand((5, 300), 35).cuda()
    want, qw, sw = layer(x), layer.QW.view(torch.uint8).clone(), layer.SW.view(torch.uint8).clone()
    layer = convert(layer)
    assert layer.QW.dtype == torch.float8_e4m3fn and layer.SW.dtype == torch.float8_e8m0fnu
    assert torch.equal(layer.QW.view(torch.uint8), qw) and torch.equal(layer.SW.view(torch.uint8), sw)
    assert torch.equal(layer(x), want)


def _norm_gradients(dr, dh, r, y, w_post, w_pre, eps):
    """dX, dY by the formulas in 64 bits, no gate, alpha 1, and the magnitudes they are made from."""
    r, y, a = r.double(), y.double(), dh.double() * w_pre.double()
    p, q = (1 / torch.sqrt((v * v).mean(dim=1, keepdim=True) + eps) for v in (r, y))
    t = p * (a - r * p * (r * p * a).mean(dim=1, keepdim=True))
    mag = p * (a.abs() + (r * p).abs() * (r * p * a).abs().mean(dim=1, keepdim=True))
    if dr is not None:
        t, mag = t + dr.double(), mag + dr.double().abs()
    b, mag_b = t * w_post.double(), mag * w_post.double()
    dy = q * (b - y * q * (y * q * b).mean(dim=1, keepdim=True))
    return t, mag, dy, 2 * q * (mag_b + (y * q).abs() * ((y * q).abs() * mag_b).mean(dim=1, keepdim=True))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,eps", [(1e13, 1e-6), (1e17, 1e-6), (1e-14, 0.0), (1e-16, 0.0)])
@pytest.mark.parametrize("D", [200, 3000])
def test_gradients_of_large_and_small_streams(D, size, eps, dtype):
    """rms^3 of these rows is beyond fp32, their gradients are not.  Bound: that of the ordinary sizes, 2^-18 of the magnitudes and a rounding."""
    M = 5
    r, y = _rand((M, D), 36, size).to(dtype), _rand((M, D), 37, size).to(dtype)
    dr, dh = _rand((M, D), 38, 0.1 / size).to(dtype), _rand((M, D), 39, 0.1).to(dtype)
    w_post, w_pre = _rand((D,), 40).abs() + 0.5, _rand((D,), 41).abs() + 0.5
    for with_dr in (True, False):
        d = dr if with_dr else None
        dx, dy, _, _, _ = tab_amd.NormResidualBackward(None if d is None else d.cuda(), dh.cuda(), r.cuda(), y.cuda(), None, w_post.cuda(), w_pre.cuda(), 1.0, eps, M, D)
        want_x, mag_x, want_y, mag_y = _norm_gradients(d, dh, r, y, w_post, w_pre, eps)
        for got, want, mag in ((dx, want_x, mag_x), (dy, want_y, mag_y)):
            got = got.cpu().double()
            off, bound = (got - want).abs(), 2.0 ** -18 * mag + ref.UNIT[dtype] * (1 + 2.0 ** -8) * want.abs() + ref.TINY[dtype]
            assert (off <= bound).all(), float((off / bound).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_and_weights_that_are_parts_of_wider_tensors(dtype):
    """A gate out of a modulation, one gate expanded over the sequences, columns of a matrix as weights: the values and the gradients of contiguous ones."""
    B, S, D = 3, 4, 200
    x, y, wide, columns = _rand((B, S, D), 50).to(dtype), _rand((B, S, D), 51).to(dtype), _rand((B, 1, 3 * D), 52).to(dtype), _rand((D, 2), 53)
    dr, dh = _rand((B, S, D), 54).to(dtype).cuda(), _rand((B, S, D), 55).to(dtype).cuda()
    a = _leaves(x, y, wide, columns)
    part = a[2].chunk(3, dim=-1)[1]
    assert not part.is_contiguous()
    got = tab_nn.norm_residual(a[0], a[1], part, a[3][:, 0], a[3][:, 1], 0.9)
    c = _leaves(x, y, wide[..., D:2 * D].contiguous(), columns[:, 0].contiguous(), columns[:, 1].contiguous())
    want = tab_nn.norm_residual(*c, 0.9)
    for g, e in zip(got, want):
        assert torch.equal(g, e)
    dx, dy, dwide, dcolumns = torch.autograd.grad(got, a, (dr, dh))
    ex, ey, egate, epost, epre = torch.autograd.grad(want, c, (dr, dh))
    assert torch.equal(dx, ex) and torch.equal(dy, ey) and torch.equal(dcolumns, torch.stack([epost, epre], dim=1))
    assert torch.equal(dwide[..., D:2 * D], egate) and not dwide[..., :D].any() and not dwide[..., 2 * D:].any()
    one = wide[:1, :, :D].cuda()
    with torch.no_grad():
        for g, e in zip(tab_nn.norm_residual(x.cuda(), y.cuda(), one.expand(B, 1, D)), tab_nn.norm_residual(x.cuda(), y.cuda(), one.contiguous())):
            assert torch.equal(g, e)


def test_gate_of_16_bits_in_a_stream_of_32():
    x, y, gate = _rand((6, 300), 56), _rand((6, 300), 57), _rand((2, 300), 58).bfloat16()
    a, c = _leaves(x, y, gate), _leaves(x, y, gate.float())
    got, want = tab_nn.norm_residual(*a), tab_nn.norm_residual(*c)
    dh = _rand((6, 300), 59).cuda()
    for g, e, leaf in zip(torch.autograd.grad(got, a, (dh, dh)), torch.autograd.grad(want, c, (dh, dh)), a):
        assert g.dtype == leaf.dtype and torch.equal(g, e.to(g.dtype))
