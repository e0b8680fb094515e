"""The operators together, as a network uses them: routed experts trained in 8 bits and served in 8 and 4, in a residual stream, on side streams and in
graphs."""
import pytest
import torch

import experts_reference as ref
import layers8_reference as ref8
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu


def _rand(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)) * scale


class Router(torch.nn.Module):
    """Plain logits."""

    def __init__(self, E, D, seed):
        super().__init__()
        self.weight = torch.nn.Parameter(_rand((E, D), seed, D ** -0.5))

    def forward(self, x):
        return (x.float() @ self.weight.float().t().contiguous())


def _mixture(D, H, E, k, seed=1, dtype=torch.float32):
    up, down = _rand((E, H, D), seed, D ** -0.5).to(dtype), _rand((E, D, H), seed + 1, H ** -0.5).to(dtype)
    return tab_nn.MixtureOfExperts(Router(E, D, seed + 2), tab_nn.Experts8(up), tab_nn.Experts8(down), k, activation=torch.nn.SiLU()).cuda()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("rows", [1, 16, 300])
def test_mixture_is_its_operators(rows, bits):
    D, H, E, k = 200, 140, 12, 3
    block, x = _mixture(D, H, E, k).packed(bits), _rand((rows, D), 5).cuda()
    with torch.no_grad():
        got = block(x)
        weights, experts, order, places, offsets = tab_amd.Route(block.router(x), rows, E, k)
        R = rows * k
        y = tab_amd.ExpertsLinear(x, order, offsets, block.up.QW, block.up.SW, rows, R, E, H, D)
        z = tab_amd.ExpertsLinear(torch.nn.functional.silu(y), None, offsets, block.down.QW, block.down.SW, R, R, E, D, H)
        assert torch.equal(got, tab_amd.Combine(z, places, weights, rows, k, R, D))
        # and one token alone gives what it gives in the batch, but for the order of the sums: the packed numbers are its own
        alone = block(x[:1])
        want, mag = ref.by_expert(ref8.value(*ref8.quantize(torch.nn.functional.silu(y).cpu(), 1, 0), 1), _values(block.down, bits), None, offsets.cpu(), D)
        token = [(int(p), float(w)) for p, w in zip(places[0], weights[0])]
        want, mag = (sum(w * v[p] for p, w in token) for v in (want, mag))
        if rows == 1:
            ref.check(alone[0], want, mag, H + k, False, "one token")
    assert got.shape == (rows, D) and torch.isfinite(got).all()


def _values(layer, bits):
    return [(ref.unpack4(q, s) if bits == 4 else ref8.unpack(q, s, 128)) for q, s in zip(layer.QW, layer.SW)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step(dtype):
    """Outputs and all gradients of a mixture, against the same network on the CPU in 64 bits with the rounded operands put in their place."""
    D, H, E, k, rows = 96, 72, 6, 2, 150
    block = _mixture(D, H, E, k, 7, dtype)
    x = _rand((3, rows // 3, D), 11).to(dtype)
    xd = x.cuda().requires_grad_()
    out = block(xd)
    assert out.shape == x.shape and out.dtype == dtype
    dout = _rand(out.shape, 12).to(dtype)
    leaves = [xd, block.router.weight, block.up.weight, block.down.weight]
    got = torch.autograd.grad(out, leaves, dout.cuda())
    for g, leaf in zip(got, leaves):
        assert g.shape == leaf.shape and g.dtype == leaf.dtype and torch.isfinite(g).all()
    # the same in fp64 without any rounding: the 8-bit operands are off by at most 2^-4 of a value each, by 2^-4 / sqrt(3) in the root of the mean
    # square, so a product of two by 2^-4 * sqrt(2 / 3) of its size; through two layers and an activation of slope at most 1.1, with the gradients'
    # third operand, below 4 times that in the root of the mean square
    x64, r64, u64, d64 = (t.detach().cpu().double().requires_grad_() for t in leaves)
    tokens = x64.reshape(-1, D)
    logits = tokens @ r64.t()
    routing = tab_nn.route(block.router(xd.detach().reshape(-1, D)), k)
    experts = routing.experts.cpu().long()
    w = torch.softmax(torch.gather(logits, 1, experts), dim=1)
    want = 0
    for j in range(k):
        h = torch.nn.functional.silu((u64[experts[:, j]] @ tokens[..., None]).squeeze(-1))
        want = want + w[:, j, None] * (d64[experts[:, j]] @ h[..., None]).squeeze(-1)
    expected = torch.autograd.grad(want.reshape(x.shape), (x64, r64, u64, d64), dout.double())
    for g, e in zip((out, *got), (want.reshape(x.shape), *expected)):
        e = e.detach()
        off = (g.detach().cpu().double() - e).square().mean().sqrt() / e.square().mean().sqrt()
        assert off < 4 * 2.0 ** -4 * (2 / 3) ** 0.5, float(off)


def test_stack_with_experts_and_weights_of_4_bits():
    D = 128
    blocks = [tab_nn.Linear4.from_float(_rand((D, D), 21, D ** -0.5)), _mixture(D, 64, 5, 2).packed(4), tab_nn.TABLinear.from_float(_rand((D, D), 22), tab_amd.TNN)]
    stack = tab_nn.ResidualStack(blocks, D, alpha=0.9, head=tab_nn.Linear4.from_float(_rand((40, D), 23, D ** -0.5))).cuda()
    for rows in (1, 20, 300):
        x = _rand((rows, D), 24).cuda()
        with torch.no_grad():
            got = stack(x)
            h, = tab_amd.Norm(x, stack.w_pre[0], ref8.EPS, rows, D)
            r = x
            for i, block in enumerate(stack.blocks):
                r, h = tab_amd.NormResidual(r, block(h), stack.gate[i], stack.w_post[i], stack.w_pre[i + 1], 0.9, ref8.EPS, rows, D)
            QH, SH = tab_amd.Quantize8(h, rows, D)
            want = tab_amd.Linear4Packed(QH, SH, stack.head.QW, stack.head.SW, rows, 40, D)
        assert got.shape == (rows, 40)
        # the norms pack what they would have stored; only the order of the products' sums may differ, which the ternary layer's thresholds may turn into another
        # sign here and there: nearly all outputs are equal
        mag = ref8.unpack(QH, SH, 1).abs() @ ref.unpack4(stack.head.QW, stack.head.SW).abs().t()
        close = (got - want).cpu().double().abs() <= 2 * D * 2.0 ** -24 * mag
        assert close.all(dim=1).float().mean() > 0.9


def test_stack_trains_through_experts():
    D = 64
    stack = tab_nn.ResidualStack([_mixture(D, 64, 4, 2, 31), _mixture(D, 32, 3, 1, 35)], D, alpha=0.9).cuda()
    x = _rand((50, D), 36).cuda().requires_grad_()
    stack(x).square().sum().backward()
    for p in (x, *stack.parameters()):
        assert p.grad is not None and torch.isfinite(p.grad).all()
    assert all(b.up.weight.grad.any() and b.down.weight.grad.any() and b.router.weight.grad.any() for b in stack.blocks[:1])


@pytest.mark.parametrize("rows", [4, 200])
@pytest.mark.parametrize("bits", [8, 4])
def test_side_stream_and_graph_replays(bits, rows):
    """Tokens, and with them all sizes on the device, change between the replays."""
    D = 192
    block = _mixture(D, 130, 9, 2).packed(bits)
    xs = [_rand((rows, D), 40 + i).cuda() for i in range(4)]
    with torch.no_grad():
        want = [block(x) for x in xs]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [block(x) for x in xs]
        side.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        static = xs[0].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(static)
        for i in (1, 3, 0, 2):
            static.copy_(xs[i])
            other = block(xs[(i + 1) % 4])  # eager work between the replays
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[i]) and torch.equal(other, want[(i + 1) % 4])


def test_two_graphs_and_training_replays():
    """Forward and backward captured, each replay against the eager result."""
    D, H, E, k, rows = 96, 80, 5, 2, 140
    block = _mixture(D, H, E, k, 50, torch.bfloat16)
    params = list(block.parameters())
    xs = [_rand((rows, D), 60 + i).to(torch.bfloat16).cuda() for i in range(3)]
    dout = _rand((rows, D), 70).to(torch.bfloat16).cuda()

    def step(x):
        x = x.detach().requires_grad_()
        return torch.autograd.grad(block(x), [x, *params], dout)

    want = [[g.clone() for g in step(x)] for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xs[0])
    torch.cuda.current_stream().wait_stream(side)
    statics, graphs, outs = [], [], []
    for _ in range(2):
        statics.append(xs[0].clone())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(statics[-1]))
    for i, j in ((1, 2), (0, 1), (2, 0)):
        statics[0].copy_(xs[i])
        statics[1].copy_(xs[j])
        graphs[0].replay()
        graphs[1].replay()
        eager = step(xs[i])
        torch.cuda.synchronize()
        for a, b, c in zip(outs[0], want[i], eager):
            assert torch.equal(a, b) and torch.equal(c, b)
        for a, b in zip(outs[1], want[j]):
            assert torch.equal(a, b)


def test_packed_experts_keep_their_weights():
    layer = tab_nn.PackedExperts.from_float(_rand((3, 30, 300), 34, 1e-6), 4)
    routing = tab_nn.route(_rand((7, 3), 35).cuda(), 2)
    x = _rand((7, 300), 36).cuda()
    want, qw = layer(x, routing), layer.QW.view(torch.uint8).clone()
    layer = layer.half().cpu().cuda()
    assert layer.QW.dtype == torch.float4_e2m1fn_x2 and torch.equal(layer.QW.view(torch.uint8), qw) and torch.equal(layer(x, routing), want)
    with pytest.raises(RuntimeError, match="inference"):
        layer(x.requires_grad_(), routing)


def test_calls_on_two_streams_at_once():
    """Nothing is shared between calls: two streams run the same layers on inputs of their own, neither waiting for the other."""
    D = 256
    block, layer = _mixture(D, 200, 6, 2).packed(8), tab_nn.Linear4.from_float(_rand((D, D), 1))
    xs = [_rand((rows, D), 90 + rows).cuda() for rows in (5, 300, 300, 70)]
    with torch.no_grad():
        want = [layer(block(x)) for x in xs]
        streams = [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        got = [[], []]
        for turn in range(6):
            for i, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    got[i].append(layer(block(xs[(turn + i) % 4])))
        torch.cuda.synchronize()
    for i in range(2):
        for turn, y in enumerate(got[i]):
            assert torch.equal(y, want[(turn + i) % 4])
