"""The operators together, as a network uses them: a residual stream through ternary and 8-bit layers with the norms between them, its training, side
streams and graphs."""
import pytest
import torch

import layers8_reference as ref
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu


def _rand(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)) * scale


def _stack(D, head=True):
    blocks = [tab_nn.TABLinear.from_float(_rand((D, D), 1), tab_amd.TNN), tab_nn.Linear8.from_float(_rand((D, D), 2, D ** -0.5)),
              tab_nn.TABLinear.from_float(_rand((D, D), 3), tab_amd.BTN)]
    stack = tab_nn.ResidualStack(blocks, D, alpha=0.9, gate_init=0.5, head=tab_nn.Linear8.from_float(_rand((40, D), 4, D ** -0.5)) if head else None)
    return stack.cuda()


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_stack_is_its_operators(rows):
    """Packed hand-over between norms and 8-bit layers, against the same operators one by one on plain tensors."""
    D = 200
    stack, x = _stack(D), _rand((rows, D), 5).cuda()
    with torch.no_grad():
        got = stack(x)
        h, = tab_amd.Norm(x, stack.w_pre[0], ref.EPS, rows, D)
        r = x
        for i, block in enumerate(stack.blocks):
            r, h = tab_amd.NormResidual(r, block(h), stack.gate[i], stack.w_post[i], stack.w_pre[i + 1], 0.9, ref.EPS, rows, D)
        QH, SH = tab_amd.Quantize8(h, rows, D)
        want = tab_amd.Linear8Packed(QH, SH, stack.head.QW, stack.head.SW, rows, 40, D)
    assert got.shape == (rows, 40)
    # the fp32 norm packs what it would have stored; only the order of the product's sums may differ (D products)
    magnitudes = ref.unpack(QH, SH, 1).abs() @ ref.unpack(stack.head.QW, stack.head.SW, 128).abs().t()
    assert ((got - want).cpu().double().abs() <= 2 * D * 2.0 ** -24 * magnitudes).all()


def test_side_stream_and_graph_replays():
    D, rows = 256, 70
    stack = _stack(D)
    xs = [_rand((rows, D), 10 + i).cuda() for i in range(4)]
    with torch.no_grad():
        want = [stack(x) for x in xs]
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [stack(x) for x in xs]
        side.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        static = xs[0].clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            stack(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = stack(static)
        for _ in range(2):
            for x, w in zip(xs, want):
                static.copy_(x)
                graph.replay()
                assert torch.equal(out, w)
                assert torch.equal(stack(x), w)  # the program's own eager work between replays
                torch.cuda.synchronize()


def test_training_step_in_a_graph():
    """Forward and backward of the differentiable operators, captured and replayed on other inputs."""
    M, D, N = 130, 200, 90
    w, gate, w_post, w_pre = (t.cuda().requires_grad_() for t in (_rand((D, D), 20, D ** -0.5), _rand((2, D), 21), torch.ones(D), torch.ones(D)))
    static = [_rand((M, D), 22).cuda(), _rand((M, D), 23, 0.1).cuda()]

    def step():
        h, = tab_nn.norm_residual(static[0], w_pre=w_pre)
        r, h = tab_nn.norm_residual(static[0], tab_nn.linear8(h, w), gate, w_post, w_pre, 0.9)
        return torch.autograd.grad((r, h), (w, gate, w_post, w_pre), (static[1], static[1]))

    inputs = [(_rand((M, D), 30 + i), _rand((M, D), 40 + i, 0.1)) for i in range(3)]
    want = []
    for pair in inputs:
        for s, v in zip(static, pair):
            s.copy_(v)
        want.append([t.clone() for t in step()])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(2):
        for pair, grads in zip(inputs, want):
            for s, v in zip(static, pair):
                s.copy_(v)
            graph.replay()
            for a, b in zip(out, grads):
                assert torch.equal(a, b)
            torch.cuda.synchronize()


def test_training_lowers_a_loss():
    """A small regression: blocks of linear8 between differentiable norms, trained by gradient descent, bf16 activations and fp32 weights."""
    class Block(torch.nn.Module):
        def __init__(self, D, seed):
            super().__init__()
            self.up, self.down = (torch.nn.Parameter(_rand(s, seed + i, s[1] ** -0.5)) for i, s in enumerate([(2 * D, D), (D, 2 * D)]))

        def forward(self, h):
            return tab_nn.linear8(torch.relu(tab_nn.linear8(h, self.up)), self.down, grad_format=tab_amd.E5M2)

    D = 96
    stack = tab_nn.ResidualStack([Block(D, 50), Block(D, 52)], D).cuda()
    x = _rand((256, D), 60).bfloat16().cuda()
    target = torch.roll(x, 1, dims=1).float()
    optimizer = torch.optim.Adam(stack.parameters(), lr=1e-2)
    losses = []
    for _ in range(30):
        loss = (stack(x).float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss))
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in stack.parameters())
    assert losses[-1] < 0.5 * losses[0], losses


def test_linear8_layer_shapes_and_packed_input():
    layer = tab_nn.Linear8.from_float(_rand((30, 300), 70), out_dtype=torch.bfloat16).cuda()
    x = _rand((2, 3, 300), 71).bfloat16().cuda()
    y = layer(x)
    assert y.shape == (2, 3, 30) and y.dtype == torch.bfloat16
    pair = tab_amd.Quantize8(x.view(6, 300), 6, 300)
    assert torch.equal(layer(pair), y.view(6, 30))
    again = tab_nn.Linear8(*[torch.empty_like(t) for t in (layer.QW, layer.SW)], 300, 30, torch.bfloat16)
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again(x), y)


def test_gates_of_a_call():
    stack, x = _stack(64, head=False), _rand((4, 5, 64), 80).cuda()
    with torch.no_grad():
        gates = [_rand((4, 64), 81).cuda(), None, None]
        a = stack(x, gates)
        assert a.shape == x.shape
        for i in range(4):  # a sequence alone takes its own gate
            assert torch.equal(stack(x[i], [gates[0][i:i + 1], None, None]), a[i])
        with pytest.raises(ValueError, match="gates for"):
            stack(x, gates[:1])
