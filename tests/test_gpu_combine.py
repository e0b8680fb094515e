"""The way back from rows to tokens against its definition in 64 bits."""
import pytest
import torch

import experts_reference as ref
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
types = pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
SIZES = [(1, 1, 1), (3, 2, 7), (5, 4, 8), (40, 3, 130), (7, 9, 1531), (300, 5, 64), (20, 2, 5000), (4100, 2, 30), (9, 8, 517)]


def _rand(shape, seed, scale=1.0):
    return torch.randn(shape, generator=torch.Generator("cpu").manual_seed(seed)) * scale


def _problem(M, k, D, dtype):
    E = 2 * k
    plan = ref.plan(M, E, k, M + D, closed=M // 5) if M < 1000 else None
    if plan is None:  # (the reference's router goes token by token)
        logits = _rand((M, E), M)
        logits[::7] = float("-inf")
        plan = [t.cpu() for t in tab_amd.Route(logits.cuda(), M, E, k)]
    y = _rand((M * k, D), 1).to(dtype)
    y[int(plan[4][-1]):] = float("nan")  # rows of no expert are read by nobody
    return plan, y


@types
@pytest.mark.parametrize("M,k,D", SIZES)
def test_combine_and_gradients(M, k, D, dtype):
    plan, y = _problem(M, k, D, dtype)
    weights, _, _, places, offsets = plan
    R, n = M * k, int(offsets[-1])
    yd, wd = y.cuda().requires_grad_(), weights.cuda().requires_grad_()
    out = tab_nn.combine(yd, tab_nn.Routing(wd, *(t.cuda() for t in plan[1:])))
    dout = _rand((M, D), 2, 1e-2).to(dtype)
    dy, dw = torch.autograd.grad(out, (yd, wd), dout.cuda())
    y64, at, chosen = y.double(), places.clamp(min=0).long(), (places >= 0)
    y64[n:] = 0
    terms = torch.where(chosen, weights.double(), 0.0)[..., None] * y64[at]
    ref.check(out, terms.sum(dim=1), terms.abs().sum(dim=1), k, False, "out")
    assert out.dtype == dtype and torch.equal(out, tab_amd.Combine(y.cuda(), places.cuda(), weights.cuda(), M, k, R, D))
    g = dout.double()
    want = torch.zeros((R, D), dtype=torch.float64)
    want[places[chosen].long()] = (weights.double()[..., None] * g[:, None])[chosen]
    ref.check(dy, want, want.abs(), 1, False, "dy")  # one product, rounded to fp32 before it is rounded to its type
    assert not dy[n:].any()
    products = torch.where(chosen[..., None], g[:, None] * y64[at], 0.0)
    ref.check(dw, products.sum(dim=2), products.abs().sum(dim=2), D, False, "dweights")
    assert dw.dtype == torch.float32 and not dw.cpu()[~chosen].any()
    # without weights: ones
    ones = y64[at] * chosen[..., None]
    ref.check(tab_amd.Combine(y.cuda(), places.cuda(), None, M, k, R, D), ones.sum(dim=1), ones.abs().sum(dim=1), k, False, "ones")
    dy1, none = tab_amd.CombineBackward(dout.cuda(), y.cuda(), places.cuda(), None, offsets.cuda(), M, k, R, D)
    want1 = torch.zeros((R, D), dtype=torch.float64)
    want1[places[chosen].long()] = g[:, None].expand(-1, k, -1)[chosen]
    assert none is None and torch.equal(dy1.cpu().double(), want1)


def test_one_gradient_alone():
    plan, y = _problem(9, 3, 200, torch.float32)
    routing, y = [t.cuda() for t in plan], torch.nan_to_num(y).cuda()
    yd, wd = y.clone().requires_grad_(), routing[0].clone().requires_grad_()
    both = torch.autograd.grad(tab_nn.combine(yd, tab_nn.Routing(wd, *routing[1:])).sum(), (yd, wd))
    dy, = torch.autograd.grad(tab_nn.combine(yd, tab_nn.Routing(*routing)).sum(), yd)
    dw, = torch.autograd.grad(tab_nn.combine(y, tab_nn.Routing(wd, *routing[1:])).sum(), wd)
    assert torch.equal(dy, both[0]) and torch.equal(dw, both[1])
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(tab_nn.combine(yd, tab_nn.Routing(*routing)).sum(), yd, create_graph=True)


def test_places_that_are_no_rows_are_left_out():
    M, k, R, D = 50, 3, 70, 90
    y, w = _rand((R, D), 3), _rand((M, k), 4)
    places = torch.randint(-5, R + 5, (M, k), generator=torch.Generator("cpu").manual_seed(5), dtype=torch.int32)
    places[0], places[1, 0] = -1, 1 << 30
    there = (places >= 0) & (places < R)
    terms = torch.where(there, w.double(), 0.0)[..., None] * y.double()[torch.where(there, places, 0).long()]
    ref.check(tab_amd.Combine(y.cuda(), places.cuda(), w.cuda(), M, k, R, D), terms.sum(dim=1), terms.abs().sum(dim=1), k, False, "out")
    dy, dw = tab_amd.CombineBackward(_rand((M, D), 6).cuda(), y.cuda(), places.cuda(), w.cuda(), None, M, k, R, D)
    assert not dw.cpu()[~there].any() and (dw.cpu()[there] != 0).all()


@types
def test_sums_are_rounded_once(dtype):
    """Rows that nearly cancel: what is left has the type's own precision."""
    y = torch.tensor([[256.0], [-255.0], [0.0078125]]).to(dtype)
    out = tab_amd.Combine(y.cuda(), torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), torch.ones((1, 3), device="cuda"), 1, 3, 3, 1)
    assert torch.equal(out.cpu(), torch.tensor([[1.0078125]]).to(dtype))


def test_gradients_are_differences():
    """Linear in the rows and in the weights: with small whole numbers the differences are exact."""
    M, k, D = 7, 2, 9
    plan = ref.plan(M, 4, k, 2, closed=1)
    g = torch.Generator("cpu").manual_seed(3)
    y, w, dout = (torch.randint(-4, 5, s, generator=g).float() for s in ((M * k, D), (M, k), (M, D)))
    f = lambda a, b: float((tab_nn.combine(a.cuda(), tab_nn.Routing(b.cuda(), *(t.cuda() for t in plan[1:]))).cpu() * dout).sum())  # noqa: E731
    yd, wd = y.cuda().requires_grad_(), w.cuda().requires_grad_()
    dy, dw = torch.autograd.grad(tab_nn.combine(yd, tab_nn.Routing(wd, *(t.cuda() for t in plan[1:]))), (yd, wd), dout.cuda())
    for r in range(0, M * k, 3):
        d = torch.zeros_like(y)
        d[r, r % D] = 1
        assert f(y + d, w) - f(y - d, w) == 2 * float(dy[r, r % D])
    for t in range(M):
        for j in range(k):
            d = torch.zeros_like(w)
            d[t, j] = 1
            assert f(y, w + d) - f(y, w - d) == 2 * float(dw[t, j])


@types
@pytest.mark.parametrize("D", [90, 700])
def test_gradients_leave_out_places_that_are_no_rows(D, dtype):
    """Rows that are some choice's place, once each, have their gradient, weights whose place is no row have none; other rows are nobody's."""
    M, k, R = 50, 3, 130
    g = torch.Generator("cpu").manual_seed(5)
    places = torch.randperm(R, generator=g)[:120].int()
    places = torch.cat((places, torch.tensor([-1, R, R + 4, 1 << 30, -7, -(1 << 31), 0x7fffffff, -1, -1, R] * 3, dtype=torch.int32)))[torch.randperm(M * k, generator=g)].view(M, k)
    there = (places >= 0) & (places < R)
    assert int(there.sum()) == 120
    y, w, dout = _rand((R, D), 3).to(dtype), _rand((M, k), 4), _rand((M, D), 6).to(dtype)
    dy, dw = tab_amd.CombineBackward(dout.cuda(), y.cuda(), places.cuda(), w.cuda(), None, M, k, R, D)
    at = places[there].long()
    want = (w.double()[..., None] * dout.double()[:, None])[there]
    ref.check(dy.cpu()[at], want, want.abs(), 1, False, "dy")
    products = torch.where(there[..., None], dout.double()[:, None] * y.double()[torch.where(there, places, 0).long()], 0.0)
    ref.check(dw, products.sum(dim=2), products.abs().sum(dim=2), D, False, "dweights")
    assert not dw.cpu()[~there].any()
    # with a number of rows that are used, those behind it are zeros, whoever's place they are not
    inside = torch.where(places < 100, places, -1)
    dy, _ = tab_amd.CombineBackward(dout.cuda(), y.cuda(), inside.cuda(), w.cuda(), torch.tensor([0, 100], dtype=torch.int32, device="cuda"), M, k, R, D)
    assert not dy[100:].any()
    on = (inside >= 0)
    want = (w.double()[..., None] * dout.double()[:, None])[on]
    ref.check(dy.cpu()[inside[on].long()], want, want.abs(), 1, False, "dy of the rows that are used")
