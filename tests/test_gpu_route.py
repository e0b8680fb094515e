"""The router against its definition in 64 bits: choices, order and places equal, weights and gradients within what their roundings allow."""
import pytest
import torch

import experts_reference as ref
import tab_amd
from tab_amd import nn as tab_nn

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
types = pytest.mark.parametrize("dtype", TYPES, ids=["fp32", "bf16", "fp16"])
normalizes = pytest.mark.parametrize("normalize", [True, False], ids=["chosen", "all"])


def _logits(M, E, seed, dtype=torch.float32, masked=True, size=3.0):
    g = torch.Generator("cpu").manual_seed(seed)
    x = size * torch.randn((M, E), generator=g)
    if masked and M > 4:
        x[3] = float("-inf")                              # a padded token
        x[4, 1:] = float("-inf")                          # one with a single open expert
        x[1] = x[1, :1]                                   # ties
        x[2, : E // 2] = float("-inf")
        x[0] = torch.finfo(dtype).min                     # the type's lowest value is a value
    return x.to(dtype)


def _check(out, logits, k, normalize):
    weights, experts, rows, places, offsets = (t.cpu() for t in out)
    w, *want, _ = ref.route(logits, k, normalize)
    for got, expected in zip((experts, rows, places, offsets), want):
        assert got.dtype == torch.int32 and torch.equal(got, expected)
    # The difference to the largest logit is rounded once (2^-24 of it, as much of its exponential), the exponential is off by 2 units, the sum of E of them in
    # a tree of at most 22 additions by 22 and by the mean of the terms' own errors (2 + ln E + 1), the quotient by one: (difference + 40) 2^-24; below 2^-126
    # an exponential may be zero
    v = logits.double()
    spread = torch.zeros_like(w)
    for t in range(v.shape[0]):
        on = experts[t] >= 0
        chosen = v[t, experts[t][on].long()]
        spread[t, on] = (chosen - chosen.max()).abs() if on.any() else chosen
    bound = (spread + 40) * 2.0 ** -24 * w + 2.0 ** -126
    off = (weights.double() - w).abs()
    nan = torch.isnan(w)
    assert torch.equal(torch.isnan(weights), nan)
    assert (off <= bound)[~nan].all()


@types
@normalizes
@pytest.mark.parametrize("M,E,k", [(1, 1, 1), (1, 64, 4), (5, 3, 3), (16, 64, 4), (7, 33, 5), (40, 65, 8), (20, 128, 32), (6, 200, 7), (9, 500, 2), (6, 1024, 32), (128, 8, 2)])
def test_route_in_one_launch(M, E, k, normalize, dtype):
    logits = _logits(M, E, M * E + k, dtype)
    _check(tab_amd.Route(logits.cuda(), M, E, k, normalize), logits, k, normalize)


@normalizes
@pytest.mark.parametrize("M,E,k", [(129, 8, 2), (300, 64, 4), (257, 1, 1), (200, 1024, 3), (150, 65, 32), (1000, 5, 5), (4097, 16, 2)])
def test_route_of_many_tokens(M, E, k, normalize):
    logits = _logits(M, E, M + E + k, torch.bfloat16)
    _check(tab_amd.Route(logits.cuda(), M, E, k, normalize), logits, k, normalize)


def test_route_of_a_long_batch():
    """More tokens than the quick reference can go through: against torch's stable sorts."""
    M, E, k = 70001, 24, 3
    logits = _logits(M, E, 1, torch.bfloat16)
    weights, experts, rows, places, offsets = (t.cpu() for t in tab_amd.Route(logits.cuda(), M, E, k))
    top, order = (t[:, :k] for t in torch.sort(logits.double(), dim=1, descending=True, stable=True))
    want = torch.where(top > float("-inf"), order, -1)
    assert torch.equal(experts.long(), want)
    key = torch.where(want < 0, E, want).flatten()
    at = torch.argsort(key, stable=True)
    n = int((key < E).sum())
    assert torch.equal(rows[:n].long(), at[:n] // k) and (rows[n:] == -1).all()
    flat = torch.full((M * k,), -1)
    flat[at[:n]] = torch.arange(n)
    assert torch.equal(places.flatten().long(), flat)
    assert offsets.tolist() == [int((key < e).sum()) for e in range(E + 1)]
    sums = torch.where((want >= 0).any(dim=1), weights.double().sum(dim=1), 1.0)
    assert ((sums - 1).abs() <= k * 2.0 ** -23).all()


@types
@normalizes
def test_infinities_and_not_a_number(normalize, dtype):
    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[1.0, nan, 3.0, nan], [inf, 1.0, inf, 0.0], [-inf, -inf, -inf, nan], [-0.0, 0.0, -0.0, 0.0], [1.0, -inf, 2.0, -inf]]).to(dtype)
    for M in (5, 200):
        x = logits.repeat((M + 4) // 5, 1)[:M]
        _check(tab_amd.Route(x.cuda(), M, 4, 3, normalize), x, 3, normalize)


def test_no_token_has_an_expert():
    for M in (3, 300):
        weights, experts, rows, places, offsets = tab_amd.Route(torch.full((M, 6), float("-inf"), device="cuda"), M, 6, 2)
        assert not weights.any() and (experts == -1).all() and (rows == -1).all() and (places == -1).all() and not offsets.any()


def test_logits_that_are_columns_of_a_wider_matrix():
    for M in (4, 200):
        wide = _logits(M, 50, 7)
        part = wide.cuda()[:, 5:25]
        for a, b in zip(tab_amd.Route(part, M, 20, 3), tab_amd.Route(part.contiguous(), M, 20, 3)):
            assert torch.equal(a, b)


@types
@normalizes
@pytest.mark.parametrize("M,E,k", [(1, 1, 1), (6, 64, 4), (33, 7, 7), (21, 130, 6), (12, 1000, 32)])
def test_gradients(M, E, k, normalize, dtype):
    logits = _logits(M, E, M + E, dtype)
    g = torch.randn((M, k), generator=torch.Generator("cpu").manual_seed(3))
    x = logits.cuda().requires_grad_()
    plan = tab_nn.route(x, k, normalize)
    assert plan.weights.requires_grad and not any(t.requires_grad for t in plan[1:])
    dx, = torch.autograd.grad(plan.weights, x, g.cuda())
    assert dx.dtype == dtype and dx.shape == logits.shape
    w, experts, *_, whole = ref.route(logits, k, normalize)
    want, mag = torch.zeros((M, E), dtype=torch.float64), torch.zeros((M, E), dtype=torch.float64)
    spread = torch.zeros((M, 1), dtype=torch.float64)
    for t in range(M):
        on = experts[t] >= 0
        if not on.any():
            continue
        e, gt, wt = experts[t][on].long(), g[t][on].double(), w[t][on]
        p, at = (torch.zeros(E, dtype=torch.float64) for _ in range(2))
        p[:] = whole[t]
        if normalize:
            p.zero_()
            p[e] = wt
        at[e] = gt
        want[t] = p * (at - (gt * wt).sum())
        mag[t] = p * (at.abs() + (gt * wt).abs().sum())
        finite = logits[t].double()
        finite = finite[finite > float("-inf")]
        spread[t] = min(float(finite.max() - finite.min()), 110.0)  # (where it is larger the weight is zero)
    # each factor as in the weights' test; the sum of k products and the last product and difference 36 more
    off = (dx.cpu().double() - want).abs()
    bound = (spread + 80) * 2.0 ** -23 * mag + ref.UNIT[dtype] * (1 + 2.0 ** -10) * want.abs() + ref.TINY[dtype] + 2.0 ** -120
    assert (off <= bound).all(), float((off / bound).max())


@normalizes
def test_gradients_are_differences(normalize):
    """Central differences of the definition in 64 bits."""
    M, E, k, h = 3, 9, 4, 1e-6
    logits = _logits(M, E, 11, masked=False, size=1.0)
    g = torch.randn((M, k), generator=torch.Generator("cpu").manual_seed(4)).double()
    x = logits.cuda().requires_grad_()
    dx, = torch.autograd.grad(tab_nn.route(x, k, normalize).weights, x, g.float().cuda())
    f = lambda v: float((ref.route(v, k, normalize)[0] * g.float().double()).sum())  # noqa: E731
    for t in range(M):
        for e in range(E):
            d = torch.zeros((M, E), dtype=torch.float64)
            d[t, e] = h
            assert abs((f(logits.double() + d) - f(logits.double() - d)) / (2 * h) - float(dx[t, e])) < 1e-5


def test_same_call_same_bits_and_more_dimensions():
    logits = _logits(600, 32, 12).cuda()
    first = tab_amd.Route(logits, 600, 32, 4)
    for _ in range(3):
        for a, b in zip(first, tab_amd.Route(logits, 600, 32, 4)):
            assert torch.equal(a, b)
    x = logits.view(6, 100, 32).clone().requires_grad_()
    plan = tab_nn.route(x, 4)
    for a, b in zip(first, plan):
        assert torch.equal(a, b)
    dx, = torch.autograd.grad(plan.weights.square().sum(), x)
    assert dx.shape == x.shape
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(tab_nn.route(x, 4).weights.sum(), x, create_graph=True)


def test_as_many_rows_as_a_call_may_have():
    """2^31 - 544 rows: the steps of a workgroup's threads past the last row must not come round to numbers below zero.  (43 GB of the GPU's memory.)"""
    k, closed = 32, 3
    M = (0x7fffffff - 512) // k
    logits = (-torch.arange(k, device="cuda", dtype=torch.bfloat16)).repeat(M, 1)
    logits[M - closed:] = float("-inf")
    weights, experts, rows, places, offsets = tab_amd.Route(logits, M, k, k)
    del logits
    n = M - closed  # rows of each expert
    assert torch.equal(offsets.cpu(), torch.arange(k + 1, dtype=torch.int32) * n)
    tokens = torch.arange(n, device="cuda", dtype=torch.int32)
    for e in range(k):
        assert torch.equal(rows[e * n:(e + 1) * n], tokens)
        assert torch.equal(places[:n, e], tokens + e * n)
        assert (experts[:n, e] == e).all() and (weights[:n, e] == weights[0, e]).all()
    assert (rows[k * n:] == -1).all() and (places[n:] == -1).all() and (experts[n:] == -1).all() and not weights[n:].any()
    want = torch.softmax(-torch.arange(k, dtype=torch.float64), 0)
    # a difference exact in fp32, an exponential, a sum of 32 and a division: as in the test of the weights
    assert ((weights[0].cpu().double() - want).abs() <= (32 + 80) * 2.0 ** -23 * want).all()
    del weights, experts, rows, places
    torch.cuda.empty_cache()


def test_gradients_of_more_tokens_than_a_launch_has_waves():
    """Past 2^25 tokens there are several launches."""
    M, E = (1 << 26) + 70001, 2
    logits = torch.randn((M, E), generator=torch.Generator("cuda").manual_seed(1), device="cuda", dtype=torch.bfloat16)
    x = logits.requires_grad_()
    routing = tab_nn.route(x, 1, normalize=False)
    g = torch.randn((M, 1), generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    dx, = torch.autograd.grad(routing.weights, x, g)
    for at in (slice(0, 1000), slice(0, None, 6007), slice((1 << 25) - 100, (1 << 25) + 100), slice(M - 100000, M)):
        v, e, gt = logits.detach()[at].double(), routing.experts[at].long(), g[at].double()
        p = torch.softmax(v, 1)
        w = p.gather(1, e)
        chosen = torch.zeros_like(p).scatter_(1, e, gt)
        want, mag = p * (chosen - gt * w), p * (chosen.abs() + (gt * w).abs())
        assert torch.equal(e, torch.where(v[:, :1] >= v[:, 1:], 0, 1))
        # as in the test of the gradients
        off, spread = (dx[at].double() - want).abs(), (v[:, :1] - v[:, 1:]).abs()
        assert (off <= (spread + 80) * 2.0 ** -23 * mag + ref.UNIT[torch.bfloat16] * (1 + 2.0 ** -10) * want.abs() + ref.TINY[torch.bfloat16]).all()
