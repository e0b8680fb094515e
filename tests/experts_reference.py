"""4-bit weights and mixtures of experts in 64 bits, on the CPU, for the tests: the definitions, element by element."""
import torch

from layers8_reference import TINY, UNIT, blocks, quantize, two_to, value

GROUP = 32
NUMBERS4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize4(x):
    """Numbers (R, padded) and scale exponents (blocks, R, 4) of x; the exponent is 128 (NaN) for a group with infinities or NaN."""
    R, K = x.shape
    v = torch.zeros((R, blocks(K) * 128), dtype=torch.float64)
    v[:, :K] = x.double()
    g = v.view(R, -1, GROUP)
    bad = ~torch.isfinite(g).all(dim=2)
    g = torch.where(bad[..., None], torch.zeros_like(g), g)
    a = g.abs().amax(dim=2)
    _, top = torch.frexp(a / 6)
    e = torch.where(a <= 6 * two_to(top - 1), top - 1, top)
    e = torch.where(a == 0, torch.full_like(e, -126), e.clamp(min=-126)).long()
    n = g / two_to(e)[..., None]
    # the nearest of the numbers, between two the one whose place is even
    off = (n.abs()[..., None] - NUMBERS4).abs()
    least = off.amin(dim=-1, keepdim=True)
    near = off == least
    first, last = near.int().argmax(dim=-1), 7 - near.flip(-1).int().argmax(dim=-1)
    place = torch.where(first % 2 == 0, first, last)
    q = torch.where(n < 0, -1.0, 1.0) * NUMBERS4[place]
    e = torch.where(bad, torch.full_like(e, 128), e)
    return q.view(R, -1), e.view(R, -1, 4).transpose(0, 1)


def numbers4(Q):
    """The numbers of the library's packed tensor (R, padded / 2) in fp64."""
    b = Q.cpu().view(torch.uint8).long()
    code = torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)
    return torch.where(code >= 8, -1.0, 1.0).double() * NUMBERS4[code & 7]


def value4(q, e):
    scale = torch.where(e == 128, torch.full(e.shape, float("nan"), dtype=torch.float64), two_to(e.clamp(max=127))).transpose(0, 1)
    return (q.view(q.shape[0], -1, 4, GROUP) * scale[..., None]).view(q.shape[0], -1)


def unpack4(Q, S):
    """What the library's packed weight stands for, (R, padded) fp64."""
    return value4(numbers4(Q), S.cpu().view(torch.uint8).long() - 127)


def route(logits, k, normalize):
    """(weights fp64, experts, rows, places, offsets, softmax) one token at a time."""
    M, E = logits.shape
    weights, experts = torch.zeros((M, k), dtype=torch.float64), torch.full((M, k), -1, dtype=torch.int32)
    whole = torch.zeros((M, E), dtype=torch.float64)
    for t in range(M):
        v = logits[t].double()
        key = [(-float("inf") if x != x else -x, e) for e, x in enumerate(v.tolist()) if x != float("-inf")]
        key.sort(key=lambda p: (0 if v[p[1]] != v[p[1]] else 1, p[0], p[1]))
        chosen = [e for _, e in key[:k]]
        if not chosen:
            continue
        if torch.isnan(v).any() or (v == float("inf")).any():
            whole[t] = float("nan")
        else:
            p = torch.exp(v - v.max())
            whole[t] = p / p.sum()
        experts[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        w = whole[t, chosen]
        if normalize:
            part = torch.exp(v[chosen] - v[chosen].max())
            w = part / part.sum()
        weights[t, :len(chosen)] = w
    rows, places, offsets = torch.full((M * k,), -1, dtype=torch.int32), torch.full((M, k), -1, dtype=torch.int32), [0]
    for e in range(E):
        for t, j in (experts == e).nonzero().tolist():
            rows[offsets[-1] + int((places.flatten() >= offsets[-1]).sum())] = t
            places[t, j] = offsets[-1] + int((places.flatten() >= offsets[-1]).sum())
        offsets.append(offsets[-1] + int((experts == e).sum()))
    return weights, experts, rows, places, torch.tensor(offsets, dtype=torch.int32), whole


def runs(offsets):
    at = offsets.tolist()
    return [(e, at[e], at[e + 1]) for e in range(len(at) - 1) if at[e] < at[e + 1]]


def plan(M, E, k, seed, closed=0, shy=()):
    """A routing of M tokens: (weights, experts, rows, places, offsets).  closed: tokens without an expert; shy: experts that nobody takes."""
    g = torch.Generator("cpu").manual_seed(seed)
    logits = torch.randn((M, E), generator=g) + torch.randn((1, E), generator=g)
    if closed:
        logits[torch.randperm(M, generator=g)[:closed]] = float("-inf")
    logits[:, list(shy)] = float("-inf")
    w, *rest, _ = route(logits, k, True)
    return [w.float(), *rest]


def check(got, want, magnitudes, terms, sixteen, what):
    """Sums of `terms` products: in fp32 at most `terms` roundings of partial sums, each bounded by the sum of magnitudes; towards 16 bits, besides, each product
    of a group of eight in K loses at most 2^-13 of the group's largest, which is at most the group's sum of magnitudes: 2^-10 of the sum of magnitudes
    over all groups.  Then one rounding to the output's type."""
    dtype = got.dtype
    bound = (terms * 2.0 ** -24 + (2.0 ** -10 if sixteen else 0)) * magnitudes + UNIT[dtype] * (1 + 2.0 ** -10) * want.abs() + TINY[dtype]
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    if dtype == torch.float16:  # beyond the type's range it is an infinity
        inside = want.abs() < 65000
        got, want, bound = got[inside], want[inside], bound[inside]
    off = (got - want).abs()
    assert (off <= bound).all(), (what, float((off / bound).max()))


def product(a, b):
    """a b^T and the sums of its magnitudes."""
    return a @ b.t(), a.abs() @ b.abs().t()


def by_expert(x, w, rows, offsets, N):
    """y and its magnitudes (R, N) from what the tokens (or sorted rows, rows None) and the experts' weights stand for."""
    R = x.shape[0] if rows is None else rows.numel()
    y, mag = torch.zeros((R, N), dtype=torch.float64), torch.zeros((R, N), dtype=torch.float64)
    for e, a, b in runs(offsets):
        xe = x[a:b] if rows is None else x[rows[a:b].long()]
        y[a:b], mag[a:b] = product(xe, w[e])
    return y, mag


def rounded(x, block_rows, format):
    """What x stands for once packed in 8 bits."""
    return value(*quantize(x, block_rows, format), block_rows)[:, :x.shape[1]]
