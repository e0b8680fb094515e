"""Workloads of the 4-bit layers and of the mixtures of experts, one dict of plain values per case.

With `own` true, `run` makes the calls a user makes of tab_amd; with `own` false it computes the same operators from
elementary torch operations in 32 bits, rounded once at the end.  The operators:

  linear4  Linear4: the activation quantized on the way (E4M3, blocks of 128), times weights of 4 bits (E2M1) with a power-of-two
           scale per group of 32
  route    nn.route: the k best experts of each token, their weights, the order of the rows by expert; with its gradient
  experts  ExpertsLinear: rows sorted by expert times their expert's packed weight (8 bits in blocks of 128x128, or 4 bits); the rows
           are the tokens' own, gathered on the way, or come sorted from a product before
  train    nn.experts_linear8 forward and backward: output, gradient of the tokens and of every expert's weight
  combine  nn.combine: a token's rows times their weights, added up; with its gradients
"""
import math

import torch

own = False

BLOCK = 128
GROUP = 32
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# 8-bit formats: dtype, largest number, explicit mantissa bits, exponent of the smallest normal number
FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0, 3, -6), "e5m2": (torch.float8_e5m2, 57344.0, 2, -14)}
NUMBERS4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _linear4(M, N, K, dtype, wide=0):
    return {"op": "linear4", "M": M, "N": N, "K": K, "dtype": dtype, "wide": wide}


def _route(M, E, k, dtype, normalize, masked, backward):
    """masked: some tokens are padding, and some experts are closed to some tokens."""
    return {"op": "route", "M": M, "E": E, "k": k, "dtype": dtype, "normalize": normalize, "masked": masked, "backward": backward}


def _experts(M, k, E, N, K, dtype, bits, gather):
    """M tokens of k experts each; gather: the rows are those of the tokens, else they come sorted."""
    return {"op": "experts", "M": M, "k": k, "E": E, "N": N, "K": K, "dtype": dtype, "bits": bits, "gather": gather}


def _train(M, k, E, N, K, dtype, grad_format, gather):
    return {"op": "train", "M": M, "k": k, "E": E, "N": N, "K": K, "dtype": dtype, "grad_format": grad_format, "gather": gather}


def _combine(M, k, D, dtype, backward):
    return {"op": "combine", "M": M, "k": k, "D": D, "dtype": dtype, "backward": backward}


def listed():
    return [
        # one token of an interactive user through a square projection: the weights' bytes and the call itself
        dict(_linear4(1, 4096, 4096, "bf16"), name="linear4_one_token"),
        # a ragged batch of requests into a classifier head of odd sizes, its input a slice of a wider projection
        dict(_linear4(24, 1003, 2050, "fp16", wide=62), name="linear4_head_ragged"),
        # a long prompt through the same projection
        dict(_linear4(4096, 4096, 4096, "bf16"), name="linear4_prompt"),
        # the tokens of sixteen users at one step of their answers
        dict(_route(16, 64, 4, "fp32", True, False, False), name="route_step"),
        # the batch of a training step with padded sequences, forward and backward
        dict(_route(16384, 64, 4, "bf16", True, True, True), name="route_train"),
        # sixteen users' step through experts of 4 bits: the bytes of the experts that are chosen
        dict(_experts(16, 4, 64, 2048, 4096, "bf16", 4, True), name="experts4_step"),
        # the second product of a step, rows sorted by the first, odd sizes
        dict(_experts(20, 3, 24, 1003, 776, "fp16", 8, False), name="experts8_rows_odd"),
        # a prompt through many experts of 8 bits, the numbers of their tokens far apart
        dict(_experts(4096, 4, 32, 2048, 4096, "bf16", 8, True), name="experts8_prompt"),
        # a training step of a layer of experts, gradients in the format of wide range
        dict(_train(8192, 2, 16, 2048, 2048, "bf16", "e5m2", True), name="train_experts"),
        # a training step of a small layer of no round sizes in full precision
        dict(_train(500, 3, 7, 390, 520, "fp32", "e4m3", True), name="train_experts_odd_fp32"),
        # the experts' rows of a prompt back to its tokens
        dict(_combine(8192, 4, 4096, "bf16", False), name="combine_prompt"),
        # the same in a training step of odd sizes in full precision
        dict(_combine(777, 3, 1531, "fp32", True), name="combine_train_odd_fp32"),
    ]


def _log(rng, low, high):
    """A whole number, even over its logarithm; half of them rounded to a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, v // 64 * 64) if rng.random() < 0.5 and v >= 64 else v


def draw(rng):
    largest = max(work(c)["flops"] for c in listed()), max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(("linear4", "linear4", "route", "experts", "experts", "experts", "train", "combine"))
        dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
        M, E = _log(rng, 1, 16384), _log(rng, 1, 128)
        k = rng.randint(1, min(8, E))
        if op == "linear4":
            c = _linear4(M, _log(rng, 64, 8192), _log(rng, 64, 8192), dtype, rng.choice((0, 0, rng.randint(1, 200))))
        elif op == "route":
            c = _route(M, E, k, dtype, rng.random() < 0.6, rng.random() < 0.5, rng.random() < 0.5)
        elif op == "experts":
            c = _experts(M, k, E, _log(rng, 64, 4096), _log(rng, 64, 4096), dtype, rng.choice((8, 4)), rng.random() < 0.6)
        elif op == "train":
            c = _train(_log(rng, 64, 8192), k, E, _log(rng, 64, 2048), _log(rng, 64, 2048), dtype, rng.choice(("e4m3", "e5m2")), rng.random() < 0.6)
        else:
            c = _combine(M, k, _log(rng, 64, 8192), dtype, rng.random() < 0.5)
        w = work(c)
        if w["flops"] <= largest[0] and w["bytes"] <= largest[1]:
            return c


def _size(dtype):
    return 4 if dtype == "fp32" else 2


def work(case):
    op, M = case["op"], case["M"]
    if op == "linear4":
        N, K, e = case["N"], case["K"], _size(case["dtype"])
        return {"bytes": M * K * e + N * K * 17 // 32 + M * N * e, "flops": 2 * M * N * K}
    k = case["k"]
    R = M * k
    if op == "route":
        E, e = case["E"], _size(case["dtype"])
        # the logits in; weights, experts, rows and places out; backward the weights' gradients in and the logits' out
        return {"bytes": M * E * e * (2 if case["backward"] else 1) + R * (20 if case["backward"] else 16) + 4 * (E + 1), "flops": M * E * (8 if case["backward"] else 4)}
    if op == "combine":
        D, e = case["D"], _size(case["dtype"])
        # the rows in, the tokens out; backward the tokens' gradients in, the rows' gradients out
        rows, tokens = (2 * R, 2 * M) if case["backward"] else (R, M)
        return {"bytes": (rows + tokens) * D * e + R * (12 if case["backward"] else 8), "flops": R * D * (6 if case["backward"] else 2)}
    E, N, K, e = case["E"], case["N"], case["K"], _size(case["dtype"])
    x = M if case["gather"] else R
    if op == "train":
        # the activation, the weights and the output's gradient read; output, the activation's and the weights' gradients written
        return {"bytes": 2 * (x * K + E * N * K + R * N) * e, "flops": 6 * R * N * K}
    chosen = E * (1 - (1 - k / E) ** M)  # experts that have a row, about
    weight = N * K * 17 // 32 if case["bits"] == 4 else N * K
    return {"bytes": int(x * K * e + chosen * weight + R * N * e), "flops": 2 * R * N * K}


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _activation(g, M, K, dtype, wide=0):
    """Rows of different sizes, a few channels that stand out, and rows of zeros as padded batches hold them; with `wide`,
    a slice of a wider tensor."""
    x = torch.randn((M, K + wide), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((M, 1), generator=g, device="cuda"))
    x *= torch.where(torch.rand((1, K + wide), generator=g, device="cuda") < 0.01, 8.0, 1.0)
    if M >= 16:
        x[torch.rand(M, generator=g, device="cuda") < 0.02] = 0
    return x.to(TYPES[dtype])[:, wide // 2:wide // 2 + K]


def _weight(g, rows, K, dtype=torch.float32):
    return (torch.randn((rows, K), generator=g, device="cuda") * K ** -0.5).to(dtype)


def _logits(g, M, E, dtype, masked):
    """Router logits: experts of different popularity; with `masked`, a sixteenth of the tokens is padding (closed to every
    expert) and another sixteenth is closed to half of the experts."""
    x = torch.randn((M, E), generator=g, device="cuda") + 0.7 * torch.randn((1, E), generator=g, device="cuda")
    if masked:
        part = torch.rand((M, 1), generator=g, device="cuda")
        closed = torch.rand((M, E), generator=g, device="cuda") < 0.5
        x = x.masked_fill((part < 1 / 16) | ((part < 1 / 8) & closed), float("-inf"))
    return x.to(TYPES[dtype])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    op, M = case["op"], case["M"]
    if op == "linear4":
        s["x"] = _activation(g, M, case["K"], case["dtype"], case["wide"])
        s["qw"], s["sw"] = _pack4(_weight(g, case["N"], case["K"]))  # as the weights are kept
        return s
    k = case["k"]
    if op == "route":
        s["logits"] = _logits(g, M, case["E"], case["dtype"], case["masked"])
        s["dweights"] = torch.randn((M, k), generator=g, device="cuda") * 1e-2
        return s
    # a step of routing that came before: a batch with some padding where there are enough tokens
    E = case.get("E", 4 * k)
    s["plan"] = _plain_route(_logits(g, M, E, "fp32", M >= 64), k, True)
    R = M * k
    if op == "combine":
        s["y"] = _activation(g, R, case["D"], case["dtype"])
        s["y"][int(s["plan"][4][-1]):] = 0  # rows of no expert
        s["dout"] = (torch.randn((M, case["D"]), generator=g, device="cuda") * 1e-2).to(TYPES[case["dtype"]])
        return s
    N, K = case["N"], case["K"]
    s["x"] = _activation(g, M if case["gather"] else R, K, case["dtype"])
    if op == "train":
        s["w"] = _weight(g, E * N, K, TYPES[case["dtype"]]).view(E, N, K)
        s["dy"] = (torch.randn((R, N), generator=g, device="cuda") * 1e-3).to(TYPES[case["dtype"]])
        return s
    packed = [_pack4(_weight(g, N, K)) if case["bits"] == 4 else _pack(_weight(g, N, K), 128, "e4m3") for _ in range(E)]
    # (stacked as bytes: the types of few bits know no stacking)
    s["qw"], s["sw"] = (torch.stack([p[i].view(torch.uint8) for p in packed]).view(packed[0][i].dtype) for i in range(2))
    return s


# ---- the operators in elementary operations, 32 bits ---------------------------------------------------------------------


def _power_of_two(e):
    """2^e as fp32, from the bits of its exponent."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax, largest):
    """The smallest e, from -126, with amax <= largest * 2^e."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    top_mantissa, top_exponent = math.frexp(largest)
    e = torch.where(mantissa <= top_mantissa, exponent - top_exponent, exponent - top_exponent + 1)
    return torch.where(amax == 0, torch.full_like(e, -126), e.clamp(min=-126))


def _pack(x, block_rows, format):
    """[M, K] -> 8-bit numbers [M, 128*ceil(K/128)] (zeros past K) and E8M0 scales [ceil(K/128), M or ceil(M/128)]."""
    dtype, largest, _, _ = FORMATS[format]
    M, K = x.shape
    KB, MB = (K + BLOCK - 1) // BLOCK, (M + block_rows - 1) // block_rows
    v = torch.nn.functional.pad(x.float(), (0, KB * BLOCK - K, 0, MB * block_rows - M)).view(MB, block_rows, KB, BLOCK)
    e = _exponent(v.abs().amax(dim=(1, 3)), largest)
    q = (v * _power_of_two(-e)[:, None, :, None]).to(dtype).view(MB * block_rows, KB * BLOCK)[:M]
    return q.contiguous(), (e + 127).to(torch.uint8).t().contiguous().view(torch.float8_e8m0fnu)


def _value(q, s, block_rows):
    """The numbers that a packed operand stands for, [M, 128*ceil(K/128)] fp32."""
    M = q.shape[0]
    scale = _power_of_two(s.view(torch.uint8).to(torch.int32) - 127).t()  # [rows or row blocks, KB]
    if block_rows > 1:
        scale = scale.repeat_interleave(block_rows, dim=0)[:M]
    return (q.float().view(M, -1, BLOCK) * scale[:, :, None]).view(M, -1)


def _rounded(x, block_rows, format):
    if x.shape[0] == 0:
        return x.float()
    q, s = _pack(x, block_rows, format)
    return _value(q, s, block_rows)[:, :x.shape[1]]


def _pack4(x):
    """[M, K] -> 4-bit numbers, two a byte, the first in the low bits, [M, 64*ceil(K/128)] (zeros past K) and E8M0 scales
    [ceil(K/128), M, 4]: the smallest power of two, from 2^-126, with which a group's largest magnitude fits."""
    M, K = x.shape
    KB = (K + BLOCK - 1) // BLOCK
    v = torch.nn.functional.pad(x.float(), (0, KB * BLOCK - K)).view(M, KB, BLOCK // GROUP, GROUP)
    e = _exponent(v.abs().amax(dim=3), NUMBERS4[-1])
    v = v * _power_of_two(-e)[..., None]
    # the nearest of the eight magnitudes, half to even: units of 1/2 below 2, of 1 below 4, of 2 below
    a = v.abs()
    code = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4)).to(torch.uint8)
    code = (code | (v < 0).to(torch.uint8) << 3).view(M, KB * BLOCK)
    q = code[:, 0::2] | code[:, 1::2] << 4
    return q.contiguous().view(torch.float4_e2m1fn_x2), (e + 127).to(torch.uint8).transpose(0, 1).contiguous().view(torch.float8_e8m0fnu)


def _value4(q, s):
    """The numbers that packed weights of 4 bits stand for, [M, 128*ceil(K/128)] fp32."""
    q = q.view(torch.uint8)
    table = torch.tensor(NUMBERS4 + tuple(-n for n in NUMBERS4), device=q.device)
    v = table[torch.stack((q & 15, q >> 4), dim=2).long()].view(q.shape[0], -1, BLOCK // GROUP, GROUP)
    return (v * _power_of_two(s.view(torch.uint8).to(torch.int32) - 127).transpose(0, 1)[..., None]).view(q.shape[0], -1)


def _plain_route(logits, k, normalize):
    """[weights, experts, rows, places, offsets]; ties go to the lowest index, -inf is never chosen."""
    M, E = logits.shape
    v = logits.float()
    top, experts = (t[:, :k] for t in torch.sort(v, dim=1, descending=True, stable=True))
    open = top > float("-inf")
    most = torch.where(open[:, :1], top[:, :1], 0.0)
    part = torch.where(open, torch.exp(top - most), 0.0)
    whole = part if normalize else torch.exp(v - most)
    weights = torch.where(open, part / whole.sum(dim=1, keepdim=True), 0.0)
    experts = torch.where(open, experts, -1)
    key = torch.where(experts < 0, E, experts).reshape(-1)
    order = torch.argsort(key, stable=True)
    counts = (key[None, :] == torch.arange(E, device=key.device)[:, None]).sum(dim=1)
    offsets = torch.nn.functional.pad(torch.cumsum(counts, dim=0), (1, 0))
    behind = torch.arange(M * k, device=key.device) >= offsets[-1]
    rows = torch.where(behind, -1, order // k)
    places = torch.empty_like(order)
    places[order] = torch.arange(M * k, device=key.device)
    places = torch.where(key == E, -1, places).view(M, k)
    return [weights] + [t.to(torch.int32).contiguous() for t in (experts, rows, places, offsets)]


def _plain_route_grad(logits, weights, experts, dweights, normalize):
    chosen, at = experts >= 0, experts.clamp(min=0).long()
    mean = (dweights * weights).sum(dim=1, keepdim=True)
    if normalize:
        p, g = torch.zeros_like(logits, dtype=torch.float32), torch.zeros_like(logits, dtype=torch.float32)
        p.scatter_add_(1, at, torch.where(chosen, weights, 0.0))
    else:
        v = logits.float()
        most = v.amax(dim=1, keepdim=True)
        p = torch.exp(v - torch.where(most > float("-inf"), most, 0.0))
        p = p / p.sum(dim=1, keepdim=True).clamp(min=1e-30)
        g = torch.zeros_like(p)
    g.scatter_add_(1, at, torch.where(chosen, dweights, 0.0))
    return (p * (g - mean)).to(logits.dtype)


def _plain_experts(s):
    c = s["case"]
    _, _, rows, _, offsets = s["plan"]
    at = offsets.tolist()
    x = _rounded(s["x"], 1, "e4m3")
    y = torch.zeros((c["M"] * c["k"], c["N"]), device="cuda")
    for e in range(c["E"]):
        if at[e] < at[e + 1]:
            w = _value4(s["qw"][e], s["sw"][e]) if c["bits"] == 4 else _value(s["qw"][e], s["sw"][e], 128)
            own_rows = slice(at[e], at[e + 1])
            y[own_rows] = x[rows[own_rows].long() if c["gather"] else own_rows] @ w[:, :c["K"]].t()
    return [y.to(TYPES[c["dtype"]])]


def _plain_train(s):
    c = s["case"]
    _, _, rows, _, offsets = s["plan"]
    at = offsets.tolist()
    R, x, dy = c["M"] * c["k"], s["x"], s["dy"]
    qx, qdy = _rounded(x, 1, "e4m3"), _rounded(dy, 1, c["grad_format"])
    y, dx, dw = torch.zeros((R, c["N"]), device="cuda"), torch.zeros(x.shape, device="cuda"), torch.zeros(s["w"].shape, device="cuda")
    for e in range(c["E"]):
        if at[e] == at[e + 1]:
            continue
        own_rows = slice(at[e], at[e + 1])
        mine = rows[own_rows].long() if c["gather"] else torch.arange(at[e], at[e + 1], device="cuda")
        w = _rounded(s["w"][e], 128, "e4m3")
        y[own_rows] = qx[mine] @ w.t()
        dx.index_add_(0, mine, qdy[own_rows] @ w)
        dw[e] = _rounded(dy[own_rows].t(), 1, c["grad_format"]) @ _rounded(x[mine].t(), 1, "e4m3").t()
    return [t.to(TYPES[c["dtype"]]) for t in (y, dx, dw)]


def _plain_combine(s):
    c = s["case"]
    weights, _, _, places, _ = s["plan"]
    chosen, at = places >= 0, places.clamp(min=0).long()
    w = torch.where(chosen, weights, 0.0)
    out = torch.zeros((c["M"], c["D"]), device="cuda")
    for j in range(c["k"]):
        out += w[:, j, None] * s["y"][at[:, j]].float()
    out = [out.to(TYPES[c["dtype"]])]
    if c["backward"]:
        dout = s["dout"].float()
        dy, dweights = torch.zeros(s["y"].shape, device="cuda"), torch.zeros_like(weights)
        for j in range(c["k"]):
            dy.index_add_(0, at[:, j], w[:, j, None] * dout)
            dweights[:, j] = torch.where(chosen[:, j], (dout * s["y"][at[:, j]].float()).sum(dim=1), 0.0)
        out += [dy.to(TYPES[c["dtype"]]), dweights]
    return out


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "linear4":
        return [(_rounded(s["x"], 1, "e4m3") @ _value4(s["qw"], s["sw"])[:, :c["K"]].t()).to(TYPES[c["dtype"]])]
    if op == "route":
        out = _plain_route(s["logits"], c["k"], c["normalize"])
        return out + ([_plain_route_grad(s["logits"], out[0], out[1], s["dweights"], c["normalize"])] if c["backward"] else [])
    return {"experts": _plain_experts, "train": _plain_train, "combine": _plain_combine}[op](s)


# ---- the calls a user makes -----------------------------------------------------------------------------------------------


def _own(s):
    import tab_amd
    from tab_amd import nn as tab_nn

    c = s["case"]
    op, M = c["op"], c["M"]
    if op == "linear4":
        return [tab_amd.Linear4(s["x"], s["qw"], s["sw"], M, c["N"], c["K"])]
    if op == "route":
        if not c["backward"]:
            return tab_amd.Route(s["logits"], M, c["E"], c["k"], c["normalize"])
        logits = s["logits"].detach().requires_grad_()
        plan = tab_nn.route(logits, c["k"], c["normalize"])
        dlogits, = torch.autograd.grad(plan.weights, logits, s["dweights"])
        return [plan.weights.detach(), plan.experts, plan.rows, plan.places, plan.offsets, dlogits]
    R = M * c["k"]
    if op == "experts":
        rows, offsets = s["plan"][2], s["plan"][4]
        return [tab_amd.ExpertsLinear(s["x"], rows if c["gather"] else None, offsets, s["qw"], s["sw"], M if c["gather"] else R, R, c["E"], c["N"], c["K"])]
    plan = tab_nn.Routing(*s["plan"])
    if op == "train":
        x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        y = tab_nn.experts_linear8(x, w, plan, gather=c["gather"], grad_format={"e4m3": tab_amd.E4M3, "e5m2": tab_amd.E5M2}[c["grad_format"]])
        dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
        return [y.detach(), dx, dw]
    if not c["backward"]:
        return [tab_amd.Combine(s["y"], plan.places, plan.weights, M, c["k"], R, c["D"])]
    y, weights = s["y"].detach().requires_grad_(), plan.weights.detach().requires_grad_()
    out = tab_nn.combine(y, plan._replace(weights=weights))
    dy, dweights = torch.autograd.grad(out, (y, weights), s["dout"])
    return [out.detach(), dy, dweights]


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def _two_to(e):
    """2^e in fp64; from the exponent's bits, because the library's power is not exact on every device."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest8(x, block_rows, format):
    """What the packed operand of x stands for, in fp64, block by block: the nearest 8-bit numbers (a multiple of the last
    place, half to even) of x over the scale, times the scale."""
    _, largest, bits, smallest = FORMATS[format]
    out = []
    for block in x.double().split(BLOCK, dim=1):
        amax = block.abs().amax(dim=1)
        if block_rows > 1:
            amax = torch.stack([a.max() for a in amax.split(block_rows)])
        # the exponent by comparison: the guess of the logarithm is at most one off
        e = torch.floor(torch.log2(torch.clamp(amax, min=2.0 ** -140) / largest)).clamp(min=-126)
        e = torch.where(amax > largest * _two_to(e), e + 1, e)
        e = torch.where((amax <= largest * _two_to(e - 1)) & (e > -126), e - 1, e)
        scale = _two_to(e)[torch.arange(block.shape[0], device=x.device) // block_rows][:, None]
        v = block / scale
        _, ex = torch.frexp(v)
        last_place = _two_to(torch.clamp(ex - 1, min=smallest) - bits)
        out.append(torch.round(v / last_place) * last_place * scale)
    return torch.cat(out, dim=1)


def _stored(case, q, s, columns):
    """The numbers of a packed weight in fp64."""
    scale = _two_to(s.view(torch.uint8).double() - 127)
    at = torch.arange(columns, device=q.device)
    if case.get("bits", 4) == 4:
        byte = q.view(torch.uint8)[:, at // 2].long()
        nibble = torch.where(at % 2 == 0, byte & 15, byte >> 4)
        exponent, mantissa, sign = nibble >> 1 & 3, (nibble & 1).double(), 1.0 - 2.0 * (nibble >> 3)
        number = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * _two_to(exponent - 1))
        return sign * number * scale[at // BLOCK, :, at % BLOCK // GROUP].t()
    rows = torch.arange(q.shape[0], device=q.device) // BLOCK
    return q[:, :columns].double() * scale.t()[rows][:, at // BLOCK]


def _exact_route(case, s):
    """Weights in fp64, whole numbers by counting: an expert's place among its row's is the number of those before it."""
    v = s["logits"].double()
    M, E, k = case["M"], case["E"], case["k"]
    experts = torch.full((M, k), -1, dtype=torch.int64, device=v.device)
    left = v.clone()
    for j in range(k):
        best = left.amax(dim=1, keepdim=True)
        first = torch.where(left == best, torch.arange(E, device=v.device), E).amin(dim=1, keepdim=True)
        experts[:, j:j + 1] = torch.where(best > float("-inf"), first, -1)
        left.scatter_(1, first, float("-inf"))
    chosen = experts >= 0
    top = torch.where(chosen, torch.gather(v, 1, experts.clamp(min=0)), float("-inf"))
    norm = torch.logsumexp(top if case["normalize"] else v, dim=1, keepdim=True)
    weights = torch.where(chosen, torch.exp(top - torch.where(norm > float("-inf"), norm, 0.0)), 0.0)
    flat = experts.reshape(-1)
    rows = torch.cat([torch.nonzero(flat == e)[:, 0] for e in range(E)])
    offsets = torch.tensor([0] + [int((flat == e).sum()) for e in range(E)], device=v.device).cumsum(0)
    places = torch.full_like(flat, -1)
    places[rows] = torch.arange(rows.numel(), device=v.device)
    tokens = torch.full_like(flat, -1)
    tokens[:rows.numel()] = rows // k
    out = [weights] + [t.to(torch.int32) for t in (experts, tokens, places.view(M, k), offsets)]
    if case["backward"]:
        d = v.new_zeros((M, E))
        g = torch.where(chosen, s["dweights"].double(), 0.0)
        mean = (g * weights).sum(dim=1, keepdim=True)
        if case["normalize"]:
            for j in range(k):
                d[torch.arange(M, device=v.device), experts[:, j].clamp(min=0)] += weights[:, j] * (g - mean)[:, j]
        else:
            p = torch.exp(v - torch.where(norm > float("-inf"), norm, 0.0))
            d -= p * mean
            for j in range(k):
                d[torch.arange(M, device=v.device), experts[:, j].clamp(min=0)] += weights[:, j] * g[:, j]
        out.append(d)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear4":
        return [torch.matmul(_nearest8(s["x"], 1, "e4m3"), _stored(case, s["qw"], s["sw"], case["K"]).t())]
    if op == "route":
        return _exact_route(case, s)
    weights, _, rows, places, offsets = s["plan"]
    M, k = case["M"], case["k"]
    R, ends = M * k, offsets.tolist()
    if op == "combine":
        # row by row of the experts: its token, and which of the token's choices it is
        r = torch.nonzero(rows >= 0)[:, 0]
        token = rows[r].long()
        choice = (places[token] == r[:, None]).int().argmax(dim=1)
        w = weights[token, choice].double()[:, None]
        y = s["y"].double()
        out = [torch.zeros((M, case["D"]), dtype=torch.float64, device=y.device).index_add_(0, token, w * y[r])]
        if case["backward"]:
            g = s["dout"].double()[token]
            dy, dweights = torch.zeros_like(y), torch.zeros((M, k), dtype=torch.float64, device=y.device)
            dy[r] = w * g
            dweights[token, choice] = (g * y[r]).sum(dim=1)
            out += [dy, dweights]
        return out
    x = s["x"][rows.clamp(min=0).long()] if case["gather"] else s["x"]
    groups = [slice(a, b) for a, b in zip(ends, ends[1:])]
    y = torch.zeros((R, case["N"]), dtype=torch.float64, device=x.device)
    if op == "experts":
        for e, g in enumerate(groups):
            if g.start < g.stop:
                y[g] = torch.matmul(_nearest8(x[g], 1, "e4m3"), _stored(case, s["qw"][e], s["sw"][e], case["K"]).t())
        return [y]
    f = case["grad_format"]
    dx, dw = torch.zeros(x.shape, dtype=torch.float64, device=x.device), torch.zeros(s["w"].shape, dtype=torch.float64, device=x.device)
    for e, g in enumerate(groups):
        if g.start == g.stop:
            continue
        w, xe, dye = _nearest8(s["w"][e], 128, "e4m3"), x[g], s["dy"][g]
        y[g] = torch.matmul(_nearest8(xe, 1, "e4m3"), w.t())
        dx[g] = torch.matmul(_nearest8(dye, 1, f), w)
        dw[e] = torch.matmul(_nearest8(dye.t(), 1, f), _nearest8(xe.t(), 1, "e4m3").t())
    if case["gather"]:  # a token's gradient is the sum over its rows
        summed = torch.zeros((M, case["K"]), dtype=torch.float64, device=x.device)
        for j in range(k):
            p = places[:, j].long()
            summed += torch.where(p[:, None] >= 0, dx[p.clamp(min=0)], 0.0)
        dx = summed
    return [y, dx, dw]
