"""Workloads of the 8-bit layers and of the norms around a block, one dict of plain values per case.

With `own` true, `run` makes the calls a user makes of tab_amd; with `own` false it computes the same operators from
elementary torch operations in 32 bits, rounded once at the end.  The operators:

  quantize   Quantize8 / Quantize8Transposed / Quantize8Both: 8-bit numbers with a power-of-two scale per block of 128
  linear     Linear8: the activation quantized on the way, times packed weights (128x128 blocks)
  packed     Linear8Packed: both operands packed
  train      nn.linear8 forward and backward: output, gradient of the input and of the weight
  norm       Norm / NormResidual: the norm after a block, its gate, the scaled residual and the norm before the next block
  norm_grad  NormResidualBackward: gradients of the residual stream, of the block's output, of the gate and of both weights
"""
import math

import torch

own = False

BLOCK = 128
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
# 8-bit formats: dtype, largest number, explicit mantissa bits, exponent of the smallest normal number
FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0, 3, -6), "e5m2": (torch.float8_e5m2, 57344.0, 2, -14)}
EPS = 1e-6


def _quantize(M, K, dtype, block_rows, format, layout, wide=0):
    return {"op": "quantize", "M": M, "K": K, "dtype": dtype, "block_rows": block_rows, "format": format, "layout": layout, "wide": wide}


def _linear(M, N, K, dtype, wide=0):
    return {"op": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "wide": wide}


def _packed(M, N, K, dtype, format):
    return {"op": "packed", "M": M, "N": N, "K": K, "dtype": dtype, "format": format}


def _train(M, N, K, dtype, grad_format):
    return {"op": "train", "M": M, "N": N, "K": K, "dtype": dtype, "grad_format": grad_format}


def _norm(M, D, dtype, gates, output, block=True):
    """gates: rows of the gate; 0 for none.  output: "none", "plain" or "8bit" for the norm before the next block."""
    return {"op": "norm", "M": M, "D": D, "dtype": dtype, "gates": gates, "output": output, "block": block}


def _norm_grad(M, D, dtype, gates):
    return {"op": "norm_grad", "M": M, "D": D, "dtype": dtype, "gates": gates}


def listed():
    return [
        # one token of an interactive user through a square projection: the weights' bytes and the call itself
        dict(_linear(1, 4096, 4096, "bf16"), name="linear_one_token"),
        # a ragged batch of requests into a classifier head of odd sizes, its input a slice of a wider projection
        dict(_linear(24, 1003, 2050, "fp16", wide=62), name="linear_head_ragged"),
        # a prompt of moderate length, operands packed by the layer before
        dict(_packed(512, 4096, 4096, "bf16", "e4m3"), name="packed_prompt"),
        # the largest product: a long batch through a wide layer
        dict(_linear(8192, 8192, 8192, "bf16"), name="linear_large"),
        # a training step of an ordinary layer, gradients in the format of wide range
        dict(_train(4096, 4096, 2048, "bf16", "e5m2"), name="train_ordinary"),
        # a training step of a small layer of no round sizes in full precision
        dict(_train(1000, 776, 520, "fp32", "e4m3"), name="train_odd_fp32"),
        # an activation for a training step: packed along its rows and along its columns
        dict(_quantize(8192, 4096, "bf16", 1, "e4m3", "both"), name="quantize_both"),
        # a weight of odd sizes packed in 128x128 blocks out of a wider parameter
        dict(_quantize(1531, 1333, "fp32", 128, "e4m3", "rows", wide=27), name="quantize_weight_odd"),
        # one token between two 8-bit layers
        dict(_norm(1, 4096, "bf16", 1, "8bit"), name="norm_one_token"),
        # a large batch of sequences with a gate for each of them
        dict(_norm(16384, 4096, "bf16", 16, "plain"), name="norm_large"),
        # the same in training, backward
        dict(_norm_grad(16384, 4096, "bf16", 16), name="norm_grad_large"),
        # the integer sums of a ternary layer of odd width in full precision, a gate for each token, backward
        dict(_norm_grad(777, 1531, "fp32", 777), name="norm_grad_odd_fp32"),
    ]


def _log(rng, low, high):
    """A whole number, even over its logarithm; half of them rounded to a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, v // 64 * 64) if rng.random() < 0.5 and v >= 64 else v


def draw(rng):
    largest = max(work(c)["flops"] for c in listed()), max(work(c)["bytes"] for c in listed())
    while True:
        op = rng.choice(("quantize", "linear", "linear", "packed", "train", "norm", "norm", "norm_grad"))
        dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
        format = rng.choice(("e4m3", "e4m3", "e5m2"))
        rows = _log(rng, 1, 16384)
        wide = rng.choice((0, 0, rng.randint(1, 200)))
        if op == "quantize":
            c = _quantize(rows, _log(rng, 64, 8192), dtype, rng.choice((1, 1, 128)), format, rng.choice(("rows", "columns", "both")), wide)
        elif op == "linear":
            c = _linear(rows, _log(rng, 64, 8192), _log(rng, 64, 8192), dtype, wide)
        elif op == "packed":
            c = _packed(rows, _log(rng, 64, 8192), _log(rng, 64, 8192), dtype, format)
        elif op == "train":
            c = _train(_log(rng, 64, 8192), _log(rng, 64, 4096), _log(rng, 64, 4096), dtype, format)
        else:
            gates = rng.choice((0, 1, rows, max(g for g in range(1, 17) if rows % g == 0)))
            D = _log(rng, 64, 8192)
            c = _norm(rows, D, dtype, gates, rng.choice(("none", "plain", "8bit")), True) if op == "norm" else _norm_grad(rows, D, dtype, gates)
            if op == "norm" and rng.random() < 0.2:  # the first norm of a network: no block before it
                c.update(block=False, gates=0, output=rng.choice(("plain", "8bit")))
        w = work(c)
        if w["flops"] <= largest[0] and w["bytes"] <= largest[1]:
            return c


def _size(dtype):
    return 4 if dtype == "fp32" else 2


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        M, D, G, e = case["M"], case["D"], case["gates"], _size(case["dtype"])
        if op == "norm":
            packed = M * D + M * ((D + 127) // 128)
            out = {"none": 0, "plain": M * D * e, "8bit": packed}[case["output"]]
            streams = 3 if case["block"] else 1  # X, Y and R, or X alone
            weights = (4 * D if case["block"] else 0) + (4 * D if case["output"] != "none" else 0)
            return {"bytes": streams * M * D * e + out + weights + G * D * e, "flops": (12 if case["block"] else 4) * M * D}
        # dR, dH, R, Y in; dX, dY out; the gate in and out, two weights in and out
        return {"bytes": 6 * M * D * e + 2 * G * D * e + 16 * D, "flops": 30 * M * D}
    if op == "quantize":
        M, K, e = case["M"], case["K"], _size(case["dtype"])
        layouts = 2 if case["layout"] == "both" else 1
        return {"bytes": M * K * e + layouts * (M * K + M * K // (128 * case["block_rows"])), "flops": 3 * M * K}
    M, N, K, e = case["M"], case["N"], case["K"], _size(case["dtype"])
    if op == "linear":
        return {"bytes": M * K * e + N * K + M * N * e, "flops": 2 * M * N * K}
    if op == "packed":
        return {"bytes": M * K + N * K + M * N * e, "flops": 2 * M * N * K}
    # x, w and dy read; y, dx and dw written
    return {"bytes": 2 * (M * K + N * K + M * N) * e, "flops": 6 * M * N * K}


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


def _weight(g, N, K, wide=0, dtype=torch.float32):
    return (torch.randn((N, K + wide), generator=g, device="cuda") * K ** -0.5).to(dtype)[:, wide // 2:wide // 2 + K]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("norm", "norm_grad"):
        M, D, G = case["M"], case["D"], case["gates"]
        s["x"] = _activation(g, M, D, case["dtype"])
        s["y"] = _activation(g, M, D, case["dtype"]) * 3 if case.get("block", True) else None
        s["gate"] = (torch.randn((G, D), generator=g, device="cuda") * 0.3 + 0.5).to(TYPES[case["dtype"]]) if G else None
        s["w_post"] = torch.rand(D, generator=g, device="cuda") + 0.5 if case.get("block", True) else None
        s["w_pre"] = torch.rand(D, generator=g, device="cuda") + 0.5 if case.get("output") != "none" else None
        s["alpha"] = 0.875
        if op == "norm_grad":
            s["dr"] = (torch.randn((M, D), generator=g, device="cuda") * 1e-2).to(TYPES[case["dtype"]])
            s["dh"] = (torch.randn((M, D), generator=g, device="cuda") * 1e-2).to(TYPES[case["dtype"]])
    elif op == "quantize":
        if case["block_rows"] == 128:
            s["x"] = _weight(g, case["M"], case["K"], case["wide"], TYPES[case["dtype"]])
        else:
            s["x"] = _activation(g, case["M"], case["K"], case["dtype"], case["wide"])
    elif op == "train":
        s["x"] = _activation(g, case["M"], case["K"], case["dtype"])
        s["w"] = _weight(g, case["N"], case["K"]).to(TYPES[case["dtype"]])
        s["dy"] = (torch.randn((case["M"], case["N"]), generator=g, device="cuda") * 1e-3).to(TYPES[case["dtype"]])
    else:
        # the weights as they are kept: packed in 128x128 blocks
        s["qw"], s["sw"] = _pack(_weight(g, case["N"], case["K"]), 128, "e4m3")
        x = _activation(g, case["M"], case["K"], "fp32" if op == "packed" else case["dtype"], case.get("wide", 0))
        if op == "packed":
            s["qx"], s["sx"] = _pack(x, 1, case["format"])
        else:
            s["x"] = x
    return s


# ---- the operators in elementary operations, 32 bits ---------------------------------------------------------------------


def _power_of_two(e):
    """2^e as fp32, from the bits of its exponent."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pack(x, block_rows, format):
    """[M, K] -> 8-bit numbers [M, 128*ceil(K/128)] (zeros past K) and E8M0 scales [ceil(K/128), M or ceil(M/128)]: the
    smallest power of two, from 2^-126, with which a block's largest magnitude fits the format."""
    dtype, largest, _, _ = FORMATS[format]
    M, K = x.shape
    KB, MB = (K + BLOCK - 1) // BLOCK, (M + block_rows - 1) // block_rows
    v = torch.nn.functional.pad(x.float(), (0, KB * BLOCK - K, 0, MB * block_rows - M)).view(MB, block_rows, KB, BLOCK)
    amax = v.abs().amax(dim=(1, 3))
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    top_mantissa, top_exponent = math.frexp(largest)
    e = torch.where(mantissa <= top_mantissa, exponent - top_exponent, exponent - top_exponent + 1)
    e = torch.where(amax == 0, torch.full_like(e, -126), e.clamp(min=-126))
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
    q, s = _pack(x, block_rows, format)
    return _value(q, s, block_rows)[:, :x.shape[1]]


def _plain_norm(s):
    c = s["case"]
    dtype = TYPES[c["dtype"]]
    r = s["x"].float()
    if c["block"]:
        y = s["y"].float()
        z = y * torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS) * s["w_post"]
        if s["gate"] is not None:
            z = (z.view(c["gates"], -1, c["D"]) * s["gate"].float()[:, None]).view(c["M"], c["D"])
        r = s["alpha"] * r + z
    out = [r.to(dtype)] if c["block"] else []
    if c["output"] != "none":
        h = r * torch.rsqrt((r * r).mean(dim=1, keepdim=True) + EPS) * s["w_pre"]
        out += [h.to(dtype)] if c["output"] == "plain" else _pack(h, 1, "e4m3")
    return out


def _plain_norm_grad(s):
    c = s["case"]
    M, D, G = c["M"], c["D"], c["gates"]
    dtype = TYPES[c["dtype"]]
    r, y, dr, dh = s["x"].float(), s["y"].float(), s["dr"].float(), s["dh"].float()
    p = torch.rsqrt((r * r).mean(dim=1, keepdim=True) + EPS)
    a = dh * s["w_pre"]
    t = dr + p * a - r * p ** 3 * (r * a).mean(dim=1, keepdim=True)
    q = torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS)
    z = y * q * s["w_post"]
    gate = s["gate"].float().repeat_interleave(M // G, dim=0) if G else torch.ones_like(t)
    u = t * gate
    b = u * s["w_post"]
    dy = q * b - y * q ** 3 * (y * b).mean(dim=1, keepdim=True)
    out = [(s["alpha"] * t).to(dtype), dy.to(dtype), (u * y * q).sum(dim=0), (dh * r * p).sum(dim=0)]
    return out + [(t * z).view(G, M // G, D).sum(dim=1).to(dtype)] if G else out


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "norm":
        return _plain_norm(s)
    if op == "norm_grad":
        return _plain_norm_grad(s)
    if op == "quantize":
        out = []
        if c["layout"] != "columns":
            out += _pack(s["x"], c["block_rows"], c["format"])
        if c["layout"] != "rows":
            out += _pack(s["x"].t(), c["block_rows"], c["format"])
        return out
    dtype = TYPES[c["dtype"]]
    if op == "train":
        x, w, dy = s["x"], _rounded(s["w"], 128, "e4m3"), s["dy"]
        y = _rounded(x, 1, "e4m3") @ w.t()
        dx = _rounded(dy, 1, c["grad_format"]) @ w
        dw = _rounded(dy.t(), 1, c["grad_format"]) @ _rounded(x.t(), 1, "e4m3").t()
        return [y.to(dtype), dx.to(dtype), dw.to(dtype)]
    w = _value(s["qw"], s["sw"], 128)
    if op == "packed":
        return [(_value(s["qx"], s["sx"], 1) @ w.t()).to(dtype)]
    return [(_rounded(s["x"], 1, "e4m3") @ w[:, :c["K"]].t()).to(dtype)]


# ---- the calls a user makes -----------------------------------------------------------------------------------------------


def _own(s):
    import tab_amd
    from tab_amd import nn as tab_nn

    c = s["case"]
    op = c["op"]
    if op == "norm":
        M, D = c["M"], c["D"]
        output = {"none": tab_amd.NORM_NONE, "plain": tab_amd.NORM_PLAIN, "8bit": tab_amd.NORM_8BIT}[c["output"]]
        if c["block"]:
            return tab_amd.NormResidual(s["x"], s["y"], s["gate"], s["w_post"], s["w_pre"], s["alpha"], EPS, M, D, output)
        return tab_amd.Norm(s["x"], s["w_pre"], EPS, M, D, output)
    if op == "norm_grad":
        dx, dy, dgate, dw_post, dw_pre = tab_amd.NormResidualBackward(s["dr"], s["dh"], s["x"], s["y"], s["gate"], s["w_post"],
                                                                      s["w_pre"], s["alpha"], EPS, c["M"], c["D"])
        return [dx, dy, dw_post, dw_pre] + ([dgate] if dgate is not None else [])
    if op == "quantize":
        call = {"rows": tab_amd.Quantize8, "columns": tab_amd.Quantize8Transposed, "both": tab_amd.Quantize8Both}[c["layout"]]
        format = {"e4m3": tab_amd.E4M3, "e5m2": tab_amd.E5M2}[c["format"]]
        return call(s["x"], c["M"], c["K"], c["block_rows"], format)
    if op == "train":
        x, w = s["x"].detach().requires_grad_(), s["w"].detach().requires_grad_()
        y = tab_nn.linear8(x, w, grad_format={"e4m3": tab_amd.E4M3, "e5m2": tab_amd.E5M2}[c["grad_format"]])
        dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
        return [y.detach(), dx, dw]
    if op == "packed":
        return [tab_amd.Linear8Packed(s["qx"], s["sx"], s["qw"], s["sw"], c["M"], c["N"], c["K"], TYPES[c["dtype"]])]
    return [tab_amd.Linear8(s["x"], s["qw"], s["sw"], c["M"], c["N"], c["K"])]


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def _two_to(e):
    """2^e in fp64; from the exponent's bits, because the library's power is not exact on every device."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _packed8(x, block_rows, format):
    """The packed operand of x in fp64, block by block: the nearest 8-bit numbers (a multiple of the last place, half to
    even) of x over the scale, zeros past the last column, and the scales [blocks, rows or row blocks]."""
    _, largest, bits, smallest = FORMATS[format]
    numbers, scales = [], []
    for block in x.double().split(BLOCK, dim=1):
        amax = block.abs().amax(dim=1)
        if block_rows > 1:
            amax = torch.stack([a.max() for a in amax.split(block_rows)])
        # the exponent by comparison: the guess of the logarithm is at most one off
        e = torch.floor(torch.log2(torch.clamp(amax, min=2.0 ** -140) / largest)).clamp(min=-126)
        e = torch.where(amax > largest * _two_to(e), e + 1, e)
        e = torch.where((amax <= largest * _two_to(e - 1)) & (e > -126), e - 1, e)
        scales.append(_two_to(e))
        v = block / scales[-1][torch.arange(block.shape[0], device=x.device) // block_rows][:, None]
        _, ex = torch.frexp(v)
        last_place = _two_to(torch.clamp(ex - 1, min=smallest) - bits)
        numbers.append(torch.nn.functional.pad(torch.round(v / last_place) * last_place, (0, BLOCK - block.shape[1])))
    return torch.cat(numbers, dim=1), torch.stack(scales)


def _nearest8(x, block_rows, format):
    """What the packed operand of x stands for, in fp64."""
    q, scale = _packed8(x, block_rows, format)
    return _times_scale(q, scale, block_rows, x.shape[1])


def _times_scale(q, scale, block_rows, columns):
    rows = torch.arange(q.shape[0], device=q.device) // block_rows
    return q[:, :columns].double() * scale.t()[rows][:, torch.arange(columns, device=q.device) // BLOCK]


def _as_stored(q, s, block_rows, columns):
    """The numbers of a packed operand in fp64."""
    return _times_scale(q, _two_to(s.view(torch.uint8).double() - 127), block_rows, columns)


def _exact_norm(case, x, y, gate, w_post, w_pre, alpha):
    r = x
    if y is not None:
        z = y / torch.sqrt((y ** 2).mean(dim=1, keepdim=True) + EPS) * w_post
        if gate is not None:
            z = z * gate[torch.arange(case["M"], device=z.device) // (case["M"] // case["gates"])]
        r = alpha * x + z
    return r, (r / torch.sqrt((r ** 2).mean(dim=1, keepdim=True) + EPS) * w_pre if w_pre is not None else None)


def _chunks(case):
    """Rows at a time for fp64 copies of a large case, whole gate rows in each."""
    per_gate = case["M"] // max(1, case["gates"])
    step = max(1, (1 << 26) // case["D"])
    step = max(per_gate, step // per_gate * per_gate) if case["gates"] else step
    return [(m, min(case["M"], m + step)) for m in range(0, case["M"], step)]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        out = []
        for left_out, x in (("columns", s["x"]), ("rows", s["x"].t())):
            if case["layout"] != left_out:
                out += _packed8(x, case["block_rows"], case["format"])
        return out
    if op == "norm":
        w = {k: None if s[k] is None else s[k].double() for k in ("x", "y", "gate", "w_post", "w_pre")}
        r, h = _exact_norm(case, alpha=s["alpha"], **w)
        out = [r] if case["block"] else []
        if case["output"] != "none":
            out += [h] if case["output"] == "plain" else _packed8(h, 1, "e4m3")
        return out
    if op == "norm_grad":
        # R is an input here: H = norm(R) gives the gradient of R, R = alpha X + gate norm(Y) those of X, Y and the rest
        sums, rows = {}, {"dx": [], "dy": [], "dgate": []}
        per_gate = case["M"] // max(1, case["gates"])
        for a, b in _chunks(case):
            r, y = (s[k][a:b].double().requires_grad_() for k in ("x", "y"))
            w_post, w_pre = (s[k].double().requires_grad_() for k in ("w_post", "w_pre"))
            gate = s["gate"][a // per_gate:-(-b // per_gate)].double().requires_grad_() if case["gates"] else None
            part = {"M": b - a, "gates": 0 if gate is None else gate.shape[0]}
            _, h = _exact_norm(part, r, None, None, None, w_pre, 1.0)
            dr, dw_pre = torch.autograd.grad(h, (r, w_pre), s["dh"][a:b].double())
            t = dr + s["dr"][a:b].double()
            after, _ = _exact_norm(part, torch.zeros_like(y), y, gate, w_post, None, 1.0)
            wanted = [y, w_post] + ([gate] if gate is not None else [])
            got = torch.autograd.grad(after, wanted, t)
            rows["dx"].append(s["alpha"] * t)
            rows["dy"].append(got[0])
            if gate is not None:
                rows["dgate"].append(got[2])
            for k, v in (("dw_post", got[1]), ("dw_pre", dw_pre)):
                sums[k] = sums[k] + v if k in sums else v
        out = [torch.cat(rows["dx"]), torch.cat(rows["dy"]), sums["dw_post"], sums["dw_pre"]]
        return out + ([torch.cat(rows["dgate"])] if rows["dgate"] else [])
    if op == "train":
        x, w, dy = s["x"], _nearest8(s["w"], 128, "e4m3"), s["dy"]
        f = case["grad_format"]
        return [torch.matmul(_nearest8(x, 1, "e4m3"), w.t()), torch.matmul(_nearest8(dy, 1, f), w),
                torch.matmul(_nearest8(dy.t(), 1, f), _nearest8(x.t(), 1, "e4m3").t())]
    w = _as_stored(s["qw"], s["sw"], 128, case["K"])
    x = _as_stored(s["qx"], s["sx"], 1, case["K"]) if op == "packed" else _nearest8(s["x"], 1, "e4m3")
    return [torch.matmul(x, w.t())]
