"""The 8-bit layers and the norms around a block in 64 bits, on the CPU, for the tests: the definitions, element by element."""
import torch

BLOCK = 128
EPS = 1e-6
# 8-bit formats by code: dtype, largest number, explicit mantissa bits, exponent of the smallest normal number
FORMATS = {0: (torch.float8_e4m3fn, 448.0, 3, -6), 1: (torch.float8_e5m2, 57344.0, 2, -14)}
# rounding of one number to a type of p significant bits: at most 2^-p of it, and half the smallest number
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def blocks(n):
    return -(-n // BLOCK)


def two_to(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)


def nearest8(v, format):
    """Nearest 8-bit numbers to v (fp64, magnitudes at most the largest), ties to even; infinities and NaN as documented."""
    _, _, bits, smallest = FORMATS[format]
    _, ex = torch.frexp(v)
    place = two_to(torch.clamp(ex - 1, min=smallest) - bits)
    out = torch.round(v / place) * place
    out = torch.where(torch.isinf(v), torch.full_like(v, float("nan")) if format == 0 else v, out)
    return torch.where(torch.isnan(v), v, out)


def quantize(x, block_rows, format):
    """Numbers (R, padded) and scale exponents (blocks, R or row blocks) of x, one block at a time."""
    R, K = x.shape
    x = x.double()
    largest = FORMATS[format][1]
    q = torch.zeros((R, blocks(K) * BLOCK), dtype=torch.float64)
    e = torch.zeros((blocks(K), -(-R // block_rows)), dtype=torch.int64)
    for kb in range(blocks(K)):
        v = x[:, kb * BLOCK:(kb + 1) * BLOCK]
        a = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dim=1)
        a = torch.stack([p.max() for p in a.split(block_rows)])
        _, top = torch.frexp(a / largest)          # a <= largest * 2^top, and a > largest * 2^(top - 1) unless it is equal
        exponent = torch.where(a <= largest * two_to(top - 1), top - 1, top)
        exponent = torch.where(a == 0, torch.full_like(exponent, -126), exponent.clamp(min=-126)).long()
        e[kb] = exponent
        q[:, kb * BLOCK:kb * BLOCK + v.shape[1]] = nearest8(v / two_to(exponent.repeat_interleave(block_rows)[:R])[:, None], format)
    return q, e


def value(q, e, block_rows):
    """What a packed operand stands for, (R, padded) fp64."""
    scale = two_to(e).t().repeat_interleave(block_rows, dim=0)[:q.shape[0]]
    return (q.double().view(q.shape[0], -1, BLOCK) * scale[:, :, None]).view(q.shape[0], -1)


def unpack(Q, S, block_rows):
    """value() of the library's tensors."""
    return value(Q.cpu().to(torch.float32).double(), S.cpu().view(torch.uint8).long() - 127, block_rows)


def pack(x, block_rows, format):
    """quantize() as the library's tensors, on the CPU."""
    q, e = quantize(x, block_rows, format)
    return q.float().to(FORMATS[format][0]), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def norm(x, y, gate, w_post, w_pre, alpha, eps):
    """(R, H) in fp64; gate as rows of M (or None)."""
    r = x.double()
    if y is not None:
        y = y.double()
        z = y / torch.sqrt((y * y).mean(dim=1, keepdim=True) + eps)
        z = z if w_post is None else z * w_post.double()
        r = alpha * r + (z if gate is None else z * gate.double())
    h = r / torch.sqrt((r * r).mean(dim=1, keepdim=True) + eps)
    return r, h if w_pre is None else h * w_pre.double()


def gate_rows(gate, M):
    return None if gate is None else gate.repeat_interleave(M // gate.shape[0], dim=0)
