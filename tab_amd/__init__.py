"""tab_amd - MI355X (gfx950) implementation of TAB's quantize + bitwise-conv operators.

Host-side mirror of the reference's operator interface (TAB_GPU.cpp:34-65): the same two
calls, positional argument lists, return tensors and error behaviour, on top of the C ABI
in include/tab_amd.h.  The calls go through the extension tab_amd._C (csrc/torch_binding.cpp), whose
checks, allocations and stream lookup take under 2 us where the same in Python took 13; PyTorch only
supplies device memory and the current stream.

    QW, BTN_W = Quantize(w, w_ths, bitwidth, KN, KH, KW, C)
    y = Conv2d(x, QW, x_ths, BTN_W, type, pad1, pad2, stride1, stride2, N, H, W, C, KN, KH, KW)
"""
import torch

from . import _capi

_lib = _capi.load()
TabError = _capi.TabError

from . import _C  # noqa: E402  (its errors are TabError)

TNN, TBN, BTN, BNN = 0, 1, 2, 3
DRF, RTN = 4, 5  # the types of the reference's CPU path only (TAB_CPU.cpp:332-383)


def version():
    return _lib.tab_version().decode()


def _call(fn, tensors, ints, *rest):
    """The call that the extension refused for an argument's type: whatever is no tensor where one belongs is named
    (CHECK_INPUT of the reference, TAB_GPU.cpp:7-9), everything else is made an int and the call repeated."""
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    return fn(*tensors.values(), *(int(v) for v in ints), *rest)


def packed_channels(C):
    return _lib.tab_packed_channels(int(C))


def operand_words(type, operand, C):
    """int64 words per pixel of the activation (operand 0) or per tap of the weight (operand 1)."""
    return _lib.tab_operand_words(int(type), int(operand), int(C))


def out_shape(H, W, KH, KW, pad1, pad2, stride1, stride2):
    """(OH, OW) by the reference's integer-division formula (TAB_GEMM.cu:354-357)."""
    return (_lib.tab_out_extent(H, pad1, KH, stride1), _lib.tab_out_extent(W, pad2, KW, stride2))


def Quantize(X, thresholds, bitwidth, N, H, W, C):
    """Ternarize (bitwidth 2) or binarize (bitwidth 1) NHWC fp32 data and pack 64 channels
    per int64 word.  Returns [QX, BTN]: QX int64 (N,H,W,PC,bitwidth), BTN int32 (N,)
    (TAB_GPU.cpp:53-58, TAB_GEMM.cu:250-322)."""
    try:
        return _C.Quantize(X, thresholds, bitwidth, N, H, W, C)
    except TypeError:
        return _call(_C.Quantize, {"X": X, "thresholds": thresholds}, (bitwidth, N, H, W, C))


def QuantizeActivation(X, thresholds, bitwidth, N, H, W, C, nchw=False):
    """QX of Quantize (or, with nchw, of QuantizeNCHW with X given as N, C, H, W) without the BTN vector: an
    activation's counts are read by nobody, and passing NULL for them to the C ABI skips the launches that
    produce them."""
    try:
        return _C.QuantizeActivation(X, thresholds, bitwidth, N, H, W, C, nchw)
    except TypeError:
        return _call(_C.QuantizeActivation, {"X": X, "thresholds": thresholds}, (bitwidth, N, H, W, C), bool(nchw))


def QuantizeNCHW(X, thresholds, bitwidth, N, C, H, W):
    """Quantize on an NCHW fp32 tensor (the layout the reference's CPU quantizers read, TAB_CPU.cpp:20-206, and
    the argument order of its CPU binding, TAB_CPU.cpp:621): returns [QX, BTN] exactly as
    Quantize(X.permute(0, 2, 3, 1), thresholds, bitwidth, N, H, W, C) would, without the transposed copy."""
    try:
        return _C.QuantizeNCHW(X, thresholds, bitwidth, N, C, H, W)
    except TypeError:
        return _call(_C.QuantizeNCHW, {"X": X, "thresholds": thresholds}, (bitwidth, N, C, H, W))


def QuantizeFormat(X, thresholds, type, N, H, W, C):
    """Packer of conv types 4 (DoReFa 2-bit levels; QX int64 (N,H,W,PC,2), plane 0 = weight-2 bit)
    and 5 (RTN 2-bit fields; QX int64 (N,H,W,ceil(C/32))), for activations and weights alike.  The
    layouts are the ones DRFGEMM_baseline / RTNGEMM_baseline read (TAB_CPU.cpp:332-383); the
    reference has no quantizer for them, the value rules (uniform step thresholds[n]; the
    ternarizer's compares) are this library's."""
    try:
        return _C.QuantizeFormat(X, thresholds, type, N, H, W, C)
    except TypeError:
        return _call(_C.QuantizeFormat, {"X": X, "thresholds": thresholds}, (type, N, H, W, C))


def Threshold(X, N, scale=0.7):
    """ths[n] = scale * mean(|X[n]|) per item (image or filter), fp32 (N,), computed on the
    device in one pass: the threshold rule the reference leaves to the caller (README.md:45).
    Reproducible from run to run; within 1e-5 relative of an fp64 reference."""
    try:
        return _C.Threshold(X, N, scale)
    except TypeError:
        return _call(_C.Threshold, {"X": X}, (N,), float(scale))


def Conv2d(X, QW, thresholds, btn, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW):
    """Quantize the NHWC fp32 activation on the fly (ternary for types 0/1, binary for 2/3; types 4
    and 5 of the CPU path through QuantizeFormat) and convolve it with the packed weights.  Returns fp32 shaped
    (N,KN,OH,OW) whose memory is ordered (n,oh,ow,kn), exactly as the reference's reshape
    of its GEMM result (TAB_GPU.cpp:34-42, TAB_GEMM.cu:325-527)."""
    try:
        return _C.Conv2d(X, QW, thresholds, btn, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW)
    except TypeError:
        return _call(_C.Conv2d, {"X": X, "QW": QW, "thresholds": thresholds, "btn": btn},
                     (type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW))


def conv2d_launches(X, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW):
    """Kernels one Conv2d call with these arguments enqueues: 1 (quantize and convolution in one launch) or 2."""
    return _lib.tab_conv2d_launches(X.data_ptr(), *(int(v) for v in (type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW)))


def static_scratch_bytes():
    """Size of the scratch array built into the library that Conv2dStatic packs the activation into."""
    return _lib.tab_static_scratch_bytes()


def Conv2dStatic(X, QW, thresholds, btn, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW, out=None):
    """Conv2d through tab_conv2d_static: the packed activation goes to the library's built-in device scratch
    (static_scratch_bytes() bytes per GPU) instead of a workspace tensor, so the C call allocates nothing.
    With `out` (fp32, N*OH*OW*KN elements) given, this wrapper allocates nothing either.  Calls that may
    overlap on one GPU race on the shared scratch."""
    try:
        return _C.Conv2dStatic(X, QW, thresholds, btn, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW, out)
    except TypeError:
        return _call(_C.Conv2dStatic, {"X": X, "QW": QW, "thresholds": thresholds, "btn": btn},
                     (type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW), out)


def Conv2dPacked(QX, QW, btn, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW):
    """Conv2d on an activation already packed by Quantize (bitwidth 2 for types 0/1,
    1 for types 2/3) or by QuantizeFormat (types 4/5): the pad + im2row + GEMM stages of
    TAB_GEMM.cu:447-509 only."""
    try:
        return _C.Conv2dPacked(QX, QW, btn, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW)
    except TypeError:
        return _call(_C.Conv2dPacked, {"QX": QX, "QW": QW, "btn": btn},
                     (type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW))


def Conv2dPackedOut(QX, QW, btn, type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW,
                    out_thresholds, out_bitwidth):
    """Conv2dPacked whose output is quantized and packed in the kernel's epilogue: returns QY int64
    (N, OH, OW, ceil(KN/64), out_bitwidth), equal bit for bit to
    Quantize(Conv2dPacked(...), out_thresholds, out_bitwidth, N, OH, OW, KN)[0] - the conv output's
    (n, oh, ow, kn) memory read as the next layer's NHWC activation - without the fp32 tensor ever
    being written.  out_thresholds: fp32 [>=N], one threshold per image."""
    args = (type, padding1, padding2, stride1, stride2, N, H, W, C, KN, KH, KW)
    try:
        return _C.Conv2dPackedOut(QX, QW, btn, *args, out_thresholds, out_bitwidth)
    except TypeError:
        if not isinstance(out_thresholds, torch.Tensor):
            raise TypeError("out_thresholds must be a torch.Tensor")
        return _call(_C.Conv2dPackedOut, {"QX": QX, "QW": QW, "btn": btn}, args, out_thresholds, int(out_bitwidth))


E4M3, E5M2 = 0, 1                              # 8-bit formats: largest numbers 448 and 57344
NORM_NONE, NORM_PLAIN, NORM_8BIT = 0, 1, 2     # what becomes of the norm before the next block


def blocks8(K):
    """Blocks of 128 in a row of K: a packed 8-bit operand of an R x K matrix is Q (R, 128 * blocks8(K)), zeros past K, and S, its
    power-of-two scales (E8M0), (blocks8(K), R) or, with blocks of 128 x 128, (blocks8(K), blocks8(R))."""
    return _lib.tab_blocks8(int(K))


def Quantize8(X, M, K, block_rows=1, format=E4M3):
    """Pack X (M x K; fp32, bf16 or fp16; contiguous or rows of a wider matrix) in 8-bit numbers with a power-of-two scale per block of
    block_rows x 128: the smallest one, from 2^-126, with which the block's largest finite magnitude fits the format.  A packed number is
    the nearest one to X.  NaN stays NaN, an infinity becomes NaN in E4M3 and stays one in E5M2.  Activations take blocks of one row,
    weights of 128.  Returns [Q, S]: Q float8_e4m3fn or float8_e5m2, S float8_e8m0fnu."""
    try:
        return _C.Quantize8(X, M, K, block_rows, format)
    except TypeError:
        return _call(_C.Quantize8, {"X": X}, (M, K, block_rows, format))


def Quantize8Transposed(X, M, K, block_rows=1, format=E4M3):
    """Quantize8 of X transposed (K x M): [QT, ST]; what the gradient of a weight multiplies."""
    try:
        return _C.Quantize8Transposed(X, M, K, block_rows, format)
    except TypeError:
        return _call(_C.Quantize8Transposed, {"X": X}, (M, K, block_rows, format))


def Quantize8Both(X, M, K, block_rows=1, format=E4M3):
    """Quantize8 and Quantize8Transposed from one reading of X: [Q, S, QT, ST]."""
    try:
        return _C.Quantize8Both(X, M, K, block_rows, format)
    except TypeError:
        return _call(_C.Quantize8Both, {"X": X}, (M, K, block_rows, format))


def Linear8(X, QW, SW, M, N, K):
    """X (M x K, quantized on the way as Quantize8 does) times the transpose of the packed weight (N x K, E4M3, blocks of 128 x 128 or of
    one row): Y (M, N) of X's type.  Sums in fp32; towards a 16-bit Y the products of eight neighbours in K are added with 13 bits below the
    largest of them (some 1.5e-5 of Y's size, below its rounding), towards an fp32 one with all of theirs: for those from a 16-bit X, quantize it
    and call Linear8Packed.  Up to 32 rows, their packed numbers at most 72 KB, are quantized and multiplied in one launch."""
    try:
        return _C.Linear8(X, QW, SW, M, N, K)
    except TypeError:
        return _call(_C.Linear8, {"X": X, "QW": QW, "SW": SW}, (M, N, K))


def Linear8Packed(QX, SX, QW, SW, M, N, K, out_dtype=torch.float32):
    """Linear8 on an activation that is already packed (E4M3 or E5M2, blocks of one row): Y (M, N) of out_dtype, the sums of an
    fp32 one with all their bits."""
    try:
        return _C.Linear8Packed(QX, SX, QW, SW, M, N, K, out_dtype)
    except TypeError:
        if not isinstance(out_dtype, torch.dtype):
            raise TypeError("out_dtype must be a torch.dtype")
        return _call(_C.Linear8Packed, {"QX": QX, "SX": SX, "QW": QW, "SW": SW}, (M, N, K), out_dtype)


def _call_norm(fn, required, optional, floats, ints):
    """As _call, where some tensors may be None."""
    for name, t in {**required, **optional}.items():
        if not isinstance(t, torch.Tensor) and not (t is None and name in optional):
            raise TypeError(f"{name} must be a torch.Tensor" + (" or None" if name in optional else ""))
    return fn(*required.values(), *optional.values(), *(float(v) for v in floats), *(int(v) for v in ints))


def Norm(X, w, eps, M, D, output=NORM_PLAIN):
    """H = X rms(X) w by rows, rms(v) = (mean v^2 + eps)^-1/2; w fp32 (D,) or None.  Returns [H] of X's type, or with NORM_8BIT the packed
    operand [QH, SH] that Linear8Packed takes."""
    try:
        return _C.Norm(X, w, eps, M, D, output)
    except TypeError:
        return _call_norm(_C.Norm, {"X": X}, {"w": w}, (eps,), (M, D, output))


def NormResidual(X, Y, gate, w_post, w_pre, alpha, eps, M, D, output=NORM_PLAIN):
    """The norm after a block, its gate, the scaled residual and the norm before the next block, in one pass:

        R = alpha X + gate * (Y rms(Y) w_post)        H = R rms(R) w_pre

    X, Y (M x D) of one type; gate (G, D), G a divisor of M, each row for M / G consecutive rows (a gate per channel, per sequence or per
    token), fp32 or X's type, or None; w_post, w_pre fp32 (D,) or None.  Returns [R, H], [R, QH, SH] with NORM_8BIT, [R] with NORM_NONE.
    D is at most 16384."""
    try:
        return _C.NormResidual(X, Y, gate, w_post, w_pre, alpha, eps, M, D, output)
    except TypeError:
        for name, t in {"X": X, "Y": Y}.items():
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
        return _call_norm(_C.NormResidual, {"X": X, "Y": Y}, {"gate": gate, "w_post": w_post, "w_pre": w_pre}, (alpha, eps), (M, D, output))


def NormResidualBackward(dR, dH, R, Y, gate, w_post, w_pre, alpha, eps, M, D):
    """Gradients of NormResidual from those of R and H (either may be None), R and Y: [dX, dY, dgate, dw_post, dw_pre], None for a gate or
    weight that is not there.  The sums over rows have a fixed order: the same call gives the same bits."""
    try:
        return _C.NormResidualBackward(dR, dH, R, Y, gate, w_post, w_pre, alpha, eps, M, D)
    except TypeError:
        fn = lambda R, Y, dR, dH, *rest: _C.NormResidualBackward(dR, dH, R, Y, *rest)  # noqa: E731
        return _call_norm(fn, {"R": R, "Y": Y}, {"dR": dR, "dH": dH, "gate": gate, "w_post": w_post, "w_pre": w_pre}, (alpha, eps), (M, D))


def NormBackward(dH, X, w, eps, M, D):
    """Gradients of Norm: [dX, dw]."""
    try:
        return _C.NormBackward(dH, X, w, eps, M, D)
    except TypeError:
        return _call_norm(_C.NormBackward, {"dH": dH, "X": X}, {"w": w}, (eps,), (M, D))


CONV_AUTO, CONV_MATRIX, CONV_POPCOUNT = 0, 1, 2


def set_conv_kernel(kernel=CONV_AUTO, tile=-1):
    """Pick the conv kernel (process-wide): CONV_AUTO, CONV_MATRIX (tile 0..11 or -1) or
    CONV_POPCOUNT (tile 0..2 or -1).  Every choice gives bit-identical outputs."""
    _capi.check(_lib, _lib.tab_set_conv_kernel(int(kernel), int(tile)))


# names of the reference's CPU module (TAB_CPU.cpp:636-639)
TAB_Quantize = Quantize
TAB_Conv2d = Conv2d

__all__ = ["Quantize", "QuantizeNCHW", "QuantizeActivation", "conv2d_launches", "QuantizeFormat", "Conv2d", "Conv2dStatic", "static_scratch_bytes", "Conv2dPacked", "Conv2dPackedOut", "Threshold", "TAB_Quantize", "TAB_Conv2d", "TabError",
           "packed_channels", "out_shape", "version", "TNN", "TBN", "BTN", "BNN", "set_conv_kernel",
           "CONV_AUTO", "CONV_MATRIX", "CONV_POPCOUNT",
           "Quantize8", "Quantize8Transposed", "Quantize8Both", "Linear8", "Linear8Packed", "blocks8", "E4M3", "E5M2",
           "Norm", "NormResidual", "NormResidualBackward", "NormBackward", "NORM_NONE", "NORM_PLAIN", "NORM_8BIT"]
