"""Layer wrappers around the two operators: the caller the reference's demo notebook gestures
at (it imports torch.nn and autograd.Function, TAB Demo CUDA.ipynb cell 1, but ships none).
Inference only (the operators have no backward).  Beside them the 8-bit layers and the norms around a block (linear8,
norm_residual, Linear8, ResidualStack), which have one.

    layer = TABConv2d.from_float(weight_kn_c_kh_kw, conv_type=tab_amd.TNN, stride=1, padding=1)
    y = layer(x)            # x: (N, C, H, W) fp32 on the GPU -> (N, KN, OH, OW), logical NCHW
"""
import torch
from torch import nn

from . import _C, BNN, BTN, E4M3, NORM_8BIT, NORM_PLAIN, TBN, TNN, Linear8Packed, Quantize, Quantize8, Threshold

_ACT_BITS = {TNN: 2, TBN: 2, BTN: 1, BNN: 1}
_WEIGHT_BITS = {TNN: 2, TBN: 1, BTN: 2, BNN: 1}


def _pair(v):
    return (int(v), int(v)) if isinstance(v, int) else (int(v[0]), int(v[1]))


class TABConv2d(nn.Module):
    """2-D convolution with ternary/binary activations and weights.  Holds the packed weights
    (QW) and the BTN popcounts as buffers; the activation threshold is `act_scale * mean|x|` per
    image for ternary activations and 0 for binary ones.  `data_format` is the layout of the
    input and of the returned tensor: "NCHW" (PyTorch's; quantized directly from that layout, the
    result a permuted view of the operators' NHWC output) or "NHWC"."""

    def __init__(self, QW, BTN_W, conv_type, in_channels, out_channels, kernel_size, stride=1, padding=0,
                 act_scale=0.7, data_format="NCHW"):
        super().__init__()
        if conv_type not in _ACT_BITS:
            raise ValueError("conv_type must be 0 (TNN), 1 (TBN), 2 (BTN) or 3 (BNN)")
        if data_format not in ("NCHW", "NHWC"):
            raise ValueError("data_format must be 'NCHW' or 'NHWC'")
        self.conv_type = int(conv_type)
        self.in_channels, self.out_channels = int(in_channels), int(out_channels)
        self.kernel_size, self.stride, self.padding = _pair(kernel_size), _pair(stride), _pair(padding)
        self.act_scale, self.data_format = float(act_scale), data_format
        self.register_buffer("QW", QW)
        self.register_buffer("BTN_W", BTN_W)

    @classmethod
    def from_float(cls, weight, conv_type, stride=1, padding=0, weight_scale=0.7, act_scale=0.7, data_format="NCHW"):
        """Quantize an fp32 weight of PyTorch's shape (KN, C, KH, KW) on the GPU: ternary weights
        use the threshold weight_scale * mean|w| per filter, binary weights the sign."""
        KN, C, KH, KW = weight.shape
        w = weight.detach().to(torch.float32).permute(0, 2, 3, 1).contiguous().cuda()  # (KN,KH,KW,C)
        bits = _WEIGHT_BITS[conv_type]
        ths = Threshold(w, KN, weight_scale) if bits == 2 else torch.zeros(KN, device=w.device)
        QW, BTN_W = Quantize(w, ths, bits, KN, KH, KW, C)
        return cls(QW, BTN_W, conv_type, C, KN, (KH, KW), stride, padding, act_scale, data_format)

    def forward(self, x):
        # thresholds, quantizer (straight from NCHW where the input is) and convolution; the operator's output is
        # (n, oh, ow, kn) in memory (TAB_GEMM.cu:526)
        return _C.layer_forward(self, x, self.data_format == "NCHW")

    def extra_repr(self):
        names = {TNN: "TNN", TBN: "TBN", BTN: "BTN", BNN: "BNN"}
        return (f"{self.in_channels}, {self.out_channels}, kernel_size={self.kernel_size}, stride={self.stride}, "
                f"padding={self.padding}, type={names[self.conv_type]}, data_format={self.data_format}")


_PLAIN_CONV = _C.plain_class(TABConv2d)


class TABLinear(nn.Module):
    """Fully connected layer as a 1x1 convolution on a 1x1 image ("FC equals to 1x1 conv",
    TAB_CPU.cpp:487-488).  Input (N, in_features), output (N, out_features)."""

    def __init__(self, conv):
        super().__init__()
        self.conv = conv

    @classmethod
    def from_float(cls, weight, conv_type, weight_scale=0.7, act_scale=0.7):
        out_features, in_features = weight.shape
        conv = TABConv2d.from_float(weight.reshape(out_features, in_features, 1, 1), conv_type, 1, 0,
                                    weight_scale, act_scale, data_format="NHWC")
        return cls(conv)

    def forward(self, x):
        y = _C.linear_forward(self, _PLAIN_CONV, x)
        if y is None:  # calling the inner layer is more than its forward, it has another layout, or x is a tracer's proxy
            N, F = x.shape
            y = self.conv(x.reshape(N, 1, 1, F)).reshape(N, self.conv.out_channels)
        return y


class TABPackedChain(nn.Module):
    """A stack of TABConv2d layers run packed-in / packed-out: the input is quantized once, every
    layer but the last writes its output already thresholded and packed for the next layer (no fp32
    activation between layers), the last one returns fp32.  A layer's output channels must be the
    next layer's input channels.

    The threshold applied to a layer's output is the next layer's activation threshold: 0 when the
    next layer takes binary activations (types BTN, BNN) - then the chain returns exactly what
    calling the layers one after the other returns - and, when it takes ternary activations, the
    calibrated constant given in `ternary_thresholds[i]` for layer i+1 (the per-image
    `act_scale * mean|y|` of an unchained TABConv2d needs the fp32 tensor this class avoids)."""

    def __init__(self, layers, ternary_thresholds=None, data_format="NCHW"):
        super().__init__()
        self.layers = nn.ModuleList(layers)
        if not self.layers:
            raise ValueError("at least one layer")
        for a, b in zip(self.layers[:-1], self.layers[1:]):
            if a.out_channels != b.in_channels:
                raise ValueError(f"{a.out_channels} output channels feed a layer with {b.in_channels} input channels")
        self.ternary_thresholds = dict(ternary_thresholds or {})
        for i, layer in enumerate(self.layers[1:], start=1):
            if _ACT_BITS[layer.conv_type] == 2 and i not in self.ternary_thresholds:
                raise ValueError(f"layer {i} takes ternary activations: give ternary_thresholds[{i}]")
        if data_format not in ("NCHW", "NHWC"):
            raise ValueError("data_format must be 'NCHW' or 'NHWC'")
        self.data_format = data_format

    def forward(self, x):
        return _C.chain_forward(list(self.layers), self.ternary_thresholds, self.data_format == "NCHW", x)


def linear8(x, w, grad_format=E4M3):
    """x (..., K) times the transpose of w (N, K) in 8-bit numbers with a scale per block of 128: y (..., N) of x's type.  Differentiable
    in x and w: dx = dy w and dw = dy^T x are products of the same kind, dy packed in grad_format (E5M2 where its range needs more than
    a scale per block of 128 gives) along its rows and its columns.  w is packed anew in every call: for weights that stay, see Linear8.
    The sums are those of tab_amd.Linear8Packed towards x's type.  Second derivatives and forward mode are errors."""
    if not isinstance(x, torch.Tensor) or not isinstance(w, torch.Tensor):
        raise TypeError("x and w must be torch.Tensors")
    return _C.linear8(x, w, int(grad_format))


def norm_residual(x, y=None, gate=None, w_post=None, w_pre=None, alpha=1.0, eps=1e-6, output=NORM_PLAIN):
    """tab_amd.NormResidual (with a block's output y) or tab_amd.Norm (without) on tensors (..., D), differentiable in every tensor:
    [R, H], [R] with output=NORM_NONE, [H] without y.  output=NORM_8BIT gives H packed, for inference.  A row of the gate
    holds for consecutive rows of x, so (B, 1, D) or (B, D) is a gate for each sequence of x (B, S, D).  Gate and weights need not be contiguous;
    those of 16 bits, as a converted module has, are taken as fp32 (a gate of x's type as it is)."""
    return _C.norm_residual(x, y, gate, w_post, w_pre, float(alpha), float(eps), int(output))


class Linear8(nn.Module):
    """Fully connected layer on 8-bit numbers, for the layers of a low-bit network that keep more than two bits.  Holds the packed weight
    (QW, SW) as buffers.  Input (..., in_features) of fp32, bf16 or fp16, or the pair (QH, SH) that a norm packed (then `rows` x out_features
    of out_dtype); output (..., out_features)."""

    def __init__(self, QW, SW, in_features, out_features, out_dtype=torch.float32):
        super().__init__()
        self.in_features, self.out_features, self.out_dtype = int(in_features), int(out_features), out_dtype
        self.register_buffer("QW", QW)
        self.register_buffer("SW", SW)

    @classmethod
    def from_float(cls, weight, out_dtype=torch.float32):
        """Pack a weight of PyTorch's shape (out_features, in_features) on the GPU."""
        N, K = weight.shape
        QW, SW = Quantize8(weight.detach().cuda().contiguous(), N, K, 128)
        return cls(QW, SW, K, N, out_dtype)

    def _apply(self, fn, recurse=True):
        """What moves or converts the module moves the packed weight, whose types are its format: fn sees their bytes, and a conversion to another type leaves
        them as they are."""
        def bytes_alone(t):
            if t.dtype not in (torch.float8_e4m3fn, torch.float8_e8m0fnu):
                return fn(t)
            moved = fn(t.view(torch.uint8))
            return moved.view(t.dtype) if moved.dtype == torch.uint8 else t.to(moved.device)

        return super()._apply(bytes_alone, recurse)

    def forward(self, x):
        if isinstance(x, (tuple, list)):
            QX, SX = x
            return Linear8Packed(QX, SX, self.QW, self.SW, QX.shape[0], self.out_features, self.in_features, self.out_dtype)
        return _C.linear8_packed_weight(x, self.QW, self.SW, self.out_features, self.in_features)

    def extra_repr(self):
        return f"{self.in_features}, {self.out_features}"


class _NoGradient(torch.autograd.Function):
    """y, made from h by a layer without a backward pass: a gradient on its way to h ends in an error."""

    @staticmethod
    def forward(ctx, y, h):
        return y

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("TABConv2d, TABLinear and TABPackedChain have no gradient: give a block that has one, detach what comes before it, "
                           "or run under torch.no_grad()")


class ResidualStack(nn.Module):
    """A residual stream through a list of blocks, each between two norms: with x_0 = x and the first norm of x_0 as the first block's input h_0,

        y_i = block_i(h_i),   x_{i+1} = alpha x_i + gate_i * norm(y_i; w_post_i),   h_{i+1} = norm(x_{i+1}; w_pre_{i+1})

    Every block is followed by one NormResidual launch (norm, gate, residual, next norm); the output is the last norm, so that a head can
    follow.  Blocks map (rows, D) to (rows, D): TABLinear layers, Linear8, or functions of linear8 in training; TABLinear's input is fp32 also
    in a stream of 16 bits.  With a Linear8 as the next block and no gradient wanted, the norm packs its output for it.  `gates` of a call: one
    (G, D) tensor or None a block, in place of the learned gate per channel.  TABLinear layers have no backward pass: a gradient that would
    have to go through one is an error."""

    def __init__(self, blocks, D, alpha=1.0, eps=1e-6, gate_init=1.0, head=None):
        super().__init__()
        self.blocks = nn.ModuleList(blocks)
        if not self.blocks:
            raise ValueError("at least one block")
        self.head = head
        self.D, self.alpha, self.eps = int(D), float(alpha), float(eps)
        n = len(self.blocks)
        self.w_pre = nn.ParameterList([nn.Parameter(torch.ones(D)) for _ in range(n + 1)])
        self.w_post = nn.ParameterList([nn.Parameter(torch.ones(D)) for _ in range(n)])
        self.gate = nn.ParameterList([nn.Parameter(torch.full((1, D), float(gate_init))) for _ in range(n)])

    def _output(self, i):
        """How the norm before block i (or before the head) leaves its result."""
        follower = self.blocks[i] if i < len(self.blocks) else self.head
        return NORM_8BIT if isinstance(follower, Linear8) and not torch.is_grad_enabled() else NORM_PLAIN

    @staticmethod
    def _input(layer, h):
        return h if len(h) > 1 else h[0].float() if isinstance(layer, TABLinear) else h[0]

    def forward(self, x, gates=None):
        if gates is not None and len(gates) != len(self.blocks):
            raise ValueError(f"{len(gates)} gates for {len(self.blocks)} blocks")
        for gate in () if gates is None else gates:
            if gate is not None:
                _C.check_gate(gate, x.shape)
        shape, x = x.shape, x.reshape(-1, x.shape[-1])
        h = norm_residual(x, w_pre=self.w_pre[0], eps=self.eps, output=self._output(0))
        for i, block in enumerate(self.blocks):
            y = block(self._input(block, h))
            if h[0].requires_grad and not y.requires_grad and torch.is_grad_enabled() and any(
                    isinstance(m, (TABConv2d, TABLinear, TABPackedChain)) for m in block.modules()):
                y = _NoGradient.apply(y, h[0])
            gate = self.gate[i] if gates is None or gates[i] is None else gates[i]
            x, *h = norm_residual(x, y.to(x.dtype), gate, self.w_post[i], self.w_pre[i + 1], self.alpha, self.eps, self._output(i + 1))
        out = h[0] if self.head is None else self.head(self._input(self.head, h))
        return out.reshape(*shape[:-1], out.shape[-1])
