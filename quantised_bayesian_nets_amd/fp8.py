"""Linear layers in 8-bit floating point with one scale for each block of 128: the operand type, its quantiser, the product and the
stochastic layer built on them.

The int8 layers (layers.py) carry one calibrated scale per tensor; a block of 128 brings its own, so an input needs no calibration run and a
few large weights (mu + sigma eps has no bound) do not cost the others their precision.  As everywhere here the S Monte-Carlo samples of a
layer run in one launch, there is no CPU path, and nothing is differentiated: the engine evaluates.
"""
import torch
from torch.autograd import forward_ad

from . import _lib, layers, models_f32
from .layers import _MC

FLOAT_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # include/qbnn.h: QBNN_F32, QBNN_BF16, QBNN_F16
_F8 = 3                                                                    # QBNN_F8
BLOCK = 128


def padded_columns(columns):
    """Columns a row of e4m3 values occupies, and exponent bytes a row of blocks occupies."""
    blocks = -(-columns // BLOCK)
    return blocks * BLOCK, -(-blocks // 4) * 4


class F8Tensor:
    """`data` float8_e4m3fn [..., R, Kp] and `exponent` uint8 [..., Rb, Sp] (127 = 2^0) of a [..., R, columns] matrix: one exponent for each
    block of 128 columns and `block_rows` rows (1: activations, 128: weights).  Kp = columns up to a multiple of 128, zeros behind the
    last; Sp = blocks up to a multiple of 4; Rb = ceil(R / block_rows).  Values are data * 2^(exponent - 127)."""

    __slots__ = ("data", "exponent", "columns", "block_rows")

    def __init__(self, data, exponent, columns, block_rows):
        shape = data.shape
        kp, sp = padded_columns(columns)
        if block_rows != 1 and block_rows != BLOCK:
            raise ValueError("block_rows is 1 or 128")
        if data.dtype != torch.float8_e4m3fn or exponent.dtype != torch.uint8:
            raise TypeError("an F8Tensor holds float8_e4m3fn values and uint8 exponents")
        if len(shape) < 2 or columns < 1 or shape[-1] != kp or exponent.shape != (*shape[:-2], -(-shape[-2] // block_rows), sp):
            raise ValueError("data is [..., R, %d] and exponent [..., ceil(R / %d), %d] for %d columns" % (kp, block_rows, sp, columns))
        if data.device != exponent.device or not data.is_contiguous() or not exponent.is_contiguous():
            raise ValueError("data and exponent are contiguous, on one device")
        self.data, self.exponent, self.columns, self.block_rows = data, exponent, int(columns), int(block_rows)

    @property
    def shape(self):
        *lead, _ = self.data.shape
        return torch.Size((*lead, self.columns))

    @property
    def device(self):
        return self.data.device

    def reshape(self, *lead):
        """The same values with other leading dimensions ([*lead, R, columns])."""
        return F8Tensor(self.data.reshape(*lead, *self.data.shape[-2:]), self.exponent.reshape(*lead, *self.exponent.shape[-2:]), self.columns, self.block_rows)

    def dequantize(self, dtype=torch.float32):
        blocks, rows = self.data.shape[-1] // BLOCK, self.data.shape[-2]
        scale = (self.exponent[..., :blocks].to(torch.int32) << 23).view(torch.float32)
        scale = scale.repeat_interleave(self.block_rows, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)
        return (self.data.to(torch.float32) * scale)[..., :self.columns].to(dtype)


def _device(*tensors):
    """The device of a call's tensors (None entries left out).  Refuses what the engine would silently get wrong: tensors off the GPU, on several devices, or
    waiting for a gradient (backward, or a tangent in forward mode)."""
    dev, dual = None, forward_ad._current_level >= 0
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("qbnn layers run on an MI355X only (no CPU fallback)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("tensors on %s and %s in one call" % (dev, t.device))
        if t.requires_grad and torch.is_grad_enabled() or dual and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the engine evaluates only: call it under torch.no_grad() or with tensors that do not require a gradient")
    return dev


def _launch(key, dev, fn, *args):
    """fn(*args, stream) on the current stream of `dev`: a call's tensors decide the device, not the caller's current one."""
    if dev.index == torch.cuda.current_device() and layers.PROFILE is None:
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(dev.index)))
        return
    with torch.cuda.device(dev), layers.timed(key):
        _lib.check(fn(*args, _lib.current_stream()))


def _room(dev, *sizes):
    """One allocation for a call's workspaces (bytes): its tensor and each one's address, at multiples of 256."""
    at, places = 0, []
    for n in sizes:
        places.append(at)
        at += (n + 255) & ~255
    t = torch.empty(at, dtype=torch.uint8, device=dev)
    base = t.data_ptr()
    return t, [base + p for p in places]


def _float(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype not in FLOAT_TYPES:
        raise TypeError("%s is a float32, bfloat16 or float16 tensor" % name)
    return t


def quantize_fp8(x, block_rows=1):
    """x float [..., R, K] -> F8Tensor: each block's scale is the smallest power of two (>= 2^-126) that brings its largest finite magnitude
    to 448 or below (1 for zeros), values rounded to nearest even; what is not finite becomes NaN.  block_rows 1 for activations, 128 for weights."""
    _float(x, "x")
    if x.dim() < 2 or x.shape[-1] < 1:
        raise ValueError("x is [..., R, K] with K >= 1")
    if block_rows != 1 and block_rows != BLOCK:
        raise ValueError("block_rows is 1 or 128")
    dev = _device(x)
    lead, (R, K) = x.shape[:-2], x.shape[-2:]
    x = _rows(x)
    kp, sp = padded_columns(K)
    q = torch.empty((*lead, R, kp), dtype=torch.float8_e4m3fn, device=dev)
    e = torch.empty((*lead, -(-R // block_rows), sp), dtype=torch.uint8, device=dev)
    _launch("quantize_f8", dev, _lib.lib().qbnn_quantize_f8, x.data_ptr(), FLOAT_TYPES[x.dtype], (x.stride(0) if x.dim() == 3 else R * K), x.stride(-2), lead.numel(),
            R, K, block_rows, q.data_ptr(), e.data_ptr())
    return F8Tensor(q, e, K, block_rows)


def _rows(x):
    """x as the quantiser reads it: at most three dimensions with strides of their own, columns side by side (a copy where they are not)."""
    return x.contiguous() if x.stride(-1) != 1 and x.shape[-1] > 1 or x.dim() > 3 else x


def _bias(bias, shapes, what):
    if bias is None:
        return None
    if bias.dtype != torch.float32 or bias.shape not in shapes:
        raise ValueError("bias is float32 %s" % what)
    return bias.contiguous()


def linear_fp8(x, w, bias=None, relu=False, out_dtype=None):
    """act(x w^T + bias) for S Monte-Carlo samples in one launch.

    x: float, or an F8Tensor with block_rows 1, [S or 1, B, K] (or [B, K]); w: F8Tensor with block_rows 128, [S or 1, N, K] (or [N, K]);
    bias float32 [N] or [S, N].  A leading 1 is shared by the samples.  Returns [S, B, N] ([B, N] if both operands are matrices) in `out_dtype`
    (x's type; bfloat16 for an F8Tensor), or an F8Tensor (block_rows 1) with out_dtype torch.float8_e4m3fn.  Sums are taken in fp32;
    for a result of 16 or 8 bits of more than 16 rows a sample the matrix unit cuts the products of 8 neighbouring columns off 2^-13 below the largest of them first (1.3e-5 of the
    result's norm), for a float32 result or fewer rows nothing is cut, at half the matrix rate (of
    blocks with magnitudes below 2^-109 alone, what lies below 2^-133 is)."""
    if not isinstance(w, F8Tensor) or w.block_rows != BLOCK:
        raise TypeError("w is an F8Tensor with block_rows 128 (quantize_fp8(w, 128))")
    if isinstance(x, F8Tensor):
        if x.block_rows != 1:
            raise TypeError("x is a float tensor or an F8Tensor with block_rows 1")
        out_dtype = out_dtype or torch.bfloat16
    else:
        out_dtype = out_dtype or _float(x, "x").dtype
    xs, ws = x.shape, w.shape
    if len(xs) not in (2, 3) or len(ws) not in (2, 3) or xs[-1] != ws[-1]:
        raise ValueError("x [S or 1, B, K] and w [S or 1, N, K] do not fit: %s and %s" % (tuple(xs), tuple(ws)))
    B, K, N = xs[-2], xs[-1], ws[-2]
    sx, sw = (xs[0] if len(xs) == 3 else 1), (ws[0] if len(ws) == 3 else 1)
    S = sw if sx == 1 else sx
    if sw not in (1, S):
        raise ValueError("x holds %d samples, w %d" % (sx, sw))
    if N < 1:
        raise ValueError("w has no rows")
    if out_dtype not in FLOAT_TYPES and out_dtype != torch.float8_e4m3fn:
        raise TypeError("out_dtype is float32, bfloat16, float16 or float8_e4m3fn")
    bias = _bias(bias, ((N,), (S, N)), "[N] or [S, N]")
    held = isinstance(x, F8Tensor)
    dev = _device(x.data if held else x, w.data, bias)
    lead = (S, B) if len(xs) == 3 or len(ws) == 3 else (B,)
    ye = None
    if out_dtype == torch.float8_e4m3fn:
        np_, sp = padded_columns(N)
        y = torch.empty((*lead, np_), dtype=out_dtype, device=dev)
        ye = torch.empty((*lead, sp), dtype=torch.uint8, device=dev)
    else:
        y = torch.empty((*lead, N), dtype=out_dtype, device=dev)
    if S * B:
        kp, sp = padded_columns(K)
        xf = xf_ss = xf_rs = x_type = 0
        if held:
            xq, xe = x.data.data_ptr(), x.exponent.data_ptr()
        else:
            x = _rows(x)
            xf, xf_ss, xf_rs, x_type = x.data_ptr(), (x.stride(0) if len(xs) == 3 else 0), x.stride(-2), FLOAT_TYPES[x.dtype]
            room, (xq, xe) = _room(dev, sx * B * kp, sx * B * sp)
        _launch("linear_f8", dev, _lib.lib().qbnn_linear_f8_mc, _lib.F8_LINEAR.pack(
            xf, xf_ss, xf_rs, xq, xe, (B * kp if sx > 1 else 0), (B * sp if sx > 1 else 0),
            w.data.data_ptr(), w.exponent.data_ptr(), (N * kp if sw > 1 else 0), (-(-N // BLOCK) * sp if sw > 1 else 0),
            0 if bias is None else bias.data_ptr(), N if bias is not None and bias.dim() == 2 and S > 1 else 0,
            y.data_ptr(), 0 if ye is None else ye.data_ptr(), B, N, K, S, bool(relu), FLOAT_TYPES.get(out_dtype, _F8), x_type))
    return y if ye is None else F8Tensor(y, ye, N, 1)


class Linear(models_f32.Linear):
    """models_f32.Linear with its product in 8-bit floating point: the same parameters, state and noise stream (W_s = mu + eps_s softplus(rho)), each
    sample's weights quantised in blocks of 128 x 128, inputs in blocks of 128 as they come.  act: 0 none, 1 ReLU."""

    def forward(self, x, act=0, eps=None, out_dtype=None):
        """x float (or F8Tensor, block_rows 1) [S or 1, B, in_features] -> [S, B, out_features]."""
        if act not in (0, 1):
            raise ValueError("act is 0 or 1")
        w = quantize_fp8(self.sampled(x.device, eps).view(_MC.samples, self.out_features, self.in_features), BLOCK)
        y = linear_fp8(x, w, self._bias_dev, relu=act == 1, out_dtype=out_dtype)
        return y
