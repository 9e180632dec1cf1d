"""Products of microscaled (MX) matrices: low-bit operands with shared power-of-two scales on the tensor cores.

The exact products of this package split float64 operands into INT8 planes with one power of two per row and column;
these operators do the same to a model's operands with one power of two per 32 elements, and keep the split operand:

    Wq = mx_quantize(W, "e2m1")                      # W (n, k): 4-bit codes, blocks along k; once
    Xq, h = mx_rms_norm(x, gain, residual=h)         # norm of x + h straight into an 8-bit operand, and the new h
    Y = mx_matmul(Xq, Wq)                            # (m, n) = Xq Wq^T, bf16
    Y = mx_grouped_matmul(Xq, Eq, ends)              # rows ends[e-1] .. ends[e] with expert e of Eq (experts, n, k)
    y = mx_linear(x, W)                              # differentiable: its three products are MX products

A number is code x 2^(s - 127): an element of 4 bits ("e2m1": 0, .5, 1, 1.5, 2, 3, 4, 6) or 8 bits ("e4m3", up to 448)
and one scale byte s per block of 32 along the contracted axis (255: the block held a NaN or an infinite value, and
everything it touches is NaN).  Any sizes; the operands are laid out for the tensor cores once, by the quantisation.

All calls are enqueued on the current stream of the operand's device and may be captured in a CUDA graph (after one
eager call on that device).  A product whose bounded waits ran out leaves a flag that ``mx_check_errors`` raises.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import OzkError, check

FORMATS = {"e2m1": 0, "e4m3": 1}
RULES = {"floor": 0, "ceil": 1}
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
BLOCK = 32
TILE = 128
TILE_BYTES = 512
MAX_GROUPS = 1024
KMAX = 1 << 28
_INT_MAX = 2 ** 31 - 1

_error_words = {}                # device index -> int32 word that the products' launches OR their flags into


def _padded(k: int) -> int:
    return (k + TILE - 1) // TILE * TILE


class _On:
    """Makes ``device`` (an index) current for a launch if it is not, and gives its current stream's handle."""

    __slots__ = ("device", "before")

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.device:
            torch.cuda.set_device(self.device)
        return torch._C._cuda_getCurrentRawStream(self.device)

    def __exit__(self, *_):
        if self.before != self.device:
            torch.cuda.set_device(self.before)


def _error_word(device: int):
    w = _error_words.get(device)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            raise OzkError("the first MX product on a device allocates its error word: make one call before capturing")
        w = _error_words[device] = torch.zeros(1, dtype=torch.int32, device=f"cuda:{device}")
        torch.cuda.synchronize(device)               # products on any stream may use it from here on
    return w.data_ptr()


def mx_check_errors(device=None) -> None:
    """Raise OzkError if a product launched on ``device`` (default: the current one) gave up a wait since the last
    check; synchronises the device."""
    device = torch.cuda.current_device() if device is None else torch.device(device).index
    w = _error_words.get(device)
    if w is None:
        return
    torch.cuda.synchronize(device)
    word = int(w.item())
    if word:
        w.zero_()
        raise OzkError(f"device error flag {word:#x} raised by an MX product (a bounded wait ran out); the results of "
                       "the calls since the last check are invalid")


def _format(fmt):
    code = FORMATS.get(fmt)
    if code is None:
        raise ValueError(f"unknown element format {fmt!r}: one of {', '.join(FORMATS)}")
    return code


def _rule(rule):
    code = RULES.get(rule)
    if code is None:
        raise ValueError(f"unknown scale rule {rule!r}: one of {', '.join(RULES)}")
    return code


def _dtype(dtype, what):
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what}: float32, float16 or bfloat16 required, not {dtype}")
    return code


def _tensor(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: CUDA tensor required (there is no CPU path)")
    return _dtype(t.dtype, what)


class MXMatrix:
    """An operand of the MX products: ``rows`` vectors of length ``k`` (times ``groups``, for experts; None: a plain
    matrix) in element format ``fmt``.  Made by ``mx_quantize``, ``mx_rms_norm`` or ``MXMatrix.from_codes``."""

    __slots__ = ("fmt", "groups", "rows", "k", "device", "_fmt", "_buffer", "_code_ptr", "_scale_ptr", "_code_bytes")

    def __init__(self, fmt, groups, rows, k, device: int):
        """An operand with uninitialised contents."""
        self._fmt = _format(fmt)
        g = 1 if groups is None else groups
        if k < 1 or k > KMAX:
            raise ValueError(f"contracted axis of length {k}: 1 to {KMAX} required")
        if rows > _INT_MAX or g > _INT_MAX or g * -(-rows // TILE) * (_padded(k) // TILE) > _INT_MAX:
            raise ValueError(f"operand of {g} x {rows} x {k} elements is too large")
        self.fmt, self.groups, self.rows, self.k, self.device = fmt, groups, rows, k, device
        kp = _padded(k)
        self._code_bytes = g * rows * (kp // 2 if self._fmt == 0 else kp)
        scale_bytes = g * -(-rows // TILE) * (kp // TILE) * TILE_BYTES
        # one allocation: the codes (a multiple of 64 bytes), then the scales
        self._buffer = torch.empty(self._code_bytes + scale_bytes, dtype=torch.uint8, device=torch.device("cuda", device))
        self._code_ptr = self._buffer.data_ptr()
        self._scale_ptr = self._code_ptr + self._code_bytes

    @property
    def shape(self):
        return (self.rows, self.k) if self.groups is None else (self.groups, self.rows, self.k)

    def __repr__(self):
        return f"MXMatrix({self.fmt}, shape={self.shape}, device='cuda:{self.device}')"

    @property
    def _g(self):
        return 1 if self.groups is None else self.groups

    def codes(self):
        """The element codes as uint8 (..., rows, ceil(k / 2)) for e2m1 (two a byte, the even one in the lower half)
        or (..., rows, k) for e4m3: a copy in the order in which checkpoints store them."""
        per = (self.k + 1) // 2 if self._fmt == 0 else self.k
        pitch = _padded(self.k) // (2 if self._fmt == 0 else 1)
        c = self._buffer[:self._code_bytes].view(self._g, self.rows, pitch)[..., :per].contiguous()
        return c if self.groups is not None else c[0]

    def scales(self):
        """The scale bytes as uint8 (..., rows, ceil(k / 32)): a copy in the order in which checkpoints store them."""
        rt, kt = -(-self.rows // TILE), _padded(self.k) // TILE
        s = self._buffer[self._code_bytes:].view(self._g, rt, kt, 32, 4, 4)
        s = s.permute(0, 1, 4, 3, 2, 5).reshape(self._g, rt * TILE, kt * 4)
        s = s[:, :self.rows, :-(-self.k // BLOCK)].contiguous()
        return s if self.groups is not None else s[0]

    @classmethod
    def from_codes(cls, codes, scales, fmt, k=None):
        """An operand from element codes and scale bytes as ``codes()`` and ``scales()`` give them (a checkpoint's
        weights); ``k`` is needed where an odd number of 4-bit codes ends in half a byte."""
        code = _format(fmt)
        for t, what in ((codes, "codes"), (scales, "scales")):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.uint8 or t.dim() not in (2, 3):
                raise ValueError(f"{what}: uint8 CUDA tensor of 2 or 3 axes required")
        per = codes.shape[-1]
        if k is None:
            k = 2 * per if code == 0 else per
        if per != ((k + 1) // 2 if code == 0 else k):
            raise ValueError(f"{per} bytes of {fmt} codes a row do not hold {k} elements")
        if tuple(scales.shape) != (*codes.shape[:-1], -(-k // BLOCK)) or scales.device != codes.device:
            raise ValueError(f"scales of shape {tuple(codes.shape[:-1])} + ({-(-k // BLOCK)},) on the codes' device "
                             f"required, not {tuple(scales.shape)}")
        groups = codes.shape[0] if codes.dim() == 3 else None
        rows = codes.shape[-2]
        out = cls(fmt, groups, rows, k, codes.device.index)
        g = out._g
        c = out._buffer[:out._code_bytes].view(g, rows, _padded(k) // (2 if code == 0 else 1))
        c[..., :per] = codes.reshape(g, rows, per)
        if code == 0 and k % 2:
            c[..., per - 1] &= 15
        c[..., per:] = 0
        rt, kt = -(-rows // TILE), _padded(k) // TILE
        s = torch.nn.functional.pad(scales.reshape(g, rows, scales.shape[-1]), (0, 4 * kt - scales.shape[-1], 0, rt * TILE - rows))
        out._buffer[out._code_bytes:].view(g, rt, kt, 32, 4, 4).copy_(
            s.view(g, rt, 4, 32, kt, 4).permute(0, 1, 4, 3, 2, 5))
        return out

    def dequantize(self, dtype=torch.bfloat16):
        """The numbers the operand stands for, as a contiguous tensor (bfloat16 and float32 hold them exactly while
        their scales are ordinary)."""
        d = _dtype(dtype, "dequantize")
        out = torch.empty(self.shape, dtype=dtype, device=self._buffer.device)
        if self.rows and self._g:
            with _On(self.device) as stream:
                check(_lib.lib().ozk_mx_dequantize(self._code_ptr, self._scale_ptr, self._fmt, self._g, self.rows,
                                                   self.k, out.data_ptr(), d, stream), "ozk_mx_dequantize")
        return out


def mx_quantize(x, fmt="e2m1", axis=-1, rule="floor"):
    """The MX operand of ``x`` with blocks of 32 along ``axis``, the axis that the product contracts.

    x: float32, float16 or bfloat16 CUDA tensor of any strides, (rows, k) or, for experts, (groups, rows, k); with the
    other of the last two axes given, its vectors are the columns: a right operand (k, n) is quantised with axis=-2.
    rule: the scale puts the block's largest value at the format's top exponent ("floor", which saturates what lies
    above the format's largest number) or one higher where it would saturate ("ceil").  Values go to the nearest
    number, ties to the even code."""
    d = _tensor(x, "x")
    code, up = _format(fmt), _rule(rule)
    dim = x.dim()
    if dim not in (2, 3):
        raise ValueError(f"x: 2 or 3 axes required, not {dim}")
    if not -2 <= axis < dim:
        raise ValueError(f"axis {axis} out of range for {dim} axes")
    at = axis % dim
    if at < dim - 2:
        raise ValueError("the groups of x cannot be contracted: axis is one of the last two")
    other = 2 * dim - 3 - at
    shape, stride = x.shape, x.stride()
    rows, k = shape[other], shape[at]
    groups = shape[0] if dim == 3 else None
    device = x.device.index
    out = MXMatrix(fmt, groups, rows, k, device)
    if rows and groups != 0:
        with _On(device) as stream:
            check(_lib.lib().ozk_mx_quantize(x.data_ptr(), d, groups or 1, rows, k, stride[0] if dim == 3 else 0,
                                             stride[other], stride[at], code, up, out._code_ptr, out._scale_ptr,
                                             stream), "ozk_mx_quantize")
    return out


def _operands(A, B):
    if not isinstance(A, MXMatrix) or not isinstance(B, MXMatrix):
        raise ValueError("A and B: MXMatrix required (see mx_quantize)")
    if A.device != B.device:
        raise ValueError(f"A on cuda:{A.device}, B on cuda:{B.device}: one device required")
    if A.k != B.k:
        raise ValueError(f"contracted axes differ: {A.k} and {B.k}")
    if A.groups is not None:
        raise ValueError("A: a plain matrix required, not groups")


def _result(C, rows, cols, dtype, device):
    """The output tensor, its dtype code and row stride."""
    if C is None:
        d = _dtype(dtype, "dtype")
        return torch.empty((rows, cols), dtype=dtype, device=torch.device("cuda", device)), d, max(cols, 1)
    d = _tensor(C, "C")
    if C.device.index != device or tuple(C.shape) != (rows, cols) or (cols > 1 and C.stride(1) != 1) \
            or (rows > 1 and C.stride(0) < cols):
        raise ValueError(f"C: ({rows}, {cols}) on cuda:{device} with contiguous, separate rows required")
    return C, d, C.stride(0) if rows > 1 else max(cols, 1)


def mx_matmul(A, B, C=None, dtype=torch.bfloat16):
    """C = A B^T for MX operands A (m, k) and B (n, k) of any formats: sums in FP32, one rounding to ``dtype`` (or to
    the type of a given ``C``, whose rows may be strided)."""
    _operands(A, B)
    if B.groups is not None:
        raise ValueError("B: a plain matrix required (see mx_grouped_matmul)")
    C, d, ldc = _result(C, A.rows, B.rows, dtype, A.device)
    if A.rows and B.rows:
        with _On(A.device) as stream:
            check(_lib.lib().ozk_mx_gemm(A._code_ptr, A._scale_ptr, A._fmt, B._code_ptr, B._scale_ptr, B._fmt, A.rows,
                                         B.rows, A.k, C.data_ptr(), ldc, d, _error_word(A.device), stream),
                  "ozk_mx_gemm")
    return C


def mx_grouped_matmul(A, B, ends, C=None, dtype=torch.bfloat16):
    """Rows ends[g - 1] .. ends[g] - 1 of C (from row 0 for g = 0) = the same rows of A times group g of B transposed:
    the products of tokens sorted by expert.  A (rows, k), B (groups, n, k); ends: int32 CUDA tensor of the groups'
    ends, ascending, read on the device (so routing needs no host synchronisation); a group may be empty.  An end below
    the one before it, or beyond the rows, counts as the nearest in order.  Rows behind the last end are zero, or left
    as they were in a given ``C``."""
    _operands(A, B)
    if B.groups is None:
        raise ValueError("B: groups (experts, n, k) required")
    if not 1 <= B.groups <= MAX_GROUPS:
        raise ValueError(f"{B.groups} groups: 1 to {MAX_GROUPS} required")
    if not isinstance(ends, torch.Tensor) or ends.dtype != torch.int32 or ends.device != A._buffer.device \
            or tuple(ends.shape) != (B.groups,) or not ends.is_contiguous():
        raise ValueError(f"ends: contiguous int32 tensor of {B.groups} ends on cuda:{A.device} required")
    fill = C is None
    C, d, ldc = _result(C, A.rows, B.rows, dtype, A.device)
    if A.rows and B.rows:
        with _On(A.device) as stream:
            check(_lib.lib().ozk_mx_grouped_gemm(A._code_ptr, A._scale_ptr, A._fmt, B._code_ptr, B._scale_ptr, B._fmt,
                                                 A.rows, B.rows, A.k, B.groups, ends.data_ptr(), int(fill),
                                                 C.data_ptr(), ldc, d, _error_word(A.device), stream),
                  "ozk_mx_grouped_gemm")
    return C


def mx_rms_norm(x, weight, residual=None, eps=1e-6, fmt="e4m3", rule="floor"):
    """Root-mean-square norm into an MX operand: t = x + residual, y = t / sqrt(mean(t^2) + eps) * weight over the last
    axis, in FP32 from the loads to the codes.  Returns (y as MXMatrix (rows, d) with the leading axes of x as rows, t
    rounded to the type of x and in its shape, or None without a residual)."""
    d = _tensor(x, "x")
    code, up = _format(fmt), _rule(rule)
    if x.dim() < 1:
        raise ValueError("x: at least one axis required")
    n = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.device != x.device or tuple(weight.shape) != (n,) \
            or not (weight.dtype == x.dtype or weight.dtype == torch.float32) or not weight.is_contiguous():
        raise ValueError(f"weight: contiguous ({n},) tensor of x's type or float32 on its device required")
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"eps {eps}: a positive number required")
    x2 = x.reshape(-1, n) if n else x.reshape(0, 0)
    if n and x2.stride(1) != 1 and n > 1:
        x2 = x2.contiguous()
    r2 = None
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.shape != x.shape or residual.dtype != x.dtype \
                or residual.device != x.device:
            raise ValueError("residual: a tensor of x's shape, type and device required")
        r2 = residual.reshape(-1, n) if n else x2
        if n > 1 and r2.stride(1) != 1:
            r2 = r2.contiguous()
    rows, device = x2.shape[0], x.device.index
    out = MXMatrix(fmt, None, rows, n, device)
    total = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if rows:
        with _On(device) as stream:
            check(_lib.lib().ozk_mx_rms_norm(x2.data_ptr(), 0 if r2 is None else r2.data_ptr(), weight.data_ptr(), d,
                                             int(weight.dtype == torch.float32), rows, n, x2.stride(0),
                                             0 if r2 is None else r2.stride(0), eps, code, up,
                                             0 if total is None else total.data_ptr(), out._code_ptr, out._scale_ptr,
                                             stream), "ozk_mx_rms_norm")
    return out, total


class _MXLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, fmt, rule):
        x2 = x.reshape(-1, x.shape[-1])
        ctx.save_for_backward(x2, weight)
        ctx.how = (fmt, rule)
        ctx.x_shape = x.shape
        y = mx_matmul(mx_quantize(x2, fmt, rule=rule), mx_quantize(weight, fmt, rule=rule), dtype=x.dtype)
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        fmt, rule = ctx.how
        dy = dy.reshape(-1, dy.shape[-1])
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = mx_matmul(mx_quantize(dy, fmt, rule=rule), mx_quantize(weight, fmt, axis=0, rule=rule), dtype=x.dtype)
            dx = dx.view(ctx.x_shape)
        if ctx.needs_input_grad[1]:
            if dy.shape[0]:
                dw = mx_matmul(mx_quantize(dy, fmt, axis=0, rule=rule), mx_quantize(x, fmt, axis=0, rule=rule),
                               dtype=weight.dtype)
            else:
                dw = torch.zeros_like(weight)
        return dx, dw, None, None


def mx_linear(x, weight, fmt="e4m3", rule="floor"):
    """y = x weight^T with MX products, forward and backward: x (..., k), weight (n, k), y (..., n) of x's type.

    Every operand is quantised along the axis its product contracts: y from x and weight along k, dx = dy weight from
    both along n, dweight = dy^T x from both along the rows of x.  The roundings themselves are passed over in the
    backward pass (their derivative is taken as one).  A second derivative is refused.  A captured backward pass needs
    what torch needs of any: no eager graph of the same leaves alive on another stream."""
    _tensor(x, "x")
    _tensor(weight, "weight")
    _format(fmt)
    _rule(rule)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or x.device != weight.device:
        raise ValueError(f"x (..., k) and weight (n, k) on one device required, not {tuple(x.shape)} and "
                         f"{tuple(weight.shape)}")
    return _MXLinear.apply(x, weight, fmt, rule)


__all__ = ["MXMatrix", "mx_quantize", "mx_matmul", "mx_grouped_matmul", "mx_rms_norm", "mx_linear", "mx_check_errors"]
