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
eager product on that device).  They call the library on the tensors' memory, which ``torch.compile`` cannot trace: it
breaks its graph at each of them.  A product whose bounded waits ran out leaves a flag that ``mx_check_errors`` raises.
Only ``mx_linear`` has gradients: ``mx_rms_norm`` refuses inputs that require one (under ``torch.no_grad()`` it takes
them), and an ``MXMatrix`` is not a tensor and carries none.
"""
from __future__ import annotations

import threading

import torch
from torch.autograd import forward_ad as _forward_ad

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
ROWS_MAX = 0x7fffff00
_INT_MAX = 2 ** 31 - 1

_empty, _uint8, _Tensor = torch.empty, torch.uint8, torch.Tensor
_current_device = torch._C._cuda_getDevice
_stream_of = torch._C._cuda_getCurrentRawStream    # handle of a device's current stream
_increment_version = torch.autograd.graph.increment_version
_error_lock = threading.Lock()
_error_words = {}                # device index -> int32 word that the products' launches OR their flags into


class _Devices(dict):
    """torch.device objects by index, made once."""

    def __missing__(self, index):
        d = self[index] = torch.device("cuda", index)
        return d


_DEVICES = _Devices()


def _operand_bytes(code, groups, rows, k):
    """(bytes of the codes, a multiple of 64; bytes of codes and scales) of an operand."""
    if not 1 <= k <= KMAX:
        raise ValueError(f"contracted axis of length {k}: 1 to {KMAX} required")
    if rows < 0 or groups < 0:
        raise ValueError(f"operand of {groups} x {rows} x {k} elements: negative sizes")
    kt, rt = -(-k // TILE), -(-rows // TILE)
    if rows > ROWS_MAX or groups * rt * kt > _INT_MAX:
        raise ValueError(f"operand of {groups} x {rows} x {k} elements is too large")
    codes = groups * rows * kt * (TILE if code else TILE // 2)
    return codes, codes + groups * rt * kt * TILE_BYTES


def _new_operand(fmt, code, groups, rows, k, device):
    """MXMatrix(fmt, groups, rows, k, device) for a format whose code is known."""
    code_bytes, total = _operand_bytes(code, 1 if groups is None else groups, rows, k)
    out = object.__new__(MXMatrix)
    out._take(fmt, code, groups, rows, k, device, code_bytes, _empty(total, dtype=_uint8, device=_DEVICES[device]))
    return out


def _from_buffer(fmt, groups, rows, k, buffer):
    """The operand whose codes and scales are ``buffer``."""
    code = _format(fmt)
    code_bytes, total = _operand_bytes(code, 1 if groups is None else groups, rows, k)
    if not isinstance(buffer, _Tensor) or not buffer.is_cuda or buffer.dtype != _uint8 or not buffer.is_contiguous() \
            or tuple(buffer.shape) != (total,):
        raise ValueError(f"an operand's {total} bytes as a contiguous uint8 CUDA tensor required")
    out = object.__new__(MXMatrix)
    out._take(fmt, code, groups, rows, k, buffer.get_device(), code_bytes, buffer)
    return out


def _padded(k: int) -> int:
    return (k + TILE - 1) // TILE * TILE


def _error_word(device: int):
    w = _error_words.get(device)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            raise OzkError("the first MX product on a device allocates its error word: make one call before capturing")
        with _error_lock:
            w = _error_words.get(device)
            if w is None:
                with torch.inference_mode(False):    # mx_check_errors clears it in whatever mode it is called
                    w = torch.zeros(1, dtype=torch.int32, device=f"cuda:{device}")
                if type(w) is not _Tensor or not w.data_ptr():      # a tracer's stand-in, which has no memory
                    raise OzkError("the first MX product on a device allocates its error word: make one call before tracing")
                torch.cuda.synchronize(device)       # products on any stream may use it from here on
                _error_words[device] = w
    return w.data_ptr()


def mx_check_errors(device=None) -> None:
    """Raise OzkError if a product launched on ``device`` (default: the current one) gave up a wait since the last
    check; synchronises the device."""
    if device is not None:
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"{device}: a CUDA device required")
        device = device.index
    if device is None:                          # or "cuda", which names the current one
        device = torch.cuda.current_device()
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
    if not isinstance(t, _Tensor) or not t.is_cuda:
        raise ValueError(f"{what}: CUDA tensor required (there is no CPU path)")
    if t.is_neg():
        raise ValueError(f"{what}: a view whose sign is still to be turned (see torch.Tensor.resolve_neg)")
    code = _DTYPES.get(t.dtype)
    return _dtype(t.dtype, what) if code is None else code


class MXMatrix:
    """An operand of the MX products: ``rows`` vectors of length ``k`` (times ``groups``, for experts; None: a plain
    matrix) in element format ``fmt``.  Made by ``mx_quantize``, ``mx_rms_norm`` or ``MXMatrix.from_codes``."""

    __slots__ = ("fmt", "groups", "rows", "k", "device", "_fmt", "_buffer", "_code_ptr", "_scale_ptr", "_code_bytes")

    def __init__(self, fmt, groups, rows, k, device: int):
        """An operand with uninitialised contents."""
        code = _format(fmt)
        code_bytes, total = _operand_bytes(code, 1 if groups is None else groups, rows, k)
        self._take(fmt, code, groups, rows, k, device, code_bytes, _empty(total, dtype=_uint8, device=_DEVICES[device]))

    def _take(self, fmt, code, groups, rows, k, device, code_bytes, buffer):
        self.fmt = fmt
        self._fmt = code
        self.groups = groups
        self.rows = rows
        self.k = k
        self.device = device
        self._buffer = buffer
        self._code_bytes = code_bytes
        self._code_ptr = p = buffer.data_ptr()               # one allocation: the codes, then the scales
        self._scale_ptr = p + code_bytes

    @property
    def shape(self):
        return (self.rows, self.k) if self.groups is None else (self.groups, self.rows, self.k)

    def __repr__(self):
        return f"MXMatrix({self.fmt}, shape={self.shape}, device='cuda:{self.device}')"

    @property
    def _g(self):
        return 1 if self.groups is None else self.groups

    def __reduce__(self):
        """Copies and pickles hold the buffer, and take their addresses from their own."""
        return _from_buffer, (self.fmt, self.groups, self.rows, self.k, self._buffer)

    def record_stream(self, stream):
        """As ``torch.Tensor.record_stream``: the operand is also used on ``stream``, so its memory is not handed out again
        before the work there is done."""
        self._buffer.record_stream(stream)

    def codes(self):
        """The element codes as uint8 (..., rows, ceil(k / 2)) for e2m1 (two a byte, the even one in the lower half)
        or (..., rows, k) for e4m3: a copy in the order in which checkpoints store them.  The half of a byte behind an odd
        number of 4-bit codes is zero."""
        per = (self.k + 1) // 2 if self._fmt == 0 else self.k
        pitch = _padded(self.k) // (2 if self._fmt == 0 else 1)
        c = self._buffer[:self._code_bytes].view(self._g, self.rows, pitch)[..., :per].clone(
            memory_format=torch.contiguous_format)
        if self._fmt == 0 and self.k % 2:
            c[..., -1] &= 15                    # a block with the NaN scale has codes behind its end too
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
        pitch = _padded(k) // (2 if code == 0 else 1)
        c = out._buffer[:out._code_bytes].view(g, rows, pitch)
        c[..., :per] = codes.reshape(g, rows, per)
        if code == 0 and k % 2:
            c[..., per - 1] &= 15
        if per < pitch:
            c[..., per:] = 0
        rt, kt = -(-rows // TILE), _padded(k) // TILE
        s = scales.reshape(g, rows, scales.shape[-1])
        if s.shape[1:] != (rt * TILE, 4 * kt):
            s = torch.nn.functional.pad(s, (0, 4 * kt - s.shape[-1], 0, rt * TILE - rows))
        s = s.contiguous()
        out._buffer[out._code_bytes:].view(g, rt, kt, 32, 4, 4).copy_(
            s.view(g, rt, 4, 32, kt, 4).permute(0, 1, 4, 3, 2, 5))
        return out

    def dequantize(self, dtype=torch.bfloat16):
        """The numbers the operand stands for, as a contiguous tensor (bfloat16 and float32 hold them exactly while
        their scales are ordinary)."""
        d = _DTYPES.get(dtype)
        if d is None:
            d = _dtype(dtype, "dequantize")
        device = self.device
        if _current_device() != device:
            with torch.cuda.device(device):
                return self.dequantize(dtype)
        out = _empty(self.shape, dtype=dtype, device=_DEVICES[device])
        if self.rows and self.groups != 0:
            rc = _lib.lib().ozk_mx_dequantize(self._code_ptr, self._scale_ptr, self._fmt, self.groups or 1, self.rows,
                                              self.k, out.data_ptr(), d, _stream_of(device))
            if rc:
                check(rc, "ozk_mx_dequantize")
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
    shape, stride = x.shape, x.stride()
    dim = len(shape)
    if dim == 2 and -2 <= axis < 2:
        at, other, groups, group_stride = axis & 1, 1 - (axis & 1), None, 0
    elif dim == 3 and axis in (-1, -2, 1, 2):
        at = axis % 3
        other, groups, group_stride = 3 - at, shape[0], stride[0]
    else:
        if dim not in (2, 3):
            raise ValueError(f"x: 2 or 3 axes required, not {dim}")
        raise ValueError(f"axis {axis} of {dim}: one of the last two is contracted")
    device = x.get_device()
    if _current_device() != device:
        with torch.cuda.device(device):
            return mx_quantize(x, fmt, axis, rule)
    rows, k = shape[other], shape[at]
    out = _new_operand(fmt, code, groups, rows, k, device)
    if rows and groups != 0:
        rc = _lib.lib().ozk_mx_quantize(x.data_ptr(), d, groups or 1, rows, k, group_stride, stride[other],
                                        stride[at], code, up, out._code_ptr, out._scale_ptr,
                                        _stream_of(device))
        if rc:
            check(rc, "ozk_mx_quantize")
    return out


def mx_quantize_both(x, fmt="e4m3", rule="floor"):
    """(mx_quantize(x, fmt, -1, rule), mx_quantize(x, fmt, 0, rule)) of a matrix from one read of it: what a training
    step needs of an operand whose two axes are contracted in turn."""
    d = _tensor(x, "x")
    code, up = _format(fmt), _rule(rule)
    if x.dim() != 2:
        raise ValueError(f"x: 2 axes required, not {x.dim()}")
    device = x.get_device()
    if _current_device() != device:
        with torch.cuda.device(device):
            return mx_quantize_both(x, fmt, rule)
    rows, cols = x.shape
    if not rows or not cols:
        raise ValueError("x: both axes are contracted in turn and cannot be empty")
    along_rows = _new_operand(fmt, code, None, rows, cols, device)
    along_cols = _new_operand(fmt, code, None, cols, rows, device)
    rc = _lib.lib().ozk_mx_quantize_both(x.data_ptr(), d, rows, cols, x.stride(0), x.stride(1), code, up,
                                         along_rows._code_ptr, along_cols._code_ptr, _stream_of(device))
    if rc:
        check(rc, "ozk_mx_quantize_both")
    return along_rows, along_cols


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
        d = _DTYPES.get(dtype)
        if d is None:
            d = _dtype(dtype, "dtype")
        return _empty((rows, cols), dtype=dtype, device=_DEVICES[device]), d, cols or 1
    d = _tensor(C, "C")
    if C.device.index != device or tuple(C.shape) != (rows, cols) or (cols > 1 and C.stride(1) != 1) \
            or (rows > 1 and C.stride(0) < cols):
        raise ValueError(f"C: ({rows}, {cols}) on cuda:{device} with contiguous, separate rows required")
    if C.requires_grad and torch.is_grad_enabled():
        raise ValueError("C: requires a gradient, which the product does not give")
    if not C.is_inference():
        _increment_version(C)                   # a backward pass that kept the old C has to notice
    return C, d, C.stride(0) if rows > 1 else max(cols, 1)


def mx_matmul(A, B, C=None, dtype=torch.bfloat16):
    """C = A B^T for MX operands A (m, k) and B (n, k) of any formats: sums in FP32, one rounding to ``dtype`` (or to
    the type of a given ``C``, whose rows may be strided)."""
    _operands(A, B)
    if B.groups is not None:
        raise ValueError("B: a plain matrix required (see mx_grouped_matmul)")
    device = A.device
    if _current_device() != device:
        with torch.cuda.device(device):
            return mx_matmul(A, B, C, dtype)
    C, d, ldc = _result(C, A.rows, B.rows, dtype, device)
    if A.rows and B.rows:
        rc = _lib.lib().ozk_mx_gemm(A._code_ptr, A._scale_ptr, A._fmt, B._code_ptr, B._scale_ptr, B._fmt, A.rows, B.rows,
                                    A.k, C.data_ptr(), ldc, d, _error_word(device), _stream_of(device))
        if rc:
            check(rc, "ozk_mx_gemm")
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
    device = A.device
    if _current_device() != device:
        with torch.cuda.device(device):
            return mx_grouped_matmul(A, B, ends, C, dtype)
    fill = C is None
    C, d, ldc = _result(C, A.rows, B.rows, dtype, device)
    if A.rows and B.rows:
        rc = _lib.lib().ozk_mx_grouped_gemm(A._code_ptr, A._scale_ptr, A._fmt, B._code_ptr, B._scale_ptr, B._fmt, A.rows,
                                            B.rows, A.k, B.groups, ends.data_ptr(), fill, C.data_ptr(), ldc, d,
                                            _error_word(device), _stream_of(device))
        if rc:
            check(rc, "ozk_mx_grouped_gemm")
    return C


def mx_rms_norm(x, weight, residual=None, eps=1e-6, fmt="e4m3", rule="floor"):
    """Root-mean-square norm into an MX operand: t = x + residual, y = t / sqrt(mean(t^2) + eps) * weight over the last
    axis, in FP32 from the loads to the codes.  Returns (y as MXMatrix (rows, d) with the leading axes of x as rows, t
    rounded to the type of x and in its shape, or None without a residual).  It has no gradient: inputs that require one
    are refused while gradients are recorded."""
    d = _tensor(x, "x")
    code, up = _format(fmt), _rule(rule)
    shape = x.shape
    if not shape:
        raise ValueError("x: at least one axis required")
    n = shape[-1]
    device, dtype = x.get_device(), x.dtype
    if not isinstance(weight, _Tensor) or weight.get_device() != device or weight.shape != shape[-1:] \
            or not (weight.dtype is dtype or weight.dtype is torch.float32) or not weight.is_contiguous() \
            or weight.is_neg():
        raise ValueError(f"weight: contiguous ({n},) tensor of x's type or float32 on its device required")
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"eps {eps}: a positive number required")
    if residual is not None and (not isinstance(residual, _Tensor) or residual.shape != shape
                                 or residual.dtype is not dtype or residual.get_device() != device or residual.is_neg()):
        raise ValueError("residual: a tensor of x's shape, type and device required")
    if (x.requires_grad or weight.requires_grad or residual is not None and residual.requires_grad) \
            and torch.is_grad_enabled():        # it would be lost without a word
        raise ValueError("mx_rms_norm has no gradient, and an input requires one (see torch.no_grad, torch.Tensor.detach)")
    if _forward_ad._current_level >= 0 and any(t is not None and _forward_ad.unpack_dual(t).tangent is not None
                                               for t in (x, weight, residual)):
        raise ValueError("mx_rms_norm has no forward-mode derivative, and an input has a tangent")
    if _current_device() != device:
        with torch.cuda.device(device):
            return mx_rms_norm(x, weight, residual, eps, fmt, rule)
    x2 = x if len(shape) == 2 and x.stride(1) == 1 else _rows(x, n)
    rows = x2.shape[0]
    out = _new_operand(fmt, code, None, rows, n, device)
    r_ptr = r_stride = t_ptr = 0
    total = None
    if residual is not None:
        r2 = residual if len(shape) == 2 and residual.stride(1) == 1 else _rows(residual, n)
        r_ptr, r_stride = r2.data_ptr(), r2.stride(0)
        total = _empty(shape, dtype=dtype, device=_DEVICES[device])
        t_ptr = total.data_ptr()
    if rows:
        rc = _lib.lib().ozk_mx_rms_norm(x2.data_ptr(), r_ptr, weight.data_ptr(), d, weight.dtype == torch.float32, rows,
                                        n, x2.stride(0), r_stride, eps, code, up, t_ptr, out._code_ptr, out._scale_ptr,
                                        _stream_of(device))
        if rc:
            check(rc, "ozk_mx_rms_norm")
    return out, total


def _rows(x, n):
    """x as a matrix of rows of length n >= 1 with contiguous elements: x itself or a view where it can be."""
    if x.dim() != 2:
        x = x.reshape(x.numel() // max(n, 1), n)
    return x if x.stride(1) == 1 or n < 2 else x.contiguous()


def _linear_forward(x2, weight, code, up, need_dx, need_dw):
    """y and what the backward pass takes, or None: one buffer of the weight along n (where dx is wanted) and of x along
    its rows (where dweight is)."""
    device = x2.get_device()
    m, k = x2.shape
    n = weight.shape[0]
    xk, wk = _operand_bytes(code, 1, m, k)[1], _operand_bytes(code, 1, n, k)[1]
    dev = _DEVICES[device]
    kept = None
    wn_ptr = xm_ptr = 0
    if need_dx or need_dw:
        wn = _operand_bytes(code, 1, k, n)[1] if need_dx else 0
        xm = _operand_bytes(code, 1, k, m)[1] if need_dw else 0
        kept = _empty(wn + xm, dtype=_uint8, device=dev)
        p = kept.data_ptr()
        wn_ptr, xm_ptr = p if need_dx else 0, p + wn if need_dw else 0
    y = _empty((m, n), dtype=x2.dtype, device=dev)
    scratch = _empty(xk + wk, dtype=_uint8, device=dev)
    p = scratch.data_ptr()
    x_row, x_col = x2.stride()
    w_row, w_col = weight.stride()
    rc = _lib.lib().ozk_mx_linear_forward(x2.data_ptr(), _DTYPES[x2.dtype], x_row, x_col, weight.data_ptr(),
                                          _DTYPES[weight.dtype], w_row, w_col, m, n, k, code, up, p, p + xk, xm_ptr, wn_ptr,
                                          y.data_ptr(), _error_word(device), _stream_of(device))
    if rc:
        check(rc, "ozk_mx_linear_forward")
    return y, kept


def _linear_backward(ctx, dy):
    kept, = ctx.saved_tensors
    if dy.is_neg():                             # of y in a conjugate's imaginary part
        dy = dy.resolve_neg()
    code, up, need_dx, need_dw, x_code, w_code, w_dtype, n, k = ctx.how
    device, m = dy.get_device(), dy.shape[0]
    dev = _DEVICES[device]
    along_n, along_m = _operand_bytes(code, 1, m, n)[1], _operand_bytes(code, 1, n, m)[1]
    dx = dw = None
    dx_ptr = dw_ptr = xm_ptr = wn_ptr = 0
    p = kept.data_ptr()
    if need_dx:
        dx = _empty((m, k), dtype=dy.dtype, device=dev)        # y, and so dy, has the type of x
        dx_ptr, wn_ptr = dx.data_ptr(), p
        p += _operand_bytes(code, 1, k, n)[1]
    if need_dw:
        dw = _empty((n, k), dtype=w_dtype, device=dev)
        dw_ptr, xm_ptr = dw.data_ptr(), p
    scratch = _empty(along_n + along_m, dtype=_uint8, device=dev)
    p = scratch.data_ptr()
    row_stride, col_stride = dy.stride()
    rc = _lib.lib().ozk_mx_linear_backward(dy.data_ptr(), x_code, row_stride, col_stride, xm_ptr, wn_ptr, m, n, k, code, up,
                                           p, p + along_n, dx_ptr, x_code, dw_ptr, w_code, _error_word(device),
                                           _stream_of(device))
    if rc:
        check(rc, "ozk_mx_linear_backward")
    return dx, dw, None, None


_linear_backward_once = torch.autograd.function.once_differentiable(_linear_backward)


class _MXLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, code, up):
        need_dx, need_dw = ctx.needs_input_grad[:2]
        y, kept = _linear_forward(x, weight, code, up, need_dx, need_dw)
        ctx.save_for_backward(kept)
        ctx.how = (code, up, need_dx, need_dw, _DTYPES[x.dtype], _DTYPES[weight.dtype], weight.dtype, *weight.shape)
        return y

    @staticmethod
    def backward(ctx, dy):
        # under create_graph the gradients must say that they cannot be differentiated again
        return _linear_backward_once(ctx, dy) if torch.is_grad_enabled() else _linear_backward(ctx, dy)


def mx_linear(x, weight, fmt="e4m3", rule="floor"):
    """y = x weight^T with MX products, forward and backward: x (..., k), weight (n, k), y (..., n) of x's type.

    Every operand is quantised along the axis its product contracts: y from x and weight along k, dx = dy weight from
    both along n, dweight = dy^T x from both along the rows of x.  The roundings themselves are passed over in the
    backward pass (their derivative is taken as one).  A second derivative and forward-mode differentiation are refused.
    A captured backward pass needs what torch needs of any: no eager graph of the same leaves alive on another stream."""
    _tensor(x, "x")
    _tensor(weight, "weight")
    code, up = _format(fmt), _rule(rule)
    shape, w_shape = x.shape, weight.shape
    device = x.get_device()
    if len(w_shape) != 2 or not shape or shape[-1] != w_shape[1] or device != weight.get_device():
        raise ValueError(f"x (..., k) and weight (n, k) on one device required, not {tuple(shape)} and {tuple(w_shape)}")
    if _current_device() != device:
        with torch.cuda.device(device):
            return mx_linear(x, weight, fmt, rule)
    n, k = w_shape
    if k == 0:
        raise ValueError("contracted axis of length 0: at least 1 required")
    if n == 0 or x.numel() == 0:
        return torch.matmul(x, weight.t().to(x.dtype))        # nothing to multiply: empty, with its gradients of zero
    plain = len(shape) == 2
    x2 = x if plain else x.reshape(-1, k)
    if (x.requires_grad or weight.requires_grad) and torch.is_grad_enabled() or _forward_ad._current_level >= 0:
        y = _MXLinear.apply(x2, weight, code, up)
    else:
        y = _linear_forward(x2, weight, code, up, False, False)[0]
    return y if plain else y.view(*shape[:-1], n)


__all__ = ["MXMatrix", "mx_quantize", "mx_quantize_both", "mx_matmul", "mx_grouped_matmul", "mx_rms_norm", "mx_linear", "mx_check_errors"]
