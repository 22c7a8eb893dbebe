"""Microscaled operators: 8- and 4-bit block-scaled tensors, their products, and the layers between two products.

A linear layer in microscaled formats keeps its operands as codes of 8 or 4 bits with a scale for every block of 32 or
16 consecutive values along the dimension that the product sums over, and multiplies them on the tensor cores' block-
scaled kinds. Formats:

    "mxfp8"   e4m3 codes, a power-of-two scale per 32 values        (1.03 bytes a value)
    "mxfp4"   e2m1 codes, a power-of-two scale per 32 values        (0.53)
    "nvfp4"   e2m1 codes, an e4m3 scale per 16 values, and one fp32 scale for the tensor   (0.56)

    quantize, dequantize           values <-> MicroTensor; `quantize(x.t(), ...)` reads a transposed view as it lies
    micro_matmul, MicroMatmul      C[M, N] = A[M, K] @ B[N, K].T of two MicroTensors of one format; one-shot, and with the
                                   family's make_runner(a, b, out=None) protocol
    micro_linear                   differentiable x @ w.T: forward and both gradients are products in the format
    rms_norm, silu_mul             the layers between two products: values out (differentiable), or written in the
                                   format the next product reads; *_backward are their gradients as plain calls
    micro_mlp                      norm -> gate and up projection -> SiLU gate -> down projection, every hand-over in the
                                   format

All of it enqueues on the current stream of the tensors' device and allocates its outputs (and the norm gradient's
workspace) from torch's allocator on that stream; nothing is kept between calls, nothing synchronises, and every call
can be captured into a CUDA graph (a training step with torch's own condition: no eager autograd graph of the same
leaves may be alive during the capture). The differentiable calls have a backward pass of first order; forward-mode
derivatives through them are refused, and nothing is differentiable through the other calls. As elsewhere with torch,
tensors made on another stream have to be ready on the current one. The product's kernels bound their waits:
`check_status()` (from cs464_b200.matmul) raises if one ran out.

The arithmetic of a quantisation is exact: which code and which scale a value gets follows from its bits alone
(include/b2g_micro.h), so results do not depend on the launch. Infinities and NaN make their block's scale NaN, and with
it the block's 32 or 16 values. Products accumulate in fp32 on the tensor cores and round once, to the output's type.
"""
from __future__ import annotations

import ctypes
import math
import struct
import weakref
from operator import attrgetter

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from cs464_b200 import _abi
from cs464_b200.matmul import _STATUS, check_status, status_word  # noqa: F401 (check_status is part of this API)

FORMATS = {"mxfp8": _abi.FMT_MXFP8, "mxfp4": _abi.FMT_MXFP4, "nvfp4": _abi.FMT_NVFP4}
BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}

_VALUES = {torch.float16: _abi.VALUE_F16, torch.bfloat16: _abi.VALUE_BF16, torch.float32: _abi.VALUE_F32}
_HALF = {torch.float16: _abi.VALUE_F16, torch.bfloat16: _abi.VALUE_BF16}

# A call of a few microseconds on the GPU is paid for on the host, so the calls below keep it short: structures go to the
# library as packed bytes, one allocation holds a tensor's codes and scales, and the checks that pass are the cheap ones
# (those that fail repeat at leisure to say why).
_pack_tensor = struct.Struct("=iiqqQqQQ").pack   # b2g_micro_tensor
_pack_matrix = struct.Struct("=Qqq").pack        # b2g_micro_matrix
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _Entry:
    """The entry points that enqueue work, bound with plain pointers for the structures, on first use."""

    _ARGS = {"tensor_scale": "pqqipp", "quantize": "pipp", "dequantize": "ppip", "matmul": "pppqipp", "plan_launch": "pp",
             "matmul_values": "ppqqqiipqipzpp",
             "rms_norm": "ppppppqqfip", "rms_norm_backward": "pppppppzqqfip", "silu_mul": "pppqqip",
             "silu_mul_backward": "pppqqip"}
    _KIND = {"p": ctypes.c_void_p, "q": ctypes.c_int64, "i": ctypes.c_int32, "f": ctypes.c_float, "z": ctypes.c_size_t}

    def __getattr__(self, name: str):
        fn = _abi.load()["b2g_micro_" + name]
        fn.argtypes = [self._KIND[k] for k in self._ARGS[name]]
        fn.restype = ctypes.c_int32
        fn.what = "b2g_micro_" + name
        setattr(self, name, fn)
        return fn


_entry = _Entry()


def _call(index: int, fn, *args) -> None:
    """Enqueue an entry point on the current stream of device `index`, with it the current device."""
    if _get_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _abi.check(rc, fn.what)


def _matrix(t: torch.Tensor) -> bytes:
    return _pack_matrix(t.data_ptr(), *t.stride())


_BYTES: dict[int, torch.Tensor] = {}  # an empty uint8 tensor per device: new_empty of it is the cheapest allocation


def _new_bytes(n: int, like: torch.Tensor) -> torch.Tensor:
    index = like.get_device()
    proto = _BYTES.get(index)
    if proto is None:
        proto = torch.empty(0, dtype=torch.uint8, device=like.device)
        if type(proto) is not torch.Tensor:  # made under a mode that replaces tensors: it must not outlive that
            raise RuntimeError(f"no kernel runs on a {type(proto).__name__}")
        _BYTES[index] = proto
    return proto.new_empty(n)


def _format(fmt: str) -> int:
    try:
        return FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"format must be one of {', '.join(FORMATS)}, not {fmt!r}") from None


def _check(t: torch.Tensor, what: str, dtypes, like: torch.Tensor | None = None) -> None:
    """Raise unless t is a CUDA tensor of one of `dtypes`, on the device of `like`."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor (there is no CPU path)")
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d)[6:] for d in dtypes)}, not {str(t.dtype)[6:]}")
    if like is not None and t.get_device() != like.get_device():
        raise ValueError(f"{what} is on {t.device}, the other tensors on {like.device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as a matrix of rows (its last dimension) whose storage holds its values: torch keeps some views negated lazily
    (the imaginary part of a conjugate; gradients of such come from autograd), which become copies."""
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.dim() == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _weight(t: torch.Tensor) -> torch.Tensor:
    """t contiguous, its storage holding its values."""
    return t if t.is_contiguous() and not t.is_neg() else t.resolve_neg().contiguous()


def _check_out(t: torch.Tensor) -> None:
    if t.is_neg():
        raise ValueError("out is a lazily negated view: its storage would hold the negated values")


def _like(t: torch.Tensor) -> torch.Tensor:
    """Uninitialised contiguous storage of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _has_tangent(*tensors: torch.Tensor | None) -> bool:
    """Whether a forward-mode derivative is being taken through one of them."""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _check_scale(scale, like: torch.Tensor) -> None:
    if (not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or scale.numel() != 1
            or scale.get_device() != like.get_device() or scale.is_neg()):
        raise ValueError(f"scale must be a float32 tensor of one element on {like.device}, not negated lazily")


def _layout(fmt: int, rows: int, cols: int) -> tuple[int, int]:
    """(pitch, scale bytes) of a tensor: b2g_micro_layout."""
    if fmt == _abi.FMT_MXFP8:
        return (cols + 31) // 32 * 32, (rows + 127) // 128 * ((cols + 127) // 128) * 512
    if fmt == _abi.FMT_MXFP4:
        return (cols + 31) // 32 * 16, (rows + 127) // 128 * ((cols + 127) // 128) * 512
    return (cols + 31) // 32 * 16, (rows + 127) // 128 * ((cols + 63) // 64) * 512


class MicroTensor:
    """A [rows, cols] matrix in a microscaled format, blocks along the columns.

    `codes`: uint8 [rows, pitch], unit column stride, rows 16 bytes (mxfp8: 32) apart or a multiple of that; two 4-bit
    codes a byte, the lower column in the low bits, what is left of an odd row's last byte zero. `scales`: uint8,
    contiguous, ceil(rows / 128) * ceil(blocks / 4) tiles of 512 bytes in the tensor cores' order (include/b2g_micro.h),
    zero where rows or blocks do not exist. `scale`: nvfp4's fp32 scale of the tensor (one element on the device), which
    other formats do not have. The constructor checks and takes the tensors as they are. None of the fields can be
    assigned: calls read the addresses packed here. Another scale is another tensor, MicroTensor(q.codes, q.scales,
    q.shape, q.format, scale); what the tensors hold may be changed in place."""

    __slots__ = ("_codes", "_scales", "_shape", "_format", "_scale", "_buf", "_raw", "__weakref__")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, format: str, scale: torch.Tensor | None = None):
        fmt = _format(format)
        rows, cols = map(int, shape)
        if rows < 0 or cols < 0:
            raise ValueError(f"bad shape {tuple(shape)}")
        _check(codes, "codes", (torch.uint8,))
        _check(scales, "scales", (torch.uint8,), codes)
        pitch, scale_bytes = _layout(fmt, rows, cols)
        at, sat = codes.data_ptr(), scales.data_ptr()
        row = pitch
        if rows and cols:
            step = 32 if fmt == _abi.FMT_MXFP8 else 16
            if rows > 1 and codes.dim() == 2:
                row = codes.stride(0)
            if (codes.dim() != 2 or codes.shape[0] != rows or codes.shape[1] < pitch or codes.stride(1) != 1
                    or row < pitch or row % step or at % 16):
                raise ValueError(f"codes of a {rows}x{cols} {format} tensor must be [{rows}, >= {pitch}] bytes, 16-byte "
                                 f"aligned, rows a multiple of {step} bytes apart, not {tuple(codes.shape)} with strides "
                                 f"{codes.stride()}")
            if scales.numel() != scale_bytes or not scales.is_contiguous() or sat % 16:
                raise ValueError(f"scales of a {rows}x{cols} {format} tensor must be {scale_bytes} contiguous, 16-byte "
                                 f"aligned bytes, not {tuple(scales.shape)} with strides {scales.stride()}")
        if fmt == _abi.FMT_NVFP4:
            _check_scale(scale, codes)
        elif scale is not None:
            raise ValueError(f"{format} has no tensor scale")
        self._codes, self._scales, self._buf = codes, scales, codes
        self._shape, self._format, self._scale = (rows, cols), format, scale
        self._raw = _pack_tensor(fmt, 0, rows, cols, at, row, sat, scale.data_ptr() if scale is not None else 0)

    @classmethod
    def _new(cls, like: torch.Tensor, fmt: int, format: str, rows: int, cols: int, scale) -> "MicroTensor":
        """Uninitialised storage (codes, then scales) on the device of `like`, for a kernel to fill."""
        self = cls.__new__(cls)
        pitch, scale_bytes = _layout(fmt, rows, cols)
        buf = self._buf = _new_bytes(rows * pitch + scale_bytes, like)
        at = buf.data_ptr()
        self._codes = self._scales = None
        self._shape, self._format, self._scale = (rows, cols), format, scale
        self._raw = _pack_tensor(fmt, 0, rows, cols, at, pitch, at + rows * pitch,
                                 scale.data_ptr() if scale is not None else 0)
        return self

    shape = property(attrgetter("_shape"))
    format = property(attrgetter("_format"))
    scale = property(attrgetter("_scale"))

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            rows, cols = self.shape
            pitch = _layout(FORMATS[self.format], rows, cols)[0]
            self._codes = self._buf[:rows * pitch].view(rows, pitch)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            rows, cols = self.shape
            self._scales = self._buf[rows * _layout(FORMATS[self.format], rows, cols)[0]:]
        return self._scales

    @property
    def device(self) -> torch.device:
        return self._buf.device

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return dequantize(self, dtype)

    def code_values(self) -> torch.Tensor:
        """mxfp8's codes as float8_e4m3fn [rows, cols], a view. (4-bit codes have no torch type: `dequantize`.)"""
        if self.format != "mxfp8":
            raise TypeError(f"{self.format} codes are packed; dequantize() gives their values")
        rows, cols = self.shape
        if self._codes is None:
            return self._buf.view(torch.float8_e4m3fn).as_strided((rows, cols), ((cols + 31) // 32 * 32, 1))
        return self._codes[:, :cols].view(torch.float8_e4m3fn)

    def scale_tiles(self) -> torch.Tensor:
        """The block scales as float8_e8m0fnu (nvfp4: float8_e4m3fn), a view [row tile, 4, 32, block tile, 4]: row
        128 t + 32 i + j and block 4 u + v at [t, i, j, u, v]."""
        rows, cols = self.shape
        tiles = -(-cols // (4 * BLOCK[self.format]))
        kind = torch.float8_e4m3fn if self.format == "nvfp4" else torch.float8_e8m0fnu
        if self._scales is None:
            buf, start = self._buf, rows * _layout(FORMATS[self.format], rows, cols)[0]
        else:
            buf, start = self._scales, self._scales.storage_offset()
        return buf.view(kind).as_strided((-(-rows // 128), 4, 32, tiles, 4), (tiles * 512, 4, 16, 512, 1), start)

    def __repr__(self) -> str:
        return f"MicroTensor({self.shape[0]}x{self.shape[1]}, {self.format}, {self.device})"


def quantize(x: torch.Tensor, format: str = "mxfp8", scale: torch.Tensor | None = None) -> MicroTensor:
    """x [rows, cols] (fp16, bf16 or fp32, any strides) in a microscaled format, blocks along the columns. No gradient
    passes (micro_linear is the differentiable layer).

    nvfp4: `scale` is the tensor's fp32 scale, one element on the device from 2^-100 to 2^117; values past 2688 times it
    saturate. Without it, x is read twice: its scale becomes the smallest power of two at which nothing saturates."""
    fmt = FORMATS.get(format)
    if fmt is None or not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _VALUES or x.dim() != 2:
        _format(format)
        _check(x, "x", _VALUES)
        raise ValueError(f"x must be a matrix, not {tuple(x.shape)}")
    if x.is_neg():
        x = x.resolve_neg()
    rows, cols = x.shape
    mat, kind, index = _pack_matrix(x.data_ptr(), *x.stride()), _VALUES[x.dtype], x.get_device()
    if fmt == _abi.FMT_NVFP4:
        if scale is None:
            scale = x.new_empty((1,), dtype=torch.float32)
            _call(index, _entry.tensor_scale, mat, rows, cols, kind, scale.data_ptr())
        else:
            _check_scale(scale, x)
    elif scale is not None:
        raise ValueError(f"{format} has no tensor scale")
    q = MicroTensor._new(x, fmt, format, rows, cols, scale)
    _call(index, _entry.quantize, mat, kind, q._raw)
    return q


def dequantize(q: MicroTensor, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of q: code * block scale (* tensor scale), rounded to `dtype` (fp16, bf16 or fp32). `out`: a tensor of
    q's shape to write them to instead, with any strides that do not overlap; its type is used."""
    if out is None:
        if dtype not in _VALUES:
            raise TypeError(f"dtype must be float16, bfloat16 or float32, not {dtype}")
        out = q._buf.new_empty(q._shape, dtype=dtype)
    else:
        _check(out, "out", _VALUES, q._buf)
        if tuple(out.shape) != q.shape:
            raise ValueError(f"out must be {q.shape[0]}x{q.shape[1]}, not {tuple(out.shape)}")
        _check_out(out)
    _call(q._buf.get_device(), _entry.dequantize, q._raw, _matrix(out), _VALUES[out.dtype])
    return out


# ---------------------------------------------------------------- products
_STATUS_AT: dict[int, int] = {}  # address of each device's status word (the words live as long as the process)


def _status(index: int) -> int:
    at = _STATUS_AT.get(index)
    if at is None:
        if index not in _STATUS and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"the first product on cuda:{index} makes the device's status word, which a stream capture "
                               "cannot hold: run a product there once before the capture")
        word = status_word(torch.device("cuda", index))
        if type(word) is not torch.Tensor:  # as in _new_bytes
            del _STATUS[index]
            raise RuntimeError(f"no kernel runs on a {type(word).__name__}")
        at = _STATUS_AT[index] = word.data_ptr()
    return at


def _output(a: MicroTensor, b: MicroTensor, out: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    if not isinstance(a, MicroTensor) or not isinstance(b, MicroTensor):
        raise TypeError("a and b must be MicroTensors (quantize makes them)")
    if a._buf.get_device() != b._buf.get_device():
        raise ValueError(f"a is on {a.device}, b on {b.device}")
    if a._format != b._format:
        raise ValueError(f"a is {a.format}, b {b.format}: a product needs one format")
    if a._shape[1] != b._shape[1]:
        raise ValueError(f"a is {a.shape[0]}x{a.shape[1]}, b {b.shape[0]}x{b.shape[1]}: their columns are summed over and "
                         "must agree")
    M, N = a._shape[0], b._shape[0]
    if out is None:
        if dtype not in _HALF:
            raise TypeError(f"dtype must be float16 or bfloat16, not {dtype}")
        return a._buf.new_empty((M, N), dtype=dtype)
    _check(out, "out", _HALF, a._buf)
    if tuple(out.shape) != (M, N) or (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
        raise ValueError(f"out must be a {M}x{N} tensor with unit column stride and rows that do not overlap, not "
                         f"{tuple(out.shape)} with strides {out.stride()}")
    _check_out(out)
    return out


def _ldc(c: torch.Tensor) -> int:
    return max(c.stride(0), c.shape[1])  # the row stride of a single row may be anything


def micro_matmul(a: MicroTensor, b: MicroTensor, out: torch.Tensor | None = None,
                 dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C[M, N] = A[M, K] @ B[N, K].T on the current stream, C in `dtype` (fp16 or bf16), or into `out` (unit column
    stride, any row stride) in its type."""
    c = _output(a, b, out, dtype)
    index = c.get_device()
    _call(index, _entry.matmul, a._raw, b._raw, c.data_ptr(), _ldc(c), _HALF[c.dtype], _status(index))
    return c


class _MicroRunner:
    """The closure MicroMatmul.make_runner returns: calling it enqueues the product and returns C."""

    __slots__ = ("_plan", "_device", "c", "status", "_keep", "_fin", "__weakref__")

    def __init__(self, plan: ctypes.c_void_p, c: torch.Tensor, status: torch.Tensor, keep):
        self._plan, self._device, self.c, self.status, self._keep = plan, c.get_device(), c, status, keep
        self._fin = weakref.finalize(self, _abi.load().b2g_micro_plan_destroy, plan)

    def __call__(self) -> torch.Tensor:
        _call(self._device, _entry.plan_launch, self._plan)
        return self.c

    def device_status(self) -> int:
        """The kernels' device status word (0 = ok; else a bounded wait ran out). Synchronises."""
        return int(self.status.item())

    def raise_on_status(self) -> None:
        s = self.device_status()
        if s:
            raise RuntimeError(f"b200 kernel status 0x{s:x}: {_abi.status_string(s)}")


class MicroMatmul:
    """Backend of the products with the family's protocol: make_runner(a, b, out=None) allocates the output and the
    launch plan once; the closure it returns allocates nothing and enqueues on the current stream."""

    family = "b200_sm100a_micro"

    def __init__(self, dtype: torch.dtype = torch.bfloat16, wait_limit_us: int = 0):
        """`wait_limit_us`: limit of the kernels' bounded device waits (0: the library's default of one second); refused for
        products that run as CTA pairs or split K over a cluster."""
        if dtype not in _HALF:
            raise TypeError(f"dtype must be float16 or bfloat16, not {dtype}")
        self.dtype, self.wait_limit_us = dtype, int(wait_limit_us)

    def make_runner(self, a: MicroTensor, b: MicroTensor, out: torch.Tensor | None = None) -> _MicroRunner:
        c = _output(a, b, out, self.dtype)
        plan = ctypes.c_void_p()
        with torch.cuda.device(a.device):
            status = torch.zeros(1, dtype=torch.int32, device=a.device)
            _abi.check(_abi.load().b2g_micro_plan_create(
                _abi.MicroTensor.from_buffer_copy(a._raw), _abi.MicroTensor.from_buffer_copy(b._raw), c.data_ptr(), _ldc(c),
                _HALF[c.dtype], status.data_ptr(), ctypes.byref(plan)), "b2g_micro_plan_create")
        run = _MicroRunner(plan, c, status, (a, b))
        if self.wait_limit_us:
            _abi.check(_abi.load().b2g_micro_plan_wait_limit(plan, self.wait_limit_us), "b2g_micro_plan_wait_limit")
        return run


def _values_product(a: torch.Tensor, b: torch.Tensor, fmt: int) -> torch.Tensor:
    """q(a) @ q(b).T of matrices of values, in their type: quantize and micro_matmul in one call."""
    M, K = a.shape
    N = b.shape[0]
    c = a.new_empty((M, N))
    pitch, a_scales = _layout(fmt, M, K)
    n = 32 + (M + N) * pitch + a_scales + _layout(fmt, N, K)[1]  # b2g_micro_matmul_values_workspace
    ws, index, kind = _new_bytes(n, a), a.get_device(), _HALF[a.dtype]
    _call(index, _entry.matmul_values, _matrix(a), _matrix(b), M, N, K, kind, fmt, c.data_ptr(), max(N, 1), kind,
          ws.data_ptr(), n, _status(index))
    return c


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, fmt):
        ctx.save_for_backward(x, w)
        ctx.fmt = fmt
        return _values_product(x, w, fmt)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        fmt, dx, dw, dy = ctx.fmt, None, None, _rows(dy)
        if ctx.needs_input_grad[0]:
            dx = _values_product(dy, w.t(), fmt)
        if ctx.needs_input_grad[1]:
            dw = _values_product(dy.t(), x.t(), fmt)
        return dx, dw, None


def micro_linear(x: torch.Tensor, w: torch.Tensor, format: str = "mxfp8") -> torch.Tensor:
    """x [..., K] @ w [N, K].T (fp16 or bf16, one type), differentiable, in a format: y = q(x) q(w)^T, and with the
    gradient passed through the quantisations dx = q(dy) q(w^T)^T and dw = q(dy^T) q(x^T)^T. Each product's operands are
    quantised along the dimension it sums over, so the backward pass quantises x, w and dy anew from their values."""
    fmt = _format(format)
    _check(x, "x", _HALF)
    _check(w, "w", (x.dtype,), x)
    if w.ndim != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x must be [..., K] and w [N, K], not {tuple(x.shape)} and {tuple(w.shape)}")
    y = _Linear.apply(_rows(x), _rows(w), fmt)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], w.shape[0])


# ---------------------------------------------------------------- the layers between two products
def _coded(x: torch.Tensor, rows: int, cols: int, format: str, scale, grad: bool) -> MicroTensor:
    """The MicroTensor [rows, cols] a layer of x writes to."""
    fmt = _format(format)
    if grad:
        raise ValueError("an output in a microscaled format has no gradient: detach the inputs, or leave format out and "
                         "let micro_linear quantise")
    if fmt == _abi.FMT_NVFP4:
        if scale is None:
            raise ValueError("nvfp4 needs the tensor's scale (calibrated: the output is not known before it is written)")
        _check_scale(scale, x)
    elif scale is not None:
        raise ValueError(f"{format} has no tensor scale")
    return MicroTensor._new(x, fmt, format, rows, cols, scale)


def _norm_forward(x, residual, weight, eps, q, rows, cols):
    h = x if residual is None else _like(x)
    y = _like(x) if q is None else None
    _call(x.get_device(), _entry.rms_norm, _matrix(x), None if residual is None else _matrix(residual), weight.data_ptr(),
          None if residual is None else _matrix(h), None if y is None else _matrix(y), None if q is None else q._raw, rows,
          cols, eps, _HALF[x.dtype])
    return (y if q is None else q), h


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        y, h = _norm_forward(x, residual, weight, eps, None, *x.shape)
        ctx.save_for_backward(h, weight)
        ctx.eps = eps
        return y if residual is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        if dy is None:
            return dh, dh, None, None
        dx, dw = rms_norm_backward(dy, h, weight, ctx.eps, dh=dh)
        return dx, (dx if ctx.needs_input_grad[1] else None), dw, None


def _norm_args(x, weight, residual) -> bool:
    """Whether rms_norm takes them: the checks that rms_norm repeats one by one where they fail."""
    try:
        dtype, index, shape = x.dtype, x.get_device(), x.shape
        return bool(dtype in _HALF and index >= 0 and weight.dtype is dtype and weight.get_device() == index
                and shape and shape[-1:] == weight.shape
                and (residual is None or (residual.dtype is dtype and residual.shape == shape
                                          and residual.get_device() == index)))
    except (AttributeError, TypeError):
        return False


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5,
             format: str | None = None, scale: torch.Tensor | None = None):
    """(y, h): h = x + residual (x itself without one), y = h * weight / sqrt(mean(h^2) + eps) over the last dimension.

    x, residual [..., cols] and weight [cols] are fp16 or bf16, of one type. The norm is that of the fp32 sum; h is the
    sum rounded to the type, the next layer's residual. Without `format` y has x's type and shape and both outputs are
    differentiable. With one, y is a MicroTensor [rows, cols], the next product's operand; nvfp4 then needs the tensor's
    `scale`."""
    if not _norm_args(x, weight, residual):
        _check(x, "x", _HALF)
        _check(weight, "weight", (x.dtype,), x)
        if x.dim() < 1 or weight.shape != x.shape[-1:]:
            raise ValueError(f"weight must be [{x.shape[-1] if x.dim() else '?'}], not {tuple(weight.shape)}")
        _check(residual, "residual", (x.dtype,), x)
        raise ValueError(f"residual is {tuple(residual.shape)}, x {tuple(x.shape)}")
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    grad = (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)) \
        and torch.is_grad_enabled() or forward_ad._current_level >= 0 and _has_tangent(x, weight, residual)
    weight = _weight(weight)
    rows, cols = x2.shape
    if format is not None:
        y, h = _norm_forward(x2, r2, weight, eps, _coded(x2, rows, cols, format, scale, grad), rows, cols)
    elif scale is not None:
        raise ValueError("scale belongs to format='nvfp4'")
    elif grad:
        out = _Norm.apply(x2, r2, weight, eps)
        y, h = (out, x2) if residual is None else out
    else:
        y, h = _norm_forward(x2, r2, weight, eps, None, rows, cols)
    if x2 is not x and x.dim() != 2:
        y = y if format is not None else y.reshape(x.shape)
        h = h.reshape(x.shape)
    return y, (x if residual is None else h)


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                      dh: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight) of rms_norm from the gradient of y and h, the sum it normalised. `dh`: the gradient that arrives at
    h itself (along the residual), added to dx. dx is the gradient of both x and the residual. The sums' order is fixed:
    results repeat bit for bit."""
    _check(h, "h", _HALF)
    _check(dy, "dy", (h.dtype,), h)
    _check(weight, "weight", (h.dtype,), h)
    if dh is not None:
        _check(dh, "dh", (h.dtype,), h)
    if h.dim() < 1 or weight.shape != h.shape[-1:] or dy.shape != h.shape or (dh is not None and dh.shape != h.shape):
        raise ValueError(f"dy {tuple(dy.shape)}, dh and h {tuple(h.shape)} must have one shape, weight "
                         f"{tuple(weight.shape)} its last dimension")
    dy2, h2, dh2 = _rows(dy), _rows(h), None if dh is None else _rows(dh)  # held until the launch: some may be copies
    weight = _weight(weight)
    rows, cols = h2.shape
    n = ctypes.c_size_t(0)
    _abi.check(_abi.load().b2g_micro_rms_norm_workspace(rows, cols, n), "b2g_micro_rms_norm_workspace")
    dx, dw = _like(h2), _like(weight)
    ws = h2.new_empty((n.value,), dtype=torch.uint8)
    _call(h.get_device(), _entry.rms_norm_backward, _matrix(dy2), _matrix(h2), weight.data_ptr(),
          None if dh is None else _matrix(dh2), _matrix(dx), dw.data_ptr(), ws.data_ptr(), n.value, rows, cols, eps,
          _HALF[h.dtype])
    return (dx if h.dim() == 2 else dx.reshape(h.shape)), dw


def _gate_forward(x, q, rows, cols):
    y = x.new_empty((rows, cols)) if q is None else None
    _call(x.get_device(), _entry.silu_mul, _matrix(x), None if y is None else _matrix(y), None if q is None else q._raw,
          rows, cols, _HALF[x.dtype])
    return y if q is None else q


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return _gate_forward(x, None, x.shape[0], x.shape[1] // 2)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return silu_mul_backward(dy, ctx.saved_tensors[0])


def _gate_input(x: torch.Tensor) -> None:
    _check(x, "gate_up", _HALF)
    if x.dim() < 1 or x.shape[-1] % 2:
        raise ValueError(f"gate_up must be [..., 2 * cols] = [gate | up], not {tuple(x.shape)}")


def silu_mul(gate_up: torch.Tensor, format: str | None = None, scale: torch.Tensor | None = None):
    """gate / (1 + exp(-gate)) * up of gate_up [..., 2 * cols] = [gate | up] (fp16 or bf16): values [..., cols] of the
    same type, differentiable, or with `format` a MicroTensor [rows, cols] for the next product (nvfp4 needs `scale`)."""
    _gate_input(gate_up)
    x = _rows(gate_up)
    grad = gate_up.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0 and _has_tangent(gate_up)
    rows, cols = x.shape
    cols //= 2
    if format is not None:
        return _gate_forward(x, _coded(x, rows, cols, format, scale, grad), rows, cols)
    if scale is not None:
        raise ValueError("scale belongs to format='nvfp4'")
    y = _Gate.apply(x) if grad else _gate_forward(x, None, rows, cols)
    return y if x is gate_up or gate_up.dim() == 2 else y.reshape(*gate_up.shape[:-1], cols)


def silu_mul_backward(dy: torch.Tensor, gate_up: torch.Tensor) -> torch.Tensor:
    """The gradient of silu_mul's input [..., 2 * cols] from that of its output."""
    _gate_input(gate_up)
    _check(dy, "dy", (gate_up.dtype,), gate_up)
    cols = gate_up.shape[-1] // 2
    if dy.shape != (*gate_up.shape[:-1], cols):
        raise ValueError(f"dy is {tuple(dy.shape)}, gate_up {tuple(gate_up.shape)}")
    x, dy2 = _rows(gate_up), _rows(dy)  # held until the launch: some may be copies
    dx = _like(x)
    _call(x.get_device(), _entry.silu_mul_backward, _matrix(dy2), _matrix(x), _matrix(dx), x.shape[0], cols,
          _HALF[x.dtype])
    return dx if gate_up.dim() == 2 else dx.reshape(gate_up.shape)


def micro_mlp(x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor, w_gate_up: MicroTensor,
              w_down: MicroTensor, eps: float = 1e-5, scales: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """A feed-forward block for inference: (down(silu_mul(gate_up(norm(x + residual)))), x + residual). w_gate_up
    [2 * F, hidden] and w_down [hidden, F] are quantised weights of one format; the norm and the gate write their outputs
    in it, so no activation is read or written in between but once. `scales`: for nvfp4, the calibrated tensor scales of
    the norm's and the gate's output."""
    if not isinstance(w_gate_up, MicroTensor) or not isinstance(w_down, MicroTensor):
        raise TypeError("w_gate_up and w_down must be MicroTensors (quantize makes them)")
    if w_gate_up.format != w_down.format:
        raise ValueError(f"w_gate_up is {w_gate_up.format}, w_down {w_down.format}: a block needs one format")
    s = scales if scales is not None else (None, None)
    n, h = rms_norm(x, norm_weight, residual=residual, eps=eps, format=w_gate_up.format, scale=s[0])
    g = silu_mul(micro_matmul(n, w_gate_up, dtype=x.dtype), format=w_down.format, scale=s[1])
    y = micro_matmul(g, w_down, dtype=x.dtype)
    return (y if x.dim() == 2 else y.reshape(*x.shape[:-1], w_down.shape[0])), h
