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
leaves may be alive during the capture). As elsewhere with torch, tensors made on another stream have to be ready on the
current one. The product's kernels bound their waits: `check_status()` (from cs464_b200.matmul) raises if one ran out.

The arithmetic of a quantisation is exact: which code and which scale a value gets follows from its bits alone
(include/b2g_micro.h), so results do not depend on the launch. Infinities and NaN make their block's scale NaN, and with
it the block's 32 or 16 values. Products accumulate in fp32 on the tensor cores and round once, to the output's type.
"""
from __future__ import annotations

import ctypes
import math
import weakref

import torch
from torch.autograd.function import once_differentiable

from cs464_b200 import _abi
from cs464_b200.matmul import _STATUS, check_status, status_word  # noqa: F401 (check_status is part of this API)

FORMATS = {"mxfp8": _abi.FMT_MXFP8, "mxfp4": _abi.FMT_MXFP4, "nvfp4": _abi.FMT_NVFP4}
BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}

_VALUES = {torch.float16: _abi.VALUE_F16, torch.bfloat16: _abi.VALUE_BF16, torch.float32: _abi.VALUE_F32}
_HALF = (torch.float16, torch.bfloat16)


def _format(fmt: str) -> int:
    try:
        return FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"format must be one of {', '.join(FORMATS)}, not {fmt!r}") from None


def _matrix(t: torch.Tensor) -> _abi.MicroMatrix:
    return _abi.MicroMatrix(t.data_ptr(), *t.stride())


def _device(t: torch.Tensor, what: str) -> torch.device:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor (there is no CPU path)")
    return t.device


def _values(t: torch.Tensor, what: str, dtypes, dev: torch.device | None = None) -> None:
    _device(t, what)
    if t.dtype not in dtypes:
        raise TypeError(f"{what} must be {' or '.join(str(d)[6:] for d in dtypes)}, not {str(t.dtype)[6:]}")
    if dev is not None and t.device != dev:
        raise ValueError(f"{what} is on {t.device}, the other tensors on {dev}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t as a matrix of rows (its last dimension)."""
    return t if t.ndim == 2 else t.reshape(math.prod(t.shape[:-1]), t.shape[-1])


def _call(dev: torch.device, what: str, *args) -> None:
    """Enqueue an entry point on the current stream of `dev`, with `dev` the current device."""
    fn = getattr(_abi.load(), what)
    if torch.cuda.current_device() == dev.index:
        rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        _abi.check(rc, what)


def _tensor_scale(scale, dev: torch.device) -> torch.Tensor:
    if not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or scale.numel() != 1 or scale.device != dev:
        raise ValueError(f"scale must be a float32 tensor of one element on {dev}")
    return scale


def _aligned(t: torch.Tensor) -> bool:
    return t.data_ptr() % 16 == 0


class MicroTensor:
    """A [rows, cols] matrix in a microscaled format, blocks along the columns.

    `codes`: uint8 [rows, pitch], unit column stride, rows 16 bytes (mxfp8: 32) apart or a multiple of that; two 4-bit
    codes a byte, the lower column in the low bits, what is left of an odd row's last byte zero. `scales`: uint8,
    contiguous, ceil(rows / 128) * ceil(blocks / 4) tiles of 512 bytes in the tensor cores' order (include/b2g_micro.h),
    zero where rows or blocks do not exist. `scale`: nvfp4's fp32 scale of the tensor (one element on the device), which
    other formats do not have. The constructor checks and takes the tensors as they are."""

    __slots__ = ("codes", "scales", "shape", "format", "scale", "_abi")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape, format: str, scale: torch.Tensor | None = None):
        fmt = _format(format)
        rows, cols = (int(n) for n in shape)
        if rows < 0 or cols < 0:
            raise ValueError(f"bad shape {tuple(shape)}")
        dev = _device(codes, "codes")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or scales.device != dev:
            raise ValueError(f"codes and scales must be uint8 tensors on one device, not {codes.dtype} on {dev} and "
                             f"{scales.dtype} on {scales.device}")
        pitch, scale_bytes = _layout(fmt, rows, cols)
        step = 32 if fmt == _abi.FMT_MXFP8 else 16
        if rows and cols:
            if (codes.ndim != 2 or codes.shape[0] != rows or codes.shape[1] < pitch or codes.stride(1) != 1
                    or (rows > 1 and (codes.stride(0) < pitch or codes.stride(0) % step)) or not _aligned(codes)):
                raise ValueError(f"codes of a {rows}x{cols} {format} tensor must be [{rows}, >= {pitch}] bytes, 16-byte "
                                 f"aligned, rows a multiple of {step} bytes apart, not {tuple(codes.shape)} with strides "
                                 f"{codes.stride()}")
            if scales.numel() != scale_bytes or not scales.is_contiguous() or not _aligned(scales):
                raise ValueError(f"scales of a {rows}x{cols} {format} tensor must be {scale_bytes} contiguous, 16-byte "
                                 f"aligned bytes, not {tuple(scales.shape)} with strides {scales.stride()}")
        if fmt == _abi.FMT_NVFP4:
            _tensor_scale(scale, dev)
        elif scale is not None:
            raise ValueError(f"{format} has no tensor scale")
        self.codes, self.scales, self.shape, self.format, self.scale = codes, scales, (rows, cols), format, scale
        self._abi = _abi.MicroTensor(fmt, 0, rows, cols, codes.data_ptr(), codes.stride(0) if rows > 1 else pitch,
                                     scales.data_ptr(), scale.data_ptr() if scale is not None else None)

    @classmethod
    def empty(cls, shape, format: str, device, scale: torch.Tensor | None = None) -> "MicroTensor":
        """Uninitialised storage for a [rows, cols] tensor, for a kernel to fill."""
        rows, cols = shape
        pitch, scale_bytes = _layout(_format(format), rows, cols)
        codes = torch.empty((rows, pitch), dtype=torch.uint8, device=device)
        return cls(codes, torch.empty(scale_bytes, dtype=torch.uint8, device=device), shape, format, scale)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return dequantize(self, dtype)

    def code_values(self) -> torch.Tensor:
        """mxfp8's codes as float8_e4m3fn [rows, cols], a view. (4-bit codes have no torch type: `dequantize`.)"""
        if self.format != "mxfp8":
            raise TypeError(f"{self.format} codes are packed; dequantize() gives their values")
        return self.codes[:, :self.shape[1]].view(torch.float8_e4m3fn)

    def scale_tiles(self) -> torch.Tensor:
        """The block scales as float8_e8m0fnu (nvfp4: float8_e4m3fn), a view [row tile, 4, 32, block tile, 4]: row
        128 t + 32 i + j and block 4 u + v at [t, i, j, u, v]."""
        rows, cols = self.shape
        tiles = self.scales.view(-(-rows // 128), -(-cols // (4 * BLOCK[self.format])), 32, 4, 4)
        kind = torch.float8_e4m3fn if self.format == "nvfp4" else torch.float8_e8m0fnu
        return tiles.permute(0, 3, 2, 1, 4).view(kind)

    def __repr__(self) -> str:
        return f"MicroTensor({self.shape[0]}x{self.shape[1]}, {self.format}, {self.device})"


def _layout(fmt: int, rows: int, cols: int) -> tuple[int, int]:
    """(pitch, scale bytes) of a tensor: b2g_micro_layout."""
    block = 16 if fmt == _abi.FMT_NVFP4 else 32
    return (-(-cols // 32) * (32 if fmt == _abi.FMT_MXFP8 else 16),
            -(-rows // 128) * -(-cols // (4 * block)) * 512)


def quantize(x: torch.Tensor, format: str = "mxfp8", scale: torch.Tensor | None = None) -> MicroTensor:
    """x [rows, cols] (fp16, bf16 or fp32, any strides) in a microscaled format, blocks along the columns.

    nvfp4: `scale` is the tensor's fp32 scale, one positive element on the device; values past 2688 times it saturate.
    Without it, x is read twice: its scale becomes the smallest power of two at which nothing saturates."""
    fmt = _format(format)
    _values(x, "x", tuple(_VALUES))
    if x.ndim != 2:
        raise ValueError(f"x must be a matrix, not {tuple(x.shape)}")
    x = x.detach()
    dev = x.device
    mat = _matrix(x)
    if fmt == _abi.FMT_NVFP4:
        if scale is None:
            scale = torch.empty(1, dtype=torch.float32, device=dev)
            _call(dev, "b2g_micro_tensor_scale", mat, x.shape[0], x.shape[1], _VALUES[x.dtype], scale.data_ptr())
        else:
            _tensor_scale(scale, dev)
    elif scale is not None:
        raise ValueError(f"{format} has no tensor scale")
    q = MicroTensor.empty(tuple(x.shape), format, dev, scale)
    _call(dev, "b2g_micro_quantize", mat, _VALUES[x.dtype], q._abi)
    return q


def dequantize(q: MicroTensor, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of q: code * block scale (* tensor scale), rounded to `dtype` (fp16, bf16 or fp32). `out`: a tensor of
    q's shape to write them to instead, with any strides that do not overlap; its type is used."""
    if out is None:
        if dtype not in _VALUES:
            raise TypeError(f"dtype must be float16, bfloat16 or float32, not {dtype}")
        out = torch.empty(q.shape, dtype=dtype, device=q.device)
    else:
        _values(out, "out", tuple(_VALUES), q.device)
        if tuple(out.shape) != q.shape:
            raise ValueError(f"out must be {q.shape[0]}x{q.shape[1]}, not {tuple(out.shape)}")
    _call(q.device, "b2g_micro_dequantize", q._abi, _matrix(out), _VALUES[out.dtype])
    return out


# ---------------------------------------------------------------- products
def _status(dev: torch.device) -> torch.Tensor:
    if dev.index not in _STATUS and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"the first product on {dev} makes the device's status word, which a stream capture cannot "
                           "hold: run a product there once before the capture")
    return status_word(dev)


def _output(a: MicroTensor, b: MicroTensor, out: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    if not isinstance(a, MicroTensor) or not isinstance(b, MicroTensor):
        raise TypeError("a and b must be MicroTensors (quantize makes them)")
    if a.device != b.device:
        raise ValueError(f"a is on {a.device}, b on {b.device}")
    if a.format != b.format:
        raise ValueError(f"a is {a.format}, b {b.format}: a product needs one format")
    if a.shape[1] != b.shape[1]:
        raise ValueError(f"a is {a.shape[0]}x{a.shape[1]}, b {b.shape[0]}x{b.shape[1]}: their columns are summed over and "
                         "must agree")
    M, N = a.shape[0], b.shape[0]
    if out is None:
        if dtype not in _HALF:
            raise TypeError(f"dtype must be float16 or bfloat16, not {dtype}")
        return torch.empty((M, N), dtype=dtype, device=a.device)
    _values(out, "out", _HALF, a.device)
    if tuple(out.shape) != (M, N) or (N > 1 and out.stride(1) != 1) or (M > 1 and out.stride(0) < N):
        raise ValueError(f"out must be a {M}x{N} tensor with unit column stride and rows that do not overlap, not "
                         f"{tuple(out.shape)} with strides {out.stride()}")
    return out


def _ldc(c: torch.Tensor) -> int:
    return max(c.stride(0), c.shape[1])  # the row stride of a single row may be anything


def micro_matmul(a: MicroTensor, b: MicroTensor, out: torch.Tensor | None = None,
                 dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """C[M, N] = A[M, K] @ B[N, K].T on the current stream, C in `dtype` (fp16 or bf16), or into `out` (unit column
    stride, any row stride) in its type."""
    c = _output(a, b, out, dtype)
    dev = a.device
    _call(dev, "b2g_micro_matmul", a._abi, b._abi, c.data_ptr(), _ldc(c), _VALUES[c.dtype], _status(dev).data_ptr())
    return c


class _MicroRunner:
    """The closure MicroMatmul.make_runner returns: calling it enqueues the product and returns C."""

    __slots__ = ("_plan", "_device", "c", "status", "_keep", "_fin", "__weakref__")

    def __init__(self, plan: ctypes.c_void_p, c: torch.Tensor, status: torch.Tensor, keep):
        self._plan, self._device, self.c, self.status, self._keep = plan, c.device, c, status, keep
        self._fin = weakref.finalize(self, _abi.load().b2g_micro_plan_destroy, plan)

    def __call__(self) -> torch.Tensor:
        _call(self._device, "b2g_micro_plan_launch", self._plan)
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

    def __init__(self, dtype: torch.dtype = torch.bfloat16):
        if dtype not in _HALF:
            raise TypeError(f"dtype must be float16 or bfloat16, not {dtype}")
        self.dtype = dtype

    def make_runner(self, a: MicroTensor, b: MicroTensor, out: torch.Tensor | None = None) -> _MicroRunner:
        c = _output(a, b, out, self.dtype)
        plan = ctypes.c_void_p()
        with torch.cuda.device(a.device):
            status = torch.zeros(1, dtype=torch.int32, device=a.device)
            _abi.check(_abi.load().b2g_micro_plan_create(a._abi, b._abi, c.data_ptr(), _ldc(c), _VALUES[c.dtype],
                                                         status.data_ptr(), ctypes.byref(plan)), "b2g_micro_plan_create")
        return _MicroRunner(plan, c, status, (a, b))


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, fmt):
        ctx.save_for_backward(x, w)
        ctx.fmt = fmt
        return micro_matmul(quantize(x, fmt), quantize(w, fmt), dtype=x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        fmt, dx, dw = ctx.fmt, None, None
        if ctx.needs_input_grad[0]:
            dx = micro_matmul(quantize(dy, fmt), quantize(w.t(), fmt), dtype=x.dtype)
        if ctx.needs_input_grad[1]:
            dw = micro_matmul(quantize(dy.t(), fmt), quantize(x.t(), fmt), dtype=w.dtype)
        return dx, dw, None


def micro_linear(x: torch.Tensor, w: torch.Tensor, format: str = "mxfp8") -> torch.Tensor:
    """x [..., K] @ w [N, K].T (fp16 or bf16, one type), differentiable, in a format: y = q(x) q(w)^T, and with the
    gradient passed through the quantisations dx = q(dy) q(w^T)^T and dw = q(dy^T) q(x^T)^T. Each product's operands are
    quantised along the dimension it sums over, so the backward pass quantises x, w and dy anew from their values."""
    _format(format)
    _values(x, "x", _HALF)
    _values(w, "w", (x.dtype,), x.device)
    if w.ndim != 2 or x.ndim < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x must be [..., K] and w [N, K], not {tuple(x.shape)} and {tuple(w.shape)}")
    y = _Linear.apply(_rows(x), w, format)
    return y if x.ndim == 2 else y.reshape(*x.shape[:-1], w.shape[0])


# ---------------------------------------------------------------- the layers between two products
def _coded(x: torch.Tensor, cols: int, format: str | None, scale, tensors) -> MicroTensor | None:
    """The MicroTensor a layer writes to, or None for values."""
    if format is None:
        if scale is not None:
            raise ValueError("scale belongs to format='nvfp4'")
        return None
    fmt = _format(format)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("an output in a microscaled format has no gradient: detach the inputs, or leave format out and "
                         "let micro_linear quantise")
    if fmt == _abi.FMT_NVFP4:
        if scale is None:
            raise ValueError("nvfp4 needs the tensor's scale (calibrated: the output is not known before it is written)")
        _tensor_scale(scale, x.device)
    elif scale is not None:
        raise ValueError(f"{format} has no tensor scale")
    return MicroTensor.empty((x.shape[0], cols), format, x.device, scale)


def _ref(m: torch.Tensor | None):
    return None if m is None else _matrix(m)


def _norm_forward(x, residual, weight, eps, q):
    h = x if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if q is None else None
    _call(x.device, "b2g_micro_rms_norm", _matrix(x), _ref(residual), weight.data_ptr(),
          None if residual is None else _matrix(h), _ref(y), None if q is None else q._abi, x.shape[0], x.shape[1], eps,
          _VALUES[x.dtype])
    return (y if q is None else q), h


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        ctx.set_materialize_grads(False)
        y, h = _norm_forward(x, residual, weight, eps, None)
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


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5,
             format: str | None = None, scale: torch.Tensor | None = None):
    """(y, h): h = x + residual (x itself without one), y = h * weight / sqrt(mean(h^2) + eps) over the last dimension.

    x, residual [..., cols] and weight [cols] are fp16 or bf16, of one type. The norm is that of the fp32 sum; h is the
    sum rounded to the type, the next layer's residual. Without `format` y has x's type and shape and both outputs are
    differentiable. With one, y is a MicroTensor [rows, cols], the next product's operand; nvfp4 then needs the tensor's
    `scale`."""
    _values(x, "x", _HALF)
    _values(weight, "weight", (x.dtype,), x.device)
    if x.ndim < 1 or weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must be [{x.shape[-1] if x.ndim else '?'}], not {tuple(weight.shape)}")
    if residual is not None:
        _values(residual, "residual", (x.dtype,), x.device)
        if residual.shape != x.shape:
            raise ValueError(f"residual is {tuple(residual.shape)}, x {tuple(x.shape)}")
    x2 = _rows(x)
    r2 = None if residual is None else _rows(residual)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    q = _coded(x2, x2.shape[1], format, scale, (x, weight, residual))
    if q is None and torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (
            residual is not None and residual.requires_grad)):
        out = _Norm.apply(x2, r2, weight, eps)
        y, h = (out, x2) if residual is None else out
    else:
        y, h = _norm_forward(x2, r2, weight, eps, q)
    if q is None and x.ndim != 2:
        y = y.reshape(x.shape)
    return y, (x if residual is None else h if x.ndim == 2 else h.reshape(x.shape))


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                      dh: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight) of rms_norm from the gradient of y and h, the sum it normalised. `dh`: the gradient that arrives at
    h itself (along the residual), added to dx. dx is the gradient of both x and the residual. The sums' order is fixed:
    results repeat bit for bit."""
    _values(h, "h", _HALF)
    for t, what in ((dy, "dy"), (weight, "weight"), (dh, "dh")):
        if t is not None:
            _values(t, what, (h.dtype,), h.device)
    if h.ndim < 1 or weight.shape != h.shape[-1:] or dy.shape != h.shape or (dh is not None and dh.shape != h.shape):
        raise ValueError(f"dy {tuple(dy.shape)}, dh and h {tuple(h.shape)} must have one shape, weight "
                         f"{tuple(weight.shape)} its last dimension")
    dy2, h2 = _rows(dy.detach()), _rows(h.detach())
    dh2 = None if dh is None else _rows(dh.detach())
    weight = weight.detach().contiguous()
    rows, cols = h2.shape
    dev = h.device
    n = ctypes.c_size_t(0)
    _abi.check(_abi.load().b2g_micro_rms_norm_workspace(rows, cols, ctypes.byref(n)), "b2g_micro_rms_norm_workspace")
    ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
    dx = torch.empty((rows, cols), dtype=h.dtype, device=dev)
    dw = torch.empty(cols, dtype=h.dtype, device=dev)
    _call(dev, "b2g_micro_rms_norm_backward", _matrix(dy2), _matrix(h2), weight.data_ptr(), _ref(dh2), _matrix(dx),
          dw.data_ptr(), ws.data_ptr(), n.value, rows, cols, eps, _VALUES[h.dtype])
    return (dx if h.ndim == 2 else dx.reshape(h.shape)), dw


def _gate_forward(x, q):
    cols = x.shape[1] // 2
    y = torch.empty((x.shape[0], cols), dtype=x.dtype, device=x.device) if q is None else None
    _call(x.device, "b2g_micro_silu_mul", _matrix(x), _ref(y), None if q is None else q._abi, x.shape[0], cols,
          _VALUES[x.dtype])
    return y if q is None else q


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return _gate_forward(x, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return silu_mul_backward(dy, ctx.saved_tensors[0])


def _gate_input(x: torch.Tensor) -> None:
    _values(x, "gate_up", _HALF)
    if x.ndim < 1 or x.shape[-1] % 2:
        raise ValueError(f"gate_up must be [..., 2 * cols] = [gate | up], not {tuple(x.shape)}")


def silu_mul(gate_up: torch.Tensor, format: str | None = None, scale: torch.Tensor | None = None):
    """gate / (1 + exp(-gate)) * up of gate_up [..., 2 * cols] = [gate | up] (fp16 or bf16): values [..., cols] of the
    same type, differentiable, or with `format` a MicroTensor [rows, cols] for the next product (nvfp4 needs `scale`)."""
    _gate_input(gate_up)
    x = _rows(gate_up)
    q = _coded(x, x.shape[1] // 2, format, scale, (gate_up,))
    y = _Gate.apply(x) if q is None and torch.is_grad_enabled() and gate_up.requires_grad else _gate_forward(x, q)
    return y if q is not None or gate_up.ndim == 2 else y.reshape(*gate_up.shape[:-1], x.shape[1] // 2)


def silu_mul_backward(dy: torch.Tensor, gate_up: torch.Tensor) -> torch.Tensor:
    """The gradient of silu_mul's input [..., 2 * cols] from that of its output."""
    _gate_input(gate_up)
    _values(dy, "dy", (gate_up.dtype,), gate_up.device)
    cols = gate_up.shape[-1] // 2
    if dy.shape != (*gate_up.shape[:-1], cols):
        raise ValueError(f"dy is {tuple(dy.shape)}, gate_up {tuple(gate_up.shape)}")
    dy2, x = _rows(dy.detach()), _rows(gate_up.detach())
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _call(x.device, "b2g_micro_silu_mul_backward", _matrix(dy2), _matrix(x), _matrix(dx), x.shape[0], cols,
          _VALUES[x.dtype])
    return dx if gate_up.ndim == 2 else dx.reshape(gate_up.shape)


def micro_mlp(x: torch.Tensor, residual: torch.Tensor | None, norm_weight: torch.Tensor, w_gate_up: MicroTensor,
              w_down: MicroTensor, eps: float = 1e-5, scales: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """A feed-forward block for inference: (down(silu_mul(gate_up(norm(x + residual)))), x + residual). w_gate_up
    [2 * F, hidden] and w_down [hidden, F] are quantised weights of one format; the norm and the gate write their outputs
    in it, so no activation is read or written in between but once. `scales`: for nvfp4, the calibrated tensor scales of
    the norm's and the gate's output."""
    if w_gate_up.format != w_down.format:
        raise ValueError(f"w_gate_up is {w_gate_up.format}, w_down {w_down.format}: a block needs one format")
    s = scales if scales is not None else (None, None)
    n, h = rms_norm(x, norm_weight, residual=residual, eps=eps, format=w_gate_up.format, scale=s[0])
    g = silu_mul(micro_matmul(n, w_gate_up, dtype=x.dtype), format=w_down.format, scale=s[1])
    y = micro_matmul(g, w_down, dtype=x.dtype)
    return (y if x.ndim == 2 else y.reshape(*x.shape[:-1], w_down.shape[0])), h
