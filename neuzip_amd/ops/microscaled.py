"""Weights in microscaled 4 bits, and the products with them.

Beside the entropy-coded weights of a :class:`~neuzip_amd.Manager` (any number
of kept mantissa bits, decoded before or inside a product) stand weights in the
form that the matrix cores multiply as it is: blocks of 32 values along a row
share a power of two, a value is an e2m1 number times that (4.25 bits per
value).  Activation rows are brought to 8 bits (e4m3, blocks of 32 likewise) on
the way into a product.  Results are rounded once, float32 ones from sums in 32
bits; for 16-bit results the matrix instruction adds eight products at a time,
each cut off below 2^-12 of the largest of the eight, and 32 bits hold the rest
(:func:`mx_linear`).  include/neuzip_hip.h states both and the format to the bit.

The kernels are part of libneuzip_hip.so; there is no fallback without a GPU.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from neuzip_amd import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


def _dtype_code(dtype: torch.dtype) -> int:
    code = _DTYPES.get(dtype)
    if code is None:
        raise RuntimeError("Unsupported data type")
    return code


# These calls take a few microseconds on the device: what surrounds them is kept short as well.  (The stream's
# address and the current device are asked for directly, 2 us less a call than through torch.cuda.)
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_tracing = torch._C._get_tracing_state
_modes = torch._C._len_torch_dispatch_stack
_PROXY = torch._C._TorchDispatchModeKey.PROXY


def _refuse_unseen(tensors) -> None:
    """Raise where a native call would be passed by in silence: a trace (of torch.jit or make_fx) would hold the
    allocation of the result only, and a tangent would end here."""
    if _tracing() is not None or torch._C._get_dispatch_mode(_PROXY) is not None:
        raise RuntimeError("this call cannot be traced: it writes its result through an address")
    if forward_ad._current_level >= 0:
        for t in tensors.values():
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("forward-mode differentiation is not supported by this call")


def _on_gpu(**tensors) -> int:
    """The index of the device that all of ``tensors`` (None aside) are on, which has to be a GPU."""
    if forward_ad._current_level >= 0 or _modes() or _tracing() is not None:
        _refuse_unseen(tensors)
    index = None
    for name, t in tensors.items():
        if t is None:
            continue
        at = t.get_device()
        if at < 0:
            raise ValueError(f"{name} must be on the GPU")
        if index is not None and at != index:
            raise ValueError(f"{name} is on {t.device}, not on cuda:{index} like the tensors before it")
        index = at
    return index


def _call(fn, index: int, *args) -> None:
    """Make a native call on the current stream of device ``index``."""
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:  # a launch goes to the device that is current
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.raise_for(rc)


def _ask(fn, index: int, *args) -> int:
    """What a native call answers for device ``index``, whose compute units count."""
    if index == _current_device():
        return fn(*args)
    with torch.cuda.device(index):
        return fn(*args)


def _as_rows(t: torch.Tensor, width: int):
    """``t`` as rows of ``width`` elements that lie next to each other (a copy only where no view does it): the
    tensor, its rows, elements from row to row."""
    if t.is_contiguous():
        n = t.numel()
        if n != 1 or not t.is_neg():
            return t, n // width if width else math.prod(t.shape[:-1]), width
    rows = t.resolve_neg().reshape(-1, width)  # its memory may hold the values with the other sign
    if rows.stride(1) != 1 and width > 1:
        rows = rows.contiguous()
    return rows, rows.shape[0], rows.stride(0)


# What sizes alone decide is asked of the library once.
@lru_cache(maxsize=1024)
def _row_sizes(cols: int, bits: int):
    """Bytes of a row's codes and of its scales."""
    L = _lib.load()
    return L.nz_mx_row_bytes(cols, bits), L.nz_mx_scale_bytes(cols)


@lru_cache(maxsize=1024)
def _product_room(index: int, m: int, n: int, k: int, code: int) -> int:
    return _ask(_lib.load().nz_mx_linear_workspace_bytes, index, m, n, k, code)


@lru_cache(maxsize=1024)
def _table_room(count: int, cols: int) -> int:
    return _lib.load().nz_embedding_gradient_workspace_bytes(count, cols)


def _workspace(room: int, like: torch.Tensor):
    """(the tensor that keeps it, its address)"""
    if not room:
        return None, None
    ws = like.new_empty(room, dtype=torch.uint8)
    return ws, ws.data_ptr()


class MXTensor:
    """A matrix (or a stack of rows) held in microscaled 4 or 8 bits.

    ``data`` and ``scales`` are the uint8 tensors of the stored form
    (include/neuzip_hip.h), one row per row of the matrix; ``shape`` is the
    shape of the values.  Made by :func:`mx_quantize`, or from stored tensors.
    """

    __slots__ = ("data", "scales", "bits", "shape")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape, bits: int = 4) -> None:
        shape = torch.Size(shape)
        if bits not in (4, 8):
            raise ValueError("bits must be 4 or 8")
        if len(shape) < 1:
            raise ValueError("a microscaled tensor has one dimension at least")
        rows, sizes = math.prod(shape[:-1]), _row_sizes(shape[-1], bits)
        for name, t, size in (("data", data, (rows, sizes[0])), ("scales", scales, (rows, sizes[1]))):
            if t.dtype != torch.uint8 or tuple(t.shape) != size or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 tensor of shape {size}")
        if data.device != scales.device:
            raise ValueError("data and scales must be on one device")
        self.data, self.scales, self.shape, self.bits = data, scales, shape, bits

    @classmethod
    def _of(cls, data, scales, shape, bits) -> "MXTensor":
        """the same of tensors that are known to fit"""
        self = object.__new__(cls)
        self.data, self.scales, self.shape, self.bits = data, scales, shape, bits
        return self

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        """bytes held"""
        return self.data.numel() + self.scales.numel()

    def to(self, device) -> "MXTensor":
        return MXTensor(self.data.to(device), self.scales.to(device), self.shape, self.bits)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values as a dense tensor (bfloat16 holds all of them without rounding, subnormals aside)."""
        code = _dtype_code(dtype)
        data = self.data
        index = _on_gpu(data=data)
        out = data.new_empty(self.shape, dtype=dtype)
        _call(_lib.load().nz_mx_dequantize, index, data.data_ptr(), self.scales.data_ptr(), data.shape[0],
              self.shape[-1], self.bits, out.data_ptr(), code)
        return out

    def __repr__(self) -> str:
        return f"MXTensor(shape={tuple(self.shape)}, bits={self.bits}, device={self.device})"


def mx_quantize(x: torch.Tensor, bits: int = 4) -> MXTensor:
    """``x`` (bfloat16, float16 or float32, on the GPU) in microscaled form:
    blocks of 32 values along the last axis share a power of two, values are
    rounded to the nearest e2m1 (``bits=4``) or e4m3 (``bits=8``) number, ties to
    the even code.  A block that holds a NaN or an infinity reads as NaN.  Autograd
    does not record it."""
    if bits not in (4, 8):
        raise ValueError("bits must be 4 or 8")
    code = _dtype_code(x.dtype)
    index = _on_gpu(x=x)
    shape = x.shape
    if not shape:
        raise ValueError("x must have one dimension at least")
    cols = shape[-1]
    rows, n, stride = _as_rows(x, cols)
    sizes = _row_sizes(cols, bits)
    data = x.new_empty((n, sizes[0]), dtype=torch.uint8)
    scales = x.new_empty((n, sizes[1]), dtype=torch.uint8)
    _call(_lib.load().nz_mx_quantize, index, rows.data_ptr(), code, n, cols, stride, bits, data.data_ptr(),
          scales.data_ptr())
    return MXTensor._of(data, scales, shape, bits)


def _check_weight(weight) -> None:
    if not isinstance(weight, MXTensor) or weight.bits != 4 or len(weight.shape) != 2:
        raise ValueError("weight must be a matrix in microscaled 4 bits (mx_quantize)")


def _product(x, weight: MXTensor, bias, dtype: torch.dtype) -> torch.Tensor:
    L = _lib.load()
    n, k = weight.shape
    code, wd = _dtype_code(dtype), weight.data
    held = isinstance(x, MXTensor)
    xt = x.data if held else x
    index = _on_gpu(x=xt, weight=wd, bias=bias)
    y = xt.new_empty((*x.shape[:-1], n), dtype=dtype)
    if k == 0:  # empty sums
        return y.copy_(bias) if bias is not None else y.zero_()
    b = None
    if bias is not None:
        bias = bias.contiguous()
        if n == 1:
            bias = bias.resolve_neg()
        b = bias.data_ptr()
    if held:
        m = xt.shape[0]
    else:
        xt, m, stride = _as_rows(x, k)
    room = _product_room(index, m, n, k, code)
    ws, at = _workspace(room, xt)
    if held:
        _call(L.nz_mx_linear_rows8, index, xt.data_ptr(), x.scales.data_ptr(), m, k, wd.data_ptr(),
              weight.scales.data_ptr(), n, b, y.data_ptr(), code, at, room)
    else:
        _call(L.nz_mx_linear, index, xt.data_ptr(), code, m, k, stride, wd.data_ptr(), weight.scales.data_ptr(), n, b,
              y.data_ptr(), at, room)
    return y


def _input_gradient(grad: torch.Tensor, weight: MXTensor) -> torch.Tensor:
    L = _lib.load()
    n, k = weight.shape
    index = _on_gpu(weight=weight.data, grad=grad)
    dx = grad.new_empty((*grad.shape[:-1], k))
    if n == 0:  # empty sums
        return dx.zero_()
    rows, m, stride = _as_rows(grad, n)
    args = (rows.data_ptr(), _dtype_code(grad.dtype), m, n, stride)
    room = _ask(L.nz_mx_linear_grad_workspace_bytes, index, *args, k)
    ws, at = _workspace(room, rows)
    _call(L.nz_mx_linear_grad, index, *args, weight.data.data_ptr(), weight.scales.data_ptr(), k, dx.data_ptr(), at,
          room)
    return dx


def _bias_gradient(grad: torch.Tensor, n: int) -> torch.Tensor:
    L, index = _lib.load(), _on_gpu(grad=grad)
    rows, m, stride = _as_rows(grad, n)
    out = rows.new_empty(n)
    room = L.nz_column_sums_workspace_bytes(m, n)
    ws, at = _workspace(room, rows)
    _call(L.nz_column_sums, index, rows.data_ptr(), _dtype_code(grad.dtype), m, n, stride, out.data_ptr(), at, room)
    return out


class MicroscaledLinear(torch.autograd.Function):
    """``y = x W^T (+ b)`` with a frozen weight in 4 bits.  Backward gives the
    gradients of ``x`` (the rounding of its rows to 8 bits is passed straight
    through) and of the bias."""

    @staticmethod
    def forward(ctx, x, weight, bias, dtype):
        ctx.weight = weight
        if ctx.needs_input_grad[0] and not weight.data.is_inference():  # an inference tensor has no version to check
            ctx.save_for_backward(weight.data, weight.scales)
        return _product(x, weight, bias, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        grad_x = grad_b = None
        if ctx.needs_input_grad[0]:
            weight, held = ctx.weight, ctx.saved_tensors  # raises if the weight has been written to since
            if held and (held[0] is not weight.data or held[1] is not weight.scales):  # a hook's
                weight = MXTensor(*held, weight.shape, weight.bits)
            grad_x = _input_gradient(grad_output, weight)
        if ctx.needs_input_grad[2]:
            grad_b = _bias_gradient(grad_output, ctx.weight.shape[0])
        return grad_x, None, grad_b, None


def mx_linear(x, weight: MXTensor, bias=None, dtype=None) -> torch.Tensor:
    """``x @ W^T (+ bias)`` for a weight ``[out, in]`` in microscaled 4 bits.

    ``x`` is a tensor ``[..., in]`` (bfloat16, float16 or float32), whose rows are
    brought to 8 bits on the way and whose type the result has; or an
    :class:`MXTensor` of 8 bits (rows that several weights share), with a result
    of type ``dtype`` (bfloat16).  ``bias`` has the type of the result.  Autograd
    records the gradients of ``x`` and ``bias``; the weight is frozen.

    A bfloat16 or float16 result may lack, of each product, what lies below 2^-12 of the
    largest of the eight consecutive products that it is added with: usually far
    below its own rounding, but not where large products cancel.  A float32 result is
    summed in 32 bits throughout, from the same rows with
    ``mx_linear(mx_quantize(x, 8), weight, dtype=torch.float32)`` (1.3 to 1.6 times the
    time of a few such rows, 2.5 times that of many)."""
    _check_weight(weight)
    n, k = weight.shape
    if isinstance(x, MXTensor):
        if x.bits != 8:
            raise ValueError("activation rows are held in 8 bits (mx_quantize(x, 8))")
        dtype = torch.bfloat16 if dtype is None else dtype
    else:
        if x.dim() < 1:
            raise ValueError("x must have one dimension at least")
        if dtype is not None and dtype != x.dtype:
            raise ValueError("the result has the type of x")
        dtype = x.dtype
    _dtype_code(dtype)
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, the weight {k}")
    if bias is not None and (tuple(bias.shape) != (n,) or bias.dtype != dtype):
        raise ValueError(f"bias must be a {dtype} tensor of {n} elements")
    if torch.is_grad_enabled() and (not isinstance(x, MXTensor) and x.requires_grad
                                    or bias is not None and bias.requires_grad):
        return MicroscaledLinear.apply(x, weight, bias, dtype)
    return _product(x, weight, bias, dtype)


def mx_embedding(indices: torch.Tensor, table: MXTensor, scale: float = 1.0, dtype: torch.dtype = torch.bfloat16,
                 status=None) -> torch.Tensor:
    """Rows ``indices`` (any integer shape) of a table in microscaled form, times
    ``scale`` in 32 bits, rounded to ``dtype``.  An index outside the table gives a row
    of zeros and sets bit 0 of ``status`` (an int32 tensor of one element).  The table is
    frozen: autograd has nothing to record."""
    if not isinstance(table, MXTensor) or len(table.shape) != 2:
        raise ValueError("table must be a matrix in microscaled form (mx_quantize)")
    if indices.dtype not in (torch.int64, torch.int32):
        raise ValueError("indices must be int64 or int32")
    code = _dtype_code(dtype)
    data = table.data
    index = _on_gpu(table=data, indices=indices, status=status)
    at = None
    if status is not None:
        if status.dtype != torch.int32 or status.numel() != 1:
            raise ValueError("status must be an int32 tensor of one element")
        at = status.data_ptr()
    idx = indices if indices.dtype == torch.int64 else indices.to(torch.int64)
    idx = idx.contiguous()
    rows, cols = table.shape
    out = data.new_empty((*indices.shape, cols), dtype=dtype)
    _call(_lib.load().nz_mx_lookup, index, data.data_ptr(), table.scales.data_ptr(), rows, cols, table.bits,
          idx.data_ptr(), idx.numel(), float(scale), out.data_ptr(), code, at)
    if status is not None:
        increment_version(status)
    return out
