"""Tensors in 8 bits with a scale for each block of 128: weights that are multiplied
as they are, and activations that a training step keeps for its backward pass.

A value is an e4m3 number times a power of two that its block shares: 128 values of
a row (activations) or 128 rows of 128 columns (weights), 1.01 bytes a value.  The
matrix cores take such rows as they are.  What a layer keeps for the gradient of its
weight (:func:`fp8_weight_gradient`), and an activation function for its own
(:func:`fp8_activation`), is half of what it is in 16 bits: these gradients are those
of the formulas at the kept values.  include/neuzip_hip.h states the format and the
sums to the bit.

The kernels are part of libneuzip_hip.so; there is no fallback without a GPU.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from neuzip_amd import _lib
from neuzip_amd.ops.microscaled import _as_rows, _ask, _bias_gradient, _call, _dtype_code, _on_gpu, _workspace

_KINDS = {"gelu": _lib.ACTIVATION_GELU, "gelu_tanh": _lib.ACTIVATION_GELU_TANH, "silu": _lib.ACTIVATION_SILU}


# What sizes alone decide is asked of the library once.
@lru_cache(maxsize=1024)
def _row_sizes(cols: int):
    """Bytes of a row's codes and of its scales."""
    L = _lib.load()
    return L.nz_fp8_row_bytes(cols), L.nz_fp8_scale_bytes(cols)


@lru_cache(maxsize=1024)
def _product_room(index: int, m: int, n: int, k: int, code: int) -> int:
    return _ask(_lib.load().nz_fp8_linear_workspace_bytes, index, m, n, k, code)


class FP8Tensor:
    """A matrix (or a stack of rows) held in 8 bits, with a scale for 128 values of a
    row (``block_rows=1``) or for 128 rows of 128 columns (``block_rows=128``).

    ``data`` and ``scales`` are the uint8 tensors of the stored form
    (include/neuzip_hip.h); ``shape`` is the shape of the values.  Made by
    :func:`fp8_quantize`, or from stored tensors.
    """

    __slots__ = ("data", "scales", "block_rows", "shape")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, shape, block_rows: int = 1) -> None:
        shape = torch.Size(shape)
        if block_rows not in (1, 128):
            raise ValueError("block_rows must be 1 or 128")
        if len(shape) < 1:
            raise ValueError("a tensor in 8 bits has one dimension at least")
        rows, sizes = math.prod(shape[:-1]), _row_sizes(shape[-1])
        for name, t, size in (("data", data, (rows, sizes[0])), ("scales", scales, (-(-rows // block_rows), sizes[1]))):
            if t.dtype != torch.uint8 or tuple(t.shape) != size or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous uint8 tensor of shape {size}")
        if data.device != scales.device:
            raise ValueError("data and scales must be on one device")
        self.data, self.scales, self.shape, self.block_rows = data, scales, shape, block_rows

    @classmethod
    def _of(cls, data, scales, shape, block_rows) -> "FP8Tensor":
        """the same of tensors that are known to fit"""
        self = object.__new__(cls)
        self.data, self.scales, self.shape, self.block_rows = data, scales, shape, block_rows
        return self

    @property
    def device(self) -> torch.device:
        return self.data.device

    @property
    def nbytes(self) -> int:
        """bytes held"""
        return self.data.numel() + self.scales.numel()

    def to(self, device) -> "FP8Tensor":
        return FP8Tensor(self.data.to(device), self.scales.to(device), self.shape, self.block_rows)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values as a dense tensor (bfloat16 holds all of them without rounding, subnormals aside, and an infinity
        for 2^128, as which magnitudes above 3.29e38 are held)."""
        code = _dtype_code(dtype)
        data = self.data
        index = _on_gpu(data=data)
        out = data.new_empty(self.shape, dtype=dtype)
        _call(_lib.load().nz_fp8_dequantize, index, data.data_ptr(), self.scales.data_ptr(), data.shape[0],
              self.shape[-1], self.block_rows, out.data_ptr(), code)
        return out

    def __repr__(self) -> str:
        return f"FP8Tensor(shape={tuple(self.shape)}, block_rows={self.block_rows}, device={self.device})"


def _room_for(like: torch.Tensor, shape, n: int, block_rows: int = 1) -> FP8Tensor:
    """n rows of 8 bits that are still to be written"""
    sizes = _row_sizes(shape[-1])
    return FP8Tensor._of(like.new_empty((n, sizes[0]), dtype=torch.uint8),
                         like.new_empty((-(-n // block_rows), sizes[1]), dtype=torch.uint8), shape, block_rows)


def fp8_quantize(x: torch.Tensor, block_rows: int = 1) -> FP8Tensor:
    """``x`` (bfloat16, float16 or float32, on the GPU) in 8 bits: 128 values of a row, or
    with ``block_rows=128`` 128 rows (all dimensions but the last counted through) of 128
    columns, share the smallest power of two with which none is above 448; values are
    rounded to the nearest e4m3 number, ties to the even code.  A block that holds a NaN
    or an infinity reads as NaN.  Autograd does not record it."""
    if block_rows not in (1, 128):
        raise ValueError("block_rows must be 1 or 128")
    code = _dtype_code(x.dtype)
    index = _on_gpu(x=x)
    shape = x.shape
    if not shape:
        raise ValueError("x must have one dimension at least")
    cols = shape[-1]
    rows, n, stride = _as_rows(x, cols)
    out = _room_for(x, shape, n, block_rows)
    _call(_lib.load().nz_fp8_quantize, index, rows.data_ptr(), code, n, cols, stride, block_rows, out.data.data_ptr(),
          out.scales.data_ptr())
    return out


def _product(x, weight: FP8Tensor, bias, dtype: torch.dtype) -> torch.Tensor:
    L = _lib.load()
    n, k = weight.shape
    code, wd = _dtype_code(dtype), weight.data
    held = isinstance(x, FP8Tensor)
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
        _call(L.nz_fp8_linear_rows8, index, xt.data_ptr(), x.scales.data_ptr(), m, k, wd.data_ptr(),
              weight.scales.data_ptr(), n, weight.block_rows, b, y.data_ptr(), code, at, room)
    else:
        _call(L.nz_fp8_linear, index, xt.data_ptr(), code, m, k, stride, wd.data_ptr(), weight.scales.data_ptr(), n,
              weight.block_rows, b, y.data_ptr(), at, room)
    return y


def _input_gradient(grad: torch.Tensor, weight: FP8Tensor) -> torch.Tensor:
    L = _lib.load()
    n, k = weight.shape
    index = _on_gpu(weight=weight.data, grad=grad)
    dx = grad.new_empty((*grad.shape[:-1], k))
    if n == 0:  # empty sums
        return dx.zero_()
    rows, m, stride = _as_rows(grad, n)
    args = (rows.data_ptr(), _dtype_code(grad.dtype), m, n, stride)
    room = _ask(L.nz_fp8_linear_grad_workspace_bytes, index, *args, k, weight.block_rows)
    ws, at = _workspace(room, rows)
    _call(L.nz_fp8_linear_grad, index, *args, weight.data.data_ptr(), weight.scales.data_ptr(), k, weight.block_rows,
          dx.data_ptr(), at, room)
    return dx


def _saved(ctx, held: FP8Tensor) -> None:
    """Save what ``held`` consists of.  An inference tensor has no version to check."""
    if not held.data.is_inference():
        ctx.save_for_backward(held.data, held.scales)


def _unsaved(ctx, held: FP8Tensor) -> FP8Tensor:
    """The same again; raises if it has been written to since.  Hooks of saved tensors may hand back others."""
    parts = ctx.saved_tensors
    if parts and (parts[0] is not held.data or parts[1] is not held.scales):
        return FP8Tensor(*parts, held.shape, held.block_rows)
    return held


class BlockLinear(torch.autograd.Function):
    """``y = x W^T (+ b)`` with a frozen weight in 8 bits.  Backward gives the
    gradients of ``x`` (the rounding of its rows to 8 bits is passed straight
    through) and of the bias."""

    @staticmethod
    def forward(ctx, x, weight, bias, dtype):
        ctx.weight = weight
        if ctx.needs_input_grad[0]:
            _saved(ctx, weight)
        return _product(x, weight, bias, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        grad_x = grad_b = None
        if ctx.needs_input_grad[0]:
            grad_x = _input_gradient(grad_output, _unsaved(ctx, ctx.weight))
        if ctx.needs_input_grad[2]:
            grad_b = _bias_gradient(grad_output, ctx.weight.shape[0])
        return grad_x, None, grad_b, None


def fp8_linear(x, weight: FP8Tensor, bias=None, dtype=None) -> torch.Tensor:
    """``x @ W^T (+ bias)`` for a weight ``[out, in]`` in 8 bits.

    ``x`` is a tensor ``[..., in]`` (bfloat16, float16 or float32), whose rows are
    brought to 8 bits on the way and whose type the result has; or an
    :class:`FP8Tensor` with a scale for each row (rows that several weights share),
    with a result of type ``dtype`` (bfloat16).  ``bias`` has the type of the result.
    Autograd records the gradients of ``x`` and ``bias``; the weight is frozen.

    A bfloat16 or float16 result may lack, of each product, what lies below 2^-12 of the
    largest of the eight consecutive products that it is added with: usually far
    below its own rounding, but not where large products cancel.  A float32 result is
    summed in 32 bits throughout; rows of any type have one by
    ``fp8_linear(fp8_quantize(x), weight, dtype=torch.float32)``."""
    if not isinstance(weight, FP8Tensor) or len(weight.shape) != 2:
        raise ValueError("weight must be a matrix in 8 bits (fp8_quantize)")
    n, k = weight.shape
    if isinstance(x, FP8Tensor):
        if x.block_rows != 1:
            raise ValueError("activation rows have a scale each (fp8_quantize(x))")
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
    if torch.is_grad_enabled() and (not isinstance(x, FP8Tensor) and x.requires_grad
                                    or bias is not None and bias.requires_grad):
        return BlockLinear.apply(x, weight, bias, dtype)
    return _product(x, weight, bias, dtype)


def fp8_weight_gradient(grad: torch.Tensor, x: FP8Tensor, out=None) -> torch.Tensor:
    """``grad^T @ x``, the gradient ``[out, in]`` of a dense weight, for the gradient
    ``grad`` (``[..., out]``) of the layer's result and its input ``x`` (``[..., in]``)
    kept in 8 bits, in the type of ``grad``.

    Sums are made in 32 bits, in an order that the sizes alone decide, and rounded
    once.  With ``out`` the gradient is added to that tensor (contiguous, of the type of
    ``grad``) before the rounding; autograd takes that for a change in place, but records
    neither it nor the gradient itself."""
    if not isinstance(x, FP8Tensor):
        raise ValueError("x must be held in 8 bits (fp8_quantize)")
    if grad.dim() < 1 or grad.shape[:-1] != x.shape[:-1]:
        raise ValueError("grad must have the dimensions of x, the last one aside")
    n, k = grad.shape[-1], x.shape[-1]
    code = _dtype_code(grad.dtype)
    index = _on_gpu(grad=grad, x=x.data, out=out)
    flags = 0
    if out is None:
        out = grad.new_empty((n, k))
    else:
        if tuple(out.shape) != (n, k) or out.dtype != grad.dtype or not out.is_contiguous() or out.is_neg():
            raise ValueError(f"out must be a contiguous {grad.dtype} tensor of shape {(n, k)}")
        flags = _lib.GRAD_ACCUMULATE
    rows, m, stride = _as_rows(grad, n)
    if m == 0:  # empty sums
        return out if flags else out.zero_()
    L = _lib.load()
    args = (rows.data_ptr(), code, m, n, stride)
    room = _ask(L.nz_fp8_weight_grad_workspace_bytes, index, *args, k)
    ws, at = _workspace(room, rows)
    _call(L.nz_fp8_weight_grad, index, *args, x.data.data_ptr(), x.scales.data_ptr(), k, x.block_rows, flags,
          out.data_ptr(), at, room)
    if flags:
        increment_version(out)
    return out


@lru_cache(maxsize=1024)
def _kept_places(rows: int, cols: int, tensors: int):
    """Where a buffer holds the codes and scales of ``tensors`` (1 or 2) tensors, and its size"""
    data, scales = (rows * size for size in _row_sizes(cols))
    first = data * tensors
    second = first + -(-scales // 16) * 16
    if tensors == 1:
        return 0, first, None, None, first + scales
    return 0, first, data, second, second + scales


def _kept_parts(at: int, places):
    """the addresses of these in a buffer at ``at``: x's codes and scales, up's"""
    x, x_scales, up, up_scales, _ = places
    return at + x, at + x_scales, None if up is None else at + up, None if up is None else at + up_scales


def _activate(x, kind: int, up, keep: bool):
    """the result, and what is kept of ``x`` and ``up``"""
    code, cols = _dtype_code(x.dtype), x.shape[-1]
    index = _on_gpu(x=x, up=up)
    y = x.new_empty(x.shape)
    rows, n, stride = _as_rows(x, cols)
    u_at, u_stride = None, 0
    if up is not None:
        u, _, u_stride = _as_rows(up, cols)
        u_at = u.data_ptr()
    kept, parts = None, (None, None, None, None)
    if keep:
        places = _kept_places(n, cols, 1 if up is None else 2)
        kept = x.new_empty(places[4], dtype=torch.uint8)
        parts = _kept_parts(kept.data_ptr(), places)
    _call(_lib.load().nz_fp8_activation, index, kind, rows.data_ptr(), code, n, cols, stride, u_at, u_stride,
          y.data_ptr(), *parts)
    return y, kept


class HeldActivation(torch.autograd.Function):
    """``f(x)``, or ``f(x) * up``, that keeps ``x`` and ``up`` in 8 bits (in one buffer)."""

    @staticmethod
    def forward(ctx, x, kind, up):
        y, kept = _activate(x, kind, up, True)
        ctx.kind, ctx.tensors = kind, 1 if up is None else 2
        ctx.save_for_backward(kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        (kept,) = ctx.saved_tensors
        index = _on_gpu(grad=grad_output, x=kept)
        cols = grad_output.shape[-1]
        rows, n, stride = _as_rows(grad_output, cols)
        dx = grad_output.new_empty(grad_output.shape)
        dup = dup_at = None
        if ctx.tensors == 2:
            dup = grad_output.new_empty(grad_output.shape)
            dup_at = dup.data_ptr()
        _call(_lib.load().nz_fp8_activation_grad, index, ctx.kind, rows.data_ptr(), _dtype_code(grad_output.dtype), n,
              cols, stride, *_kept_parts(kept.data_ptr(), _kept_places(n, cols, ctx.tensors)), dx.data_ptr(), dup_at)
        return dx, None, dup


def fp8_activation(x: torch.Tensor, kind: str = "gelu", up=None) -> torch.Tensor:
    """``f(x)``, times ``up`` where that is given: ``"gelu"`` (``x`` times the normal
    distribution's integral), ``"gelu_tanh"`` (its approximation with a hyperbolic
    tangent) or ``"silu"``, computed in 32 bits and rounded once.

    For the backward pass ``x`` and ``up`` are kept in 8 bits (blocks of 128 values of a
    row): the gradients are those of the formula at these values."""
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {', '.join(_KINDS)}")
    if x.dim() < 1:
        raise ValueError("x must have one dimension at least")
    _dtype_code(x.dtype)
    if up is not None and (up.shape != x.shape or up.dtype != x.dtype):
        raise ValueError(f"up must be a {x.dtype} tensor of shape {tuple(x.shape)}")
    if torch.is_grad_enabled() and (x.requires_grad or up is not None and up.requires_grad):
        return HeldActivation.apply(x, _KINDS[kind], up)
    return _activate(x, _KINDS[kind], up, False)[0]
