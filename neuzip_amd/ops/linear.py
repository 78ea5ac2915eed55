"""Autograd node of a Linear layer whose weight is stored compressed.

Behaviour follows the reference's ``CompressedLinear`` (neuzip/ops/linear.py:11-46):

* forward: honour an active autocast region by casting the activation by hand,
  then ``y = x @ W^T (+ b)`` with ``W`` decompressed just in time and dropped;
* backward: decompress ``W`` a second time for ``dL/dx``, accumulate ``dL/dW``
  on the parameter's ``_gradient`` slot (not in ``.grad``), and hand autograd a
  zero-size tensor for the placeholder so that post-accumulate-grad hooks of
  the compressed parameter still fire.

:class:`CompressedLinearHeld8` does the same, but keeps the activation in 8 bits
(``fp8_quantize``) for ``dL/dW``, which is then that of the kept values.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from neuzip_amd.ops.blocks8 import FP8Tensor, fp8_quantize, fp8_weight_gradient
from neuzip_amd.ops.microscaled import _DTYPES, _bias_gradient


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """Collapse all leading dimensions: [..., k] -> [m, k]."""
    return t.reshape(-1, t.shape[-1])


def _column_sums(rows: torch.Tensor) -> torch.Tensor:
    """The gradient of a bias.  A library's sum over many rows clears its counters with a node
    that the replays of a captured graph do not keep to, so there it is the kernel of the
    microscaled layers (like the library's in 32 bits and rounded once, in another order)."""
    if (rows.is_cuda and torch.cuda.is_current_stream_capturing() and rows.dtype in _DTYPES
            and not (torch.is_grad_enabled() and rows.requires_grad)):
        return _bias_gradient(rows, rows.shape[1])
    return rows.sum(0)


class CompressedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs, _p, bias):
        ctx._inputs_dtype = inputs.dtype
        x = inputs
        if torch.is_autocast_enabled():
            x = x.to(torch.get_autocast_gpu_dtype())
        ctx.save_for_backward(x, bias)
        ctx.carry = (_p,)
        return _p.linear(x, bias)

    @staticmethod
    def backward(ctx, grad_output):
        x, bias = ctx.saved_tensors
        (_p,) = ctx.carry

        x2d = _as_rows(x)
        go2d = _as_rows(grad_output)
        dense_w = _p.shared()

        grad_x = torch.mm(go2d, dense_w).reshape(x.shape).to(ctx._inputs_dtype)
        del dense_w
        grad_w = torch.mm(go2d.t(), x2d)

        if _p._gradient is None:
            _p._gradient = grad_w
        else:
            _p._gradient.add_(grad_w)

        grad_b = _column_sums(go2d) if bias is not None else None
        return grad_x, torch.empty_like(_p.data), grad_b


class CompressedLinearHeld8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, inputs, _p, bias):
        ctx._inputs_dtype = inputs.dtype
        x = inputs
        if torch.is_autocast_enabled():
            x = x.to(torch.get_autocast_gpu_dtype())
        held = fp8_quantize(x)
        ctx.carry = (_p, held.shape, bias is not None)
        ctx.save_for_backward(held.data, held.scales)  # and held by nothing else: hooks may take them elsewhere
        return _p.linear(x, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        data, scales = ctx.saved_tensors
        _p, shape, has_bias = ctx.carry
        go2d = _as_rows(grad_output)
        dense_w = _p.shared()

        grad_x = torch.mm(go2d, dense_w).reshape(shape).to(ctx._inputs_dtype)
        del dense_w
        held = FP8Tensor(data, scales, (go2d.shape[0], shape[-1]), 1)
        into = _p._gradient
        if into is None:
            _p._gradient = fp8_weight_gradient(go2d, held)
        elif into.dtype == go2d.dtype and into.is_contiguous():
            fp8_weight_gradient(go2d, held, out=into)
        else:
            into.add_(fp8_weight_gradient(go2d, held))

        grad_b = _column_sums(go2d) if has_bias else None
        return grad_x, torch.empty_like(_p.data), grad_b
