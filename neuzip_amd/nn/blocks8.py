"""``FP8Linear``: a frozen layer whose weight is held in 8 bits with a scale for each
block of 128 (``neuzip_amd.ops.fp8_quantize``); the gradients of its input and bias are
made.  ``FP8Activation``: an activation function that keeps its input in 8 bits for the
backward pass.

The stored tensors are buffers, so they travel with ``state_dict`` and ``.to``.
Whatever writes to them between a forward pass and its backward makes that an
error; ``DistributedDataParallel`` does so at every forward, unless it is told
``broadcast_buffers=False``.
"""
from __future__ import annotations

import torch

from neuzip_amd.nn.microscaled import _autocast
from neuzip_amd.ops.blocks8 import _KINDS, FP8Tensor, fp8_activation, fp8_linear, fp8_quantize


class FP8Linear(torch.nn.Module):
    """``block_rows``: 128 rows of the weight share a scale, or (1) each has its own, for
    0.8 % more bytes."""

    def __init__(self, linear: torch.nn.Linear, block_rows: int = 128) -> None:
        super().__init__()
        self.in_features = linear.in_features
        self.out_features = linear.out_features
        self.block_rows = block_rows
        if linear.bias is None:
            self.register_parameter("bias", None)
        else:
            self.bias = torch.nn.Parameter(linear.bias.data, requires_grad=linear.bias.requires_grad)
        dense = linear.weight.data
        # like a manager's write: what is not on the GPU yet is taken there
        q = fp8_quantize(dense if dense.is_cuda else dense.cuda(), block_rows)
        self.register_buffer("weight_data", q.data)
        self.register_buffer("weight_scales", q.scales)

    @property
    def weight(self) -> FP8Tensor:
        return FP8Tensor(self.weight_data, self.weight_scales, (self.out_features, self.in_features), self.block_rows)

    def nbytes_compressed(self) -> int:
        """Bytes held for the weight."""
        return self.weight_data.numel() + self.weight_scales.numel()

    def forward(self, x):
        held = isinstance(x, FP8Tensor)
        if not held:
            x = _autocast(x)
        bias = self.bias
        if bias is not None:
            bias = bias.to(torch.bfloat16 if held else x.dtype)
        return fp8_linear(x, self.weight, bias)

    def extra_repr(self) -> str:
        # the leading "!" marks a converted layer in the printed module tree
        return (f"! in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"block_rows={self.block_rows}")


class FP8Activation(torch.nn.Module):
    """``fp8_activation(x, kind)``, and with a second input that times it."""

    def __init__(self, kind: str = "gelu") -> None:
        super().__init__()
        if kind not in _KINDS:
            raise ValueError(f"kind must be one of {', '.join(_KINDS)}")
        self.kind = kind

    def forward(self, x, up=None):
        return fp8_activation(x, self.kind, up)

    def extra_repr(self) -> str:
        return f"! kind={self.kind}"
