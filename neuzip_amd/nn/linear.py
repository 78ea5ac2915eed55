"""``Linear``: drop-in for ``torch.nn.Linear`` with a compressed weight.

Counterpart of neuzip/nn/linear.py:14-35: the weight becomes a
:class:`~neuzip_amd.nn.module.Parameter` (exposed as ``.weight`` and stored
under the attribute ``_p``), the bias stays a dense ``nn.Parameter``.

What a layer keeps of its input for the gradient of its weight is the input
itself, as in the reference, or with ``saved_bits = 8`` its values in 8 bits (1.01
bytes each).  Layers that are called with the very same input share the former,
while each keeps 8 bits of its own.
"""
from __future__ import annotations

import torch

from neuzip_amd.nn.module import Parameter
from neuzip_amd.ops import CompressedLinear, CompressedLinearHeld8


class Linear(torch.nn.Module):
    saved_bits = 16  # or 8: of the input, for the gradient of the weight

    def __init__(self, manager, linear: torch.nn.Linear) -> None:
        super().__init__()
        self.manager = manager
        self.in_features = linear.in_features
        self.out_features = linear.out_features
        if linear.bias is None:
            self.register_parameter("bias", None)
        else:
            self.bias = torch.nn.Parameter(linear.bias.data)
        self._p = Parameter(manager, linear.weight.data)

    @property
    def weight(self) -> Parameter:
        return self._p

    def forward(self, x):
        if not torch.is_grad_enabled():
            # nothing to record for backward: same arithmetic without the autograd node
            if torch.is_autocast_enabled():
                x = x.to(torch.get_autocast_gpu_dtype())
            return self._p.linear(x, self.bias)
        if self.saved_bits == 8:
            return CompressedLinearHeld8.apply(x, self._p, self.bias)
        return CompressedLinear.apply(x, self._p, self.bias)

    def extra_repr(self) -> str:
        # the leading "!" marks a converted layer in the printed module tree
        has_bias = self.bias is not None
        saved = ", saved_bits=8" if self.saved_bits == 8 else ""
        return f"! in_features={self.in_features}, out_features={self.out_features}, bias={has_bias}{saved}"
