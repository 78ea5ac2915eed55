"""``MXLinear`` and ``MXEmbedding``: layers whose weights are held in microscaled
4 bits (``neuzip_amd.ops.mx_quantize``) and stay as they are: no gradient
reaches them, the gradients of a Linear's input and bias do.

The stored tensors are buffers, so they travel with ``state_dict`` and ``.to``.
Whatever writes to them between a forward pass and its backward makes that an
error; ``DistributedDataParallel`` does so at every forward, unless it is told
``broadcast_buffers=False``.
"""
from __future__ import annotations

import torch

from neuzip_amd.ops.microscaled import MXTensor, mx_embedding, mx_linear, mx_quantize


class _Microscaled(torch.nn.Module):
    def _hold(self, dense: torch.Tensor) -> None:
        # like a manager's write: what is not on the GPU yet is taken there
        q = mx_quantize(dense.detach() if dense.is_cuda else dense.detach().cuda(), 4)
        self.register_buffer("weight_data", q.data)
        self.register_buffer("weight_scales", q.scales)
        self._shape = q.shape

    @property
    def weight(self) -> MXTensor:
        return MXTensor(self.weight_data, self.weight_scales, self._shape, 4)

    def nbytes_compressed(self) -> int:
        """Bytes held for the weight."""
        return self.weight_data.numel() + self.weight_scales.numel()


def _autocast(x):
    """``x`` in the type that an autocast region asks for"""
    if not isinstance(x, MXTensor) and torch.is_autocast_enabled("cuda"):
        return x.to(torch.get_autocast_dtype("cuda"))
    return x


class MXLinear(_Microscaled):
    def __init__(self, linear: torch.nn.Linear) -> None:
        super().__init__()
        self.in_features = linear.in_features
        self.out_features = linear.out_features
        if linear.bias is None:
            self.register_parameter("bias", None)
        else:
            self.bias = torch.nn.Parameter(linear.bias.data, requires_grad=linear.bias.requires_grad)
        self._hold(linear.weight.data)

    def forward(self, x):
        x = _autocast(x)
        bias = self.bias
        if bias is not None:
            dtype = torch.bfloat16 if isinstance(x, MXTensor) else x.dtype
            bias = bias.to(dtype)
        return mx_linear(x, self.weight, bias)

    def extra_repr(self) -> str:
        # the leading "!" marks a converted layer in the printed module tree
        return f"! in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


class MXEmbedding(_Microscaled):
    """A frozen table.  Rows are multiplied by ``scale`` and have the type of the
    dense table.  ``linear(x)`` multiplies rows with the same table (an output
    projection that is tied to it)."""

    def __init__(self, embedding: torch.nn.Embedding, scale: float = 1.0) -> None:
        super().__init__()
        if embedding.max_norm is not None:
            raise ValueError("max_norm changes the table at every lookup: a table in 4 bits stays as it is")
        self.num_embeddings = embedding.num_embeddings
        self.embedding_dim = embedding.embedding_dim
        self.padding_idx = embedding.padding_idx
        self.scale = float(scale)
        # the type of the rows, which the module's own .to and .half change
        self.register_buffer("_like", embedding.weight.data.new_empty(0), persistent=False)
        self._hold(embedding.weight.data)
        self.register_buffer("_status", torch.zeros(1, dtype=torch.int32, device=self.weight_data.device),
                             persistent=False)

    def forward(self, x):
        return mx_embedding(x, self.weight, self.scale, self._like.dtype, self._status)

    def linear(self, x):
        return mx_linear(_autocast(x), self.weight)

    def check(self) -> None:
        """Raise if a lookup since the last check had an index outside the table (waits for the device)."""
        bad = int(self._status.item())
        self._status.zero_()
        if bad:
            raise RuntimeError("a lookup had an index outside the table")

    def extra_repr(self) -> str:
        return f"! num_embeddings={self.num_embeddings}, embedding_dim={self.embedding_dim}, scale={self.scale}"
