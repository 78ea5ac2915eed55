"""The gradient of an embedding table, and the autograd node of a lookup in a
table that is stored compressed."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from neuzip_amd import _lib
from neuzip_amd.ops.microscaled import _as_rows, _call, _dtype_code, _on_gpu, _table_room, _workspace


def embedding_gradient(indices: torch.Tensor, grad: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                       padding_idx=None, scale_grad_by_freq: bool = False, out=None) -> torch.Tensor:
    """The dense gradient ``[num_embeddings, dim]`` of a table looked up at
    ``indices`` (any shape) and multiplied by ``scale``, for the gradient ``grad``
    (``[*indices.shape, dim]``) of the rows.

    Tokens are sorted, a row's gradients are added in a fixed order in 32 bits and
    rounded once to the type of ``grad``: the same bits every time.  The row
    ``padding_idx`` and indices outside the table take no part;
    ``scale_grad_by_freq`` divides a row's gradient by the number of its tokens.
    With ``out`` the gradient is added to that tensor (contiguous, of the type of
    ``grad``), which reads and writes the rows of the tokens only; autograd takes that for
    a change in place, but records neither it nor the gradient itself."""
    if indices.dtype not in (torch.int64, torch.int32):
        raise ValueError("indices must be int64 or int32")
    if grad.dim() < 1 or grad.shape[:-1] != indices.shape:
        raise ValueError("grad must have the shape of indices and one dimension more")
    if num_embeddings < 0:
        raise ValueError("num_embeddings must not be negative")
    if padding_idx is not None:
        if not -num_embeddings <= padding_idx < num_embeddings:
            raise ValueError("padding_idx must be within num_embeddings")
        padding_idx %= num_embeddings
    code = _dtype_code(grad.dtype)
    index = _on_gpu(grad=grad, indices=indices, out=out)
    cols = grad.shape[-1]
    flags = _lib.GRAD_BY_FREQUENCY if scale_grad_by_freq else 0
    if out is None:
        out = grad.new_empty((num_embeddings, cols))
    else:
        if (tuple(out.shape) != (num_embeddings, cols) or out.dtype != grad.dtype or not out.is_contiguous()
                or out.is_neg()):
            raise ValueError(f"out must be a contiguous {grad.dtype} tensor of shape {(num_embeddings, cols)}")
        flags |= _lib.GRAD_ACCUMULATE
    L = _lib.load()
    idx = indices if indices.dtype == torch.int64 else indices.to(torch.int64)
    idx = idx.contiguous()
    count = idx.numel()
    g, _, stride = _as_rows(grad, cols)
    room = _table_room(count, cols)
    ws, at = _workspace(room, g)
    _call(L.nz_embedding_gradient, index, idx.data_ptr(), count, g.data_ptr(), code, stride, num_embeddings, cols,
          float(scale), -1 if padding_idx is None else padding_idx, flags, out.data_ptr(), at, room)
    if flags & _lib.GRAD_ACCUMULATE:
        increment_version(out)
    return out


class CompressedEmbedding(torch.autograd.Function):
    """Lookup in a compressed table that is being trained.  Like a compressed
    Linear's, the table's gradient goes to the parameter's ``_gradient`` slot and
    autograd gets a zero-size tensor, so that post-accumulate-grad hooks fire."""

    @staticmethod
    def forward(ctx, indices, _p, module):
        ctx.save_for_backward(indices)
        ctx.carry = (_p, module)
        return module._rows(indices)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        (indices,) = ctx.saved_tensors
        _p, module = ctx.carry
        _p._gradient = embedding_gradient(indices, grad_output, module.num_embeddings, module.scale,
                                          module.padding_idx, module.scale_grad_by_freq, out=_p._gradient)
        return None, torch.empty_like(_p.data), None
