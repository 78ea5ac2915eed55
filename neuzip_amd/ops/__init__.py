from neuzip_amd.ops.linear import CompressedLinear
from neuzip_amd.ops.microscaled import MXTensor, mx_embedding, mx_linear, mx_quantize
from neuzip_amd.ops.embedding import CompressedEmbedding, embedding_gradient

__all__ = ["CompressedLinear", "CompressedEmbedding", "MXTensor", "mx_quantize", "mx_linear", "mx_embedding",
           "embedding_gradient"]
