from neuzip_amd.ops.linear import CompressedLinear, CompressedLinearHeld8
from neuzip_amd.ops.microscaled import MXTensor, mx_embedding, mx_linear, mx_quantize
from neuzip_amd.ops.embedding import CompressedEmbedding, embedding_gradient
from neuzip_amd.ops.blocks8 import FP8Tensor, fp8_activation, fp8_linear, fp8_quantize, fp8_weight_gradient

__all__ = ["CompressedLinear", "CompressedLinearHeld8", "CompressedEmbedding", "MXTensor", "mx_quantize", "mx_linear",
           "mx_embedding", "embedding_gradient", "FP8Tensor", "fp8_quantize", "fp8_linear",
           "fp8_weight_gradient", "fp8_activation"]
