from neuzip_amd.nn.embedding import Embedding
from neuzip_amd.nn.linear import Linear
from neuzip_amd.nn.microscaled import MXEmbedding, MXLinear
from neuzip_amd.nn.blocks8 import FP8Activation, FP8Linear
from neuzip_amd.nn.module import Parameter

__all__ = ["Parameter", "Linear", "Embedding", "MXLinear", "MXEmbedding", "FP8Linear", "FP8Activation"]
