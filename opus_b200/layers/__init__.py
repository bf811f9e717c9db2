"""Capture layers (drop-in for OPUS.layers, OPUS/layers/__init__.py:8-11), and the layers between them.

ScaledEmbedding and ResidualNorm have no counterpart there: they are the
kernels' form of a model's embedding and of the joints between its blocks.
"""
from .embedding import ScaledEmbedding, scaled_embedding
from .linear import GCLinear
from .lora_layers import GCLoRALinear, LoRALinear
from .norm import ResidualNorm, residual_norm

__all__ = ["GCLinear", "GCLoRALinear", "LoRALinear", "ResidualNorm", "ScaledEmbedding", "residual_norm",
           "scaled_embedding"]
