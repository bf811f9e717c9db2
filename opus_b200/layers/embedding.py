"""Embedding layer on the package's kernels: scaled lookup, gradient by sorted tokens.

The layer in front of the capture linears.  The reference's models look tokens
up with torch's embedding; here the scale rides along and the weight's gradient
is summed in a fixed order (the same bits from every backward).
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import ops


class _ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        out = ops.embedding(tokens, weight, scale=scale)
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return None, ops.embedding_grad(grad, tokens, ctx.vocab, scale=ctx.scale, padding_idx=ctx.padding_idx), None, None


def scaled_embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: int | None = None) -> torch.Tensor:
    """scale * weight[tokens] with its gradient for weight (none for the rows of padding_idx)."""
    if padding_idx is not None and not -weight.shape[0] <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx must be within the {weight.shape[0]} rows, got {padding_idx}")
    return _ScaledEmbedding.apply(tokens, weight, float(scale), padding_idx)


class ScaledEmbedding(nn.Embedding):
    """nn.Embedding whose rows are multiplied by a fixed scale (sqrt(d), say) on the way out.

    Initialisation, weight and state dict are nn.Embedding's (padding_idx
    included); its max_norm, scale_grad_by_freq and sparse are not offered.
    """

    def __init__(self, num_embeddings: int, embedding_dim: int, padding_idx: int | None = None, scale: float = 1.0,
                 device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device, dtype=dtype)
        self.scale = float(scale)

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True, padding_idx: int | None = None,
                        scale: float = 1.0) -> "ScaledEmbedding":
        """A layer on the rows of embeddings (as they are, not a copy), which do not train while freeze is true."""
        if embeddings.dim() != 2:
            raise ValueError(f"embeddings must be [V, d], got {tuple(embeddings.shape)}")
        layer = cls(*embeddings.shape, padding_idx=padding_idx, scale=scale, device="meta", dtype=embeddings.dtype)
        layer.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return layer

    def forward(self, input: torch.Tensor) -> torch.Tensor:  # noqa: A002 - nn.Embedding's argument name
        return scaled_embedding(input, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, scale={self.scale}"
