"""Residual norm layer on the package's kernels: the joint between two blocks in one pass each way."""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import ops

_PARAMS = ("weight", "bias", "post_weight", "post_bias", "gate")


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, bias, post_weight, post_bias, gate, options):
        params = dict(zip(_PARAMS, (weight, bias, post_weight, post_bias, gate)))
        n, h, stats = ops.residual_norm(x, y, **params, **options)
        ctx.set_materialize_grads(False)
        ctx.options = {k: options[k] for k in ("post", "residual_scale", "kind")}
        ctx.n_dtype = n.dtype
        ctx.save_for_backward(h, stats, y, *params.values())
        return n, h

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_n, grad_h):
        h, stats, y, *params = ctx.saved_tensors
        if grad_n is None and grad_h is None:
            return (None,) * 8
        if grad_n is None and y is None:  # the norm's type is known from its gradient alone
            grad_n = torch.zeros(h.shape, dtype=ctx.n_dtype, device=h.device)
        params = dict(zip(_PARAMS, params))
        wanted = [k for k, need in zip(_PARAMS, ctx.needs_input_grad[2:7]) if need]
        got = ops.residual_norm_grad(grad_n, grad_h, h, stats, y, **params, **ctx.options, wanted=wanted)
        return got["x"], got.get("y"), *(got.get(k) for k in _PARAMS), None


def residual_norm(x: torch.Tensor, y: torch.Tensor | None = None, *, weight=None, bias=None, post_weight=None,
                  post_bias=None, post: bool | None = None, gate=None, residual_scale: float = 1.0, kind: str = "rms",
                  eps: float = 1e-6, out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(n, h) of ops.residual_norm with gradients for x, y and every parameter given."""
    post = (post_weight is not None or post_bias is not None) if post is None else bool(post)
    options = {"post": post, "residual_scale": float(residual_scale), "kind": kind, "eps": float(eps),
               "out_dtype": out_dtype}
    return _ResidualNorm.apply(x, y, weight, bias, post_weight, post_bias, gate, options)


class ResidualNorm(nn.Module):
    """Norm after the last block, gate, scaled residual sum and norm before the next block, as one layer.

    ``n, h = norm(x, y)``: x is the residual stream, y the output of the block
    that ended (None before the first block: h is x then, and only the norm
    before the block applies), n the input of the block that begins and h the
    new residual stream.  post=True norms y first; gate=True
    gives a learned gate of [d], and a gate can be passed to forward instead
    ([d], or one row for each sample).  bias adds biases to both norms.
    """

    def __init__(self, dim: int, kind: str = "rms", eps: float = 1e-6, bias: bool = False, post: bool = False,
                 gate: bool = False, residual_scale: float = 1.0, device=None, dtype=None):
        super().__init__()
        if kind not in ("rms", "layer"):
            raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
        like = {"device": device, "dtype": dtype}
        self.dim, self.kind, self.eps, self.residual_scale = int(dim), kind, float(eps), float(residual_scale)
        self.weight = nn.Parameter(torch.ones(dim, **like))
        self.bias = nn.Parameter(torch.zeros(dim, **like)) if bias else None
        self.post = bool(post)
        self.post_weight = nn.Parameter(torch.ones(dim, **like)) if post else None
        self.post_bias = nn.Parameter(torch.zeros(dim, **like)) if post and bias else None
        self.gate = nn.Parameter(torch.ones(dim, **like)) if gate else None

    def forward(self, x: torch.Tensor, y: torch.Tensor | None = None,
                gate: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        if y is None:  # nothing to norm or gate yet
            if gate is not None:
                raise ValueError("a gate needs y")
            return residual_norm(x, weight=self.weight, bias=self.bias, kind=self.kind, eps=self.eps)
        if gate is not None and self.gate is not None:
            raise ValueError("the layer has a gate of its own")
        return residual_norm(x, y, weight=self.weight, bias=self.bias, post_weight=self.post_weight,
                             post_bias=self.post_bias, post=self.post, gate=self.gate if gate is None else gate,
                             residual_scale=self.residual_scale, kind=self.kind, eps=self.eps)

    def extra_repr(self) -> str:
        return (f"{self.dim}, kind={self.kind!r}, eps={self.eps}, post={self.post}, gate={self.gate is not None}, "
                f"residual_scale={self.residual_scale}")
