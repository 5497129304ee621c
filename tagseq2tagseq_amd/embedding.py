"""Scaled embedding lookup on the gfx950 kernels, its weight gradient summed by
token, as a ``torch.library`` custom op with registered autograd.

The model's first operator (the reference embeds with torch's nn.Embedding,
model/modules/training_module.py:200-209) with a factor on the rows, as models
use whose head shares the table (sqrt(model_dim), so that rows of the head's
size enter the residual stream at unit size):

    out = embedding(tokens, weight, scale)       # scale weight[tokens]

The gradient groups the positions by token and adds the rows of each token in
the order of its positions, in fp32 with one rounding: the same bits on every
run, without a float32 table or atomics on its rows.

Kernels: libt2t_attn.so ``t2t_embedding`` / ``t2t_embedding_backward``.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib


@torch.library.custom_op("t2t::embedding", mutates_args=())
def embedding_op(tokens: torch.Tensor, weight: torch.Tensor, scale: float,
                 padding: int) -> torch.Tensor:
    """scale weight[tokens] ([..., C]); padding: id without a gradient, or -1."""
    return _lib.host().embedding(tokens, weight, scale)


@embedding_op.register_fake
def _embedding_fake(tokens, weight, scale, padding):
    return weight.new_empty((*tokens.shape, weight.shape[1]))


@torch.library.custom_op("t2t::embedding_backward", mutates_args=())
def embedding_backward_op(tokens: torch.Tensor, dy: torch.Tensor, num_embeddings: int,
                          scale: float, padding: int) -> torch.Tensor:
    """The weight's gradient [num_embeddings, C] (dy's dtype)."""
    return _lib.host().embedding_backward(tokens, dy, num_embeddings, scale, padding)


@embedding_backward_op.register_fake
def _embedding_backward_fake(tokens, dy, num_embeddings, scale, padding):
    return dy.new_empty((num_embeddings, dy.shape[-1]))


def _setup(ctx, inputs, output):
    tokens, weight, ctx.scale, ctx.padding = inputs
    ctx.save_for_backward(tokens)
    ctx.num_embeddings = weight.shape[0]


def _backward(ctx, dy):
    (tokens,) = ctx.saved_tensors
    return (None, embedding_backward_op(tokens, dy, ctx.num_embeddings, ctx.scale, ctx.padding),
            None, None)


embedding_op.register_autograd(_backward, setup_context=_setup)


class EmbeddingFn(torch.autograd.Function):
    """The same kernels as t2t::embedding for eager calls that something besides
    autograd watches (the others are recorded by the host module)."""

    @staticmethod
    def forward(ctx, tokens, weight, scale, padding):
        ctx.save_for_backward(tokens)
        ctx.args = weight.shape[0], scale, padding
        return _lib.host().embedding(tokens, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (tokens,) = ctx.saved_tensors
        return None, _lib.host().embedding_backward(tokens, dy, *ctx.args), None, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``: rows [..., C] (weight's dtype, bf16 or
    float32) of tokens [...] (int64 or int32) from weight [V, C], V up to 2^20.

    The weight's gradient is dense; the row ``padding_idx`` (counted from the
    end when negative) gets none.  An id outside [0, V) gives a row of NaN and
    no gradient: the ids stay on the device and are not waited for."""
    scale = float(scale)
    if not abs(scale) <= torch.finfo(torch.float32).max:
        raise ValueError(f"scale={scale!r} must be finite in float32")
    if weight.dim() != 2:
        raise ValueError(f"weight must be [V, C], got shape {tuple(weight.shape)}")
    padding, V = -1, weight.shape[0]
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx={padding_idx} is not a row of {V}")
        padding = int(padding_idx) % V
    if torch.compiler.is_compiling():
        return embedding_op(tokens, weight, scale, padding)
    if _lib.unwatched(tokens, weight):
        return _lib.host().embedding(tokens, weight, scale)
    if _lib.only_recorded(tokens, weight):
        return _lib.host().embedding_ad(tokens, weight, scale, padding)
    return EmbeddingFn.apply(tokens, weight, scale, padding)


class ScaledEmbedding(nn.Embedding):
    """nn.Embedding (same parameters and state dict) with a factor on its rows,
    on ``embedding``; a CPU table uses torch's lookup.  The table starts as
    nn.Embedding's, N(0, 1): for rows of unit size behind the factor, and logits of
    that size from a head that shares the table, multiply it by 1 / scale first."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0,
                 padding_idx: Optional[int] = None, device=None, dtype=None):
        super().__init__(num_embeddings, embedding_dim, padding_idx=padding_idx, device=device,
                         dtype=dtype)
        self.scale = float(scale)

    @classmethod
    def from_pretrained(cls, embeddings: torch.Tensor, freeze: bool = True,
                        padding_idx: Optional[int] = None,
                        scale: float = 1.0) -> "ScaledEmbedding":
        """A module of the table ``embeddings`` [V, C] itself."""
        if embeddings.dim() != 2:
            raise ValueError(f"embeddings must be [V, C], got shape {tuple(embeddings.shape)}")
        m = cls(*embeddings.shape, scale, padding_idx, device="meta", dtype=embeddings.dtype)
        m.weight = nn.Parameter(embeddings, requires_grad=not freeze)
        return m

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        if not self.weight.is_cuda:
            return super().forward(tokens) * self.scale
        return embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, scale={self.scale}"
