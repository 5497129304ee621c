"""Distillation from a teacher's top logits on the gfx950 ``t2t_distill_rows``
kernel: the loss of each row of student logits and its gradient in one pass,
for given logits and fused with a linear head.

A teacher's whole distribution over the vocabulary is too much to store or
send for every token; its K largest logits and their ids (``teacher_logits``,
``teacher_idx``) are what a distillation set keeps.  For a row of student logits z
with temperature T and weight alpha:

    p    = softmax over the K slots of teacher_logits / T
    q    = softmax(z / T)
    KD   = sum_k p_k (ln p_k - ln q[teacher_idx_k])
    loss = alpha T^2 KD + (1 - alpha) cross_entropy(z, target)

averaged over the rows whose target is not ignore_index (all rows without
targets).  Slots with a negative id are empty: a row may have fewer than K, or
none, and then only its second part.  Slots of the same id add up.  An id
outside the vocabulary makes the loss NaN, as a target outside it does: ids
stay on the device and are not waited for.  With alpha 0 the teacher is not read.

    loss = distill_loss(logits, teacher_idx, teacher_logits, targets,
                        temperature=2.0, alpha=0.5)
    loss = head_distill(x, weight, teacher_idx, teacher_logits, targets, ...)

The second takes the rows before the head, as ``head_loss`` does: per chunk of rows the
logits (a bf16 product), their gradient over them in place, and the products
for dx and dW.  It stands beside the reference's fused linear cross-entropy
(model/modules/training_module.py:127-133, 209).
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
import torch.utils.checkpoint
from torch.autograd.function import once_differentiable

from . import _lib
from .head_loss import AUTO_CHUNK_BYTES, _mm_f32, fused_head_applies, head_weight, scaled_rows
from .modules import LinearCELoss

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


@torch.library.custom_op("t2t::distill_loss", mutates_args=())
def distill_loss_op(logits: torch.Tensor, teacher_idx: torch.Tensor, teacher_logits: torch.Tensor,
                    targets: Optional[torch.Tensor], temperature: float, alpha: float,
                    ignore_index: int, reduction: int) -> torch.Tensor:
    """The loss (float32; reduction 0 none, 1 sum, 2 mean)."""
    return _lib.host().distill_loss(logits, teacher_idx, teacher_logits, targets, temperature,
                                    alpha, ignore_index, reduction, False)[0]


@distill_loss_op.register_fake
def _distill_loss_fake(logits, teacher_idx, teacher_logits, targets, temperature, alpha,
                       ignore_index, reduction):
    return logits.new_empty(() if reduction else logits.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("t2t::distill_loss_backward", mutates_args=())
def distill_loss_backward_op(g: torch.Tensor, logits: torch.Tensor, teacher_idx: torch.Tensor,
                             teacher_logits: torch.Tensor, targets: Optional[torch.Tensor],
                             temperature: float, alpha: float, ignore_index: int,
                             reduction: int) -> torch.Tensor:
    """The logits' gradient."""
    return _lib.host().distill_loss_backward(g, logits, teacher_idx, teacher_logits, targets,
                                             temperature, alpha, ignore_index, reduction, None,
                                             None)


@distill_loss_backward_op.register_fake
def _distill_loss_backward_fake(g, logits, teacher_idx, teacher_logits, targets, temperature,
                                alpha, ignore_index, reduction):
    return logits.new_empty(logits.shape)


def _setup(ctx, inputs, output):
    ctx.has_targets = inputs[3] is not None
    ctx.save_for_backward(*(t for t in inputs[:4] if t is not None))
    ctx.args = inputs[4:]


def _backward(ctx, g):
    saved = ctx.saved_tensors if ctx.has_targets else (*ctx.saved_tensors, None)
    return (distill_loss_backward_op(g, *saved, *ctx.args), *[None] * 7)


distill_loss_op.register_autograd(_backward, setup_context=_setup)


class DistillFn(torch.autograd.Function):
    """The same kernels for eager calls that something besides autograd watches
    (the others are recorded by the host module, in the same way).  A sum or mean is differentiated
    with an incoming gradient of 1 as a rule, so its gradient is written by the
    forward's pass over the logits; the backward hands it over, having the rows
    computed again (on the device, without waiting) where the incoming gradient is
    another.  Where hooks take what the graph saves (a recomputed region, offloading),
    nothing is kept and the gradient is the backward's."""

    @staticmethod
    def forward(ctx, logits, teacher_idx, teacher_logits, targets, *args):
        keep = (args[-1] != 0 and ctx.needs_input_grad[0]
                and not _lib.host().saved_tensors_hooked())
        loss, grad, inv = _lib.host().distill_loss(logits, teacher_idx, teacher_logits, targets,
                                                   *args, keep)
        ctx.save_for_backward(logits, teacher_idx, teacher_logits, targets, inv)
        ctx.args, ctx.grad = args, grad
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, teacher_idx, teacher_logits, targets, inv = ctx.saved_tensors
        kept, ctx.grad = ctx.grad, None  # handed over: a second backward computes its own
        d = _lib.host().distill_loss_backward(g, logits, teacher_idx, teacher_logits, targets,
                                              *ctx.args, inv, kept)
        return (d, *[None] * 7)


def distill_loss(logits: torch.Tensor, teacher_idx: torch.Tensor, teacher_logits: torch.Tensor,
                 targets: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
                 alpha: float = 1.0, ignore_index: int = -100,
                 reduction: str = "mean") -> torch.Tensor:
    """The distillation loss of logits [..., V] (bf16 or float32) from the
    teacher's top logits: teacher_idx [..., K] (int64 or int32, K at most 1024;
    negative: an empty slot) and teacher_logits [..., K] (bf16 or float32), mixed
    with the cross-entropy of targets [...] by ``alpha`` (1: the teacher alone;
    targets then only say which rows count).  ``temperature``: 0.01 to 100 (the
    loss is a difference of fp32 logarithms times its square).

    ``reduction``: "mean" over the counted rows (NaN when there are none, as
    torch's mean cross-entropy), "sum", or "none" (a loss a row, 0 in rows that
    do not count).  float32.  The gradient is that of the logits; the
    teacher has none."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction={reduction!r} is none of {sorted(_REDUCTIONS)}")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("the teacher gets no gradient: detach teacher_logits")
    args = float(temperature), float(alpha), int(ignore_index), _REDUCTIONS[reduction]
    if torch.compiler.is_compiling():
        return distill_loss_op(logits, teacher_idx, teacher_logits, targets, *args)
    watched = (logits, teacher_idx, teacher_logits) + (() if targets is None else (targets,))
    if _lib.unwatched(*watched):
        return _lib.host().distill_loss(logits, teacher_idx, teacher_logits, targets, *args,
                                        False)[0]
    if _lib.only_recorded(*watched):
        return _lib.host().distill_loss_ad(logits, teacher_idx, teacher_logits, targets, *args)
    return DistillFn.apply(logits, teacher_idx, teacher_logits, targets, *args)


# ---- with the linear head

def _head_pass(x, weight, teacher_idx, teacher_logits, targets, temperature, alpha, ignore_index,
               chunk, grads):
    """Per chunk of rows: logits, t2t_distill_rows over them in place, then --
    when ``grads`` -- dx and the fp32 dW.  Returns (loss, dx, dw)."""
    N, D = x.shape
    V = weight.shape[0]
    dev = x.device
    if weight.shape[1] != D:
        raise ValueError(f"weight {tuple(weight.shape)} does not match rows of width {D}")
    if teacher_idx.shape != teacher_logits.shape or teacher_idx.shape[:-1].numel() != N:
        raise ValueError(f"teacher_idx {tuple(teacher_idx.shape)} and teacher_logits "
                         f"{tuple(teacher_logits.shape)} are not [{N}, K]")
    K = teacher_idx.shape[-1]
    teacher_idx, teacher_logits = teacher_idx.reshape(N, K), teacher_logits.reshape(N, K)
    inv, scale = None, 1.0 / N if N else float("nan")
    if targets is not None:
        if targets.numel() != N:
            raise ValueError(f"{targets.numel()} targets for {N} rows")
        targets = targets.reshape(-1).to(device=dev, dtype=torch.int64).contiguous()
        inv, scale = _lib.host().distill_count(targets, ignore_index), 1.0
    w = head_weight(weight, dev)
    ld = w.shape[0]
    row_loss = torch.empty((N,), dtype=torch.float32, device=dev)
    dx = torch.empty((N, D), dtype=x.dtype, device=dev) if grads else None
    dw = None
    if chunk is None:
        chunk = max(1, AUTO_CHUNK_BYTES // (2 * ld))
    rows = max(1, min(chunk, N))
    buf = torch.empty((rows, ld), dtype=torch.bfloat16, device=dev)
    for r0 in range(0, N, rows):
        xs = x[r0:r0 + rows]
        m = xs.shape[0]
        logits = buf[:m]
        torch.mm(xs, w.t(), out=logits)
        _lib.host().distill_rows_(logits[:, :V], teacher_idx[r0:r0 + m],
                                  teacher_logits[r0:r0 + m],
                                  None if targets is None else targets[r0:r0 + m], temperature,
                                  alpha, ignore_index, inv, scale, row_loss[r0:r0 + m], grads)
        if grads:
            if ld != V:  # products of zero weights: not zeros in a row that is not finite
                logits[:, V:].zero_()
            torch.mm(logits, w, out=dx[r0:r0 + m])
            part = _mm_f32(logits.t(), xs)
            dw = part if dw is None else dw.add_(part)
    if grads and dw is None:  # no rows
        dw = torch.zeros((ld, D), dtype=torch.float32, device=dev)
    return _lib.host().distill_mean(row_loss, inv, scale), dx, dw


class HeadDistillFn(torch.autograd.Function):
    """forward(x [N, D] bf16, weight [V, D], teacher_idx, teacher_logits, targets,
    ...) -> mean loss; gradients for x and weight, computed in the forward."""

    @staticmethod
    def forward(ctx, x, weight, teacher_idx, teacher_logits, targets, *args):
        loss, dx, dw = _head_pass(x, weight, teacher_idx, teacher_logits, targets, *args,
                                  grads=True)
        ctx.save_for_backward(dx, dw)
        ctx.V, ctx.wdtype = weight.shape[0], weight.dtype
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        dx, dw = ctx.saved_tensors
        return (scaled_rows(dx, g), (dw[:ctx.V] * g).to(ctx.wdtype), *[None] * 7)


def head_distill(x: torch.Tensor, weight: torch.Tensor, teacher_idx: torch.Tensor,
                 teacher_logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *,
                 temperature: float = 1.0, alpha: float = 1.0, ignore_index: int = -100,
                 chunk: Optional[int] = None) -> torch.Tensor:
    """Mean distillation loss of the logits x W^T, as ``distill_loss``, for
    bf16 rows x [N, D] on the GPU and a bf16 / float32 head weight [V, D]; the
    gradient products run only when autograd needs them, on ``chunk`` rows
    at a time (None: as many as 2 GiB of bf16 logits hold)."""
    if not fused_head_applies(x, weight):
        raise RuntimeError("head_distill needs bf16 rows and a bf16 / float32 weight on a ROCm "
                           "device")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("the teacher gets no gradient: detach teacher_logits")
    args = float(temperature), float(alpha), int(ignore_index), chunk
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return HeadDistillFn.apply(x, weight, teacher_idx, teacher_logits, targets, *args)
    with torch.no_grad():
        return _head_pass(x, weight, teacher_idx, teacher_logits, targets, *args, grads=False)[0]


class LinearDistillLoss(LinearCELoss):
    """LinearCELoss (the same parameters) that distils where it is given the
    teacher's top logits: ``forward(x, targets, teacher_idx, teacher_logits)``.
    bf16 rows run ``head_distill``; float32 rows on the GPU are evaluated in
    chunks with recomputation.  Without a teacher it is the cross-entropy."""

    distils = True

    def __init__(self, D: int, V: int, temperature: float = 1.0, alpha: float = 0.5, **kwargs):
        super().__init__(D, V, **kwargs)
        self.temperature = float(temperature)
        self.alpha = float(alpha)

    def forward(self, x: torch.Tensor, targets: torch.Tensor,
                teacher_idx: Optional[torch.Tensor] = None,
                teacher_logits: Optional[torch.Tensor] = None) -> torch.Tensor:
        if (teacher_idx is None) != (teacher_logits is None):
            raise ValueError("teacher_idx and teacher_logits go together")
        if teacher_idx is None:
            return super().forward(x, targets)
        x = x.reshape(-1, x.shape[-1])
        N, K = x.shape[0], teacher_idx.shape[-1]
        t = targets.reshape(N)
        idx, top = teacher_idx.reshape(N, K), teacher_logits.reshape(N, K)
        if fused_head_applies(x, self.weight) and not torch.compiler.is_compiling():
            return head_distill(x, self.weight, idx, top, t, temperature=self.temperature,
                                alpha=self.alpha, ignore_index=self.ignore_index,
                                chunk=self.gpu_chunk)
        n = (t != self.ignore_index).sum()
        total = x.new_zeros((), dtype=torch.float32)
        for r0 in range(0, x.shape[0], self.chunk):
            rows = slice(r0, r0 + self.chunk)
            total = total + torch.utils.checkpoint.checkpoint(
                self._chunk_distill, x[rows], t[rows], idx[rows], top[rows], use_reentrant=False)
        return total / n

    def _chunk_distill(self, xs, ts, idx, top) -> torch.Tensor:
        logits = F.linear(xs, self.weight.to(xs.dtype)).float()
        return distill_loss(logits, idx, top, ts, temperature=self.temperature, alpha=self.alpha,
                            ignore_index=self.ignore_index, reduction="sum")
