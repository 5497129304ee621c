"""Attention-module prologue on the gfx950 kernels: QKV split + rotary
embedding in one pass, as a ``torch.library`` custom op with registered
autograd (the gradient is one pass too).

Replaces the head split and rotary embedding inside the reference's attention
module (tunalab ``FlexSelfAttention``, constructed and called at
model/modules/layer.py:16-21,33; the package is not part of the reference, so
the rotary variant -- half-split pairs turned by the negative angle, base 10000,
position = token index -- and its parity with tunalab are unpinned).

    q, k, v = qkv_rope(qkv, cos, sin, num_heads)       # qkv: [B, T, 3 C]
    cos, sin = rope_tables(head_dim, rows, device)      # float32 [rows, D/2]

Kernels: libt2t_attn.so ``t2t_qkv_rope`` / ``t2t_qkv_rope_backward``.

With RMS norms of every query and key head before the rotation (one weight of
head_dim for the queries, one for the keys; the norm that keeps attention
logits bounded), and with fewer key / value heads than query heads:

    q, k, v = qk_norm_rope(qkv, q_weight, k_weight, cos, sin, num_heads)
    q = qk_norm_rope_append(qkv, q_weight, k_weight, cos, sin, num_heads, pos,
                            k_cache, v_cache)       # new tokens, k / v cached

Kernels: ``t2t_qk_norm_rope``, ``t2t_qk_norm_rope_backward`` and
``t2t_qk_norm_rope_append`` (bf16 and float32).

Other forms of the rotation -- interleaved pairs, the first dimensions of the
head only, a position per token, tables scaled for contexts longer than the
trained ones:

    cos, sin = rotary_tables(rotary_dim, rows, device, scaling="by_parts", factor=4.0,
                             original_len=8192)
    q, k, v = qkv_rotary(qkv, cos, sin, num_heads, pos=positions, interleaved=True)

Kernels: ``t2t_qkv_rotary`` and ``t2t_qkv_rotary_backward`` (bf16 and float32).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from operator import index
from typing import Callable, Dict, Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_TABLES: Dict[Tuple, Tuple[torch.Tensor, torch.Tensor]] = {}


def _tables(key: Tuple, make: Callable[[], Tuple[torch.Tensor, torch.Tensor]]):
    """The tables of ``key``, made once.  What is kept serves every later call, so
    nothing of the mode that the first one runs under may stay in it: made
    outside of inference mode (a backward cannot save inference tensors), and
    kept only if they hold memory of their own (not fake tensors, nor those of a
    function transform)."""
    if key in _TABLES:
        return _TABLES[key]
    with torch.inference_mode(False):
        pair = make()
    if all(type(t) is torch.Tensor
           and (torch.compiler.is_dynamo_compiling()
                or not torch._C._functorch.is_functorch_wrapped_tensor(t)) for t in pair):
        _TABLES[key] = pair
    return pair


def _where(device) -> torch.device:
    """The device of a call: "cuda" is the current one, which may change."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        return torch.device("cuda", torch.cuda.current_device())
    return device


def rope_tables(head_dim: int, rows: int, device, base: float = 10000.0):
    """(cos, sin) float32 [rows, head_dim / 2]: angle[p][i] = p * base^(-i / (D/2)).
    Cached per (head_dim, rows, base, device)."""
    device = _where(device)

    def make():
        half = head_dim // 2
        inv = base ** (-torch.arange(0, half, dtype=torch.float32) / half)
        ang = torch.outer(torch.arange(rows, dtype=torch.float32), inv)
        return ang.cos().to(device), ang.sin().to(device)
    return _tables((head_dim, rows, float(base), str(device)), make)


SCALINGS = ("linear", "base", "by_parts")


def _rotary_angles(rotary_dim: int, rows: int, base: float, scaling: Optional[str], factor: float,
                   original_len: int, fast: float, slow: float) -> torch.Tensor:
    """Angles float64 [rows, rotary_dim / 2]; see rotary_tables."""
    half = rotary_dim // 2
    i = torch.arange(half, dtype=torch.float64)
    if scaling == "base":
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = base ** (-i / half)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "by_parts":
        turns = original_len * inv / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
    return torch.outer(torch.arange(rows, dtype=torch.float64), inv)


def rotary_tables(rotary_dim: int, rows: int, device, base: float = 10000.0,
                  scaling: Optional[str] = None, factor: float = 1.0, original_len: int = 0,
                  fast: float = 32.0, slow: float = 1.0, magnitude: Optional[float] = None,
                  positive: bool = False):
    """(cos, sin) float32 [rows, rotary_dim / 2], the angles p * base^(-2 i /
    rotary_dim) computed in float64 (a far position's angle keeps its fraction
    of a turn).  Cached per arguments.

    ``scaling`` fits a context ``factor`` times the trained one:
      * "linear": every angle divided by factor (position interpolation);
      * "base": base * factor^(rotary_dim / (rotary_dim - 2)), which divides the
        slowest pair's angle by factor and leaves the fastest as it is;
      * "by_parts": pairs that turn more than ``fast`` times over
        ``original_len`` positions are left, those that turn less than ``slow``
        times divided by factor, with a linear ramp over the turns between
        (the interpolation by parts of the YaRN paper).
    ``magnitude`` multiplies both tables; None is 1, or for "by_parts" the same
    paper's 1 + 0.1 ln(factor), which sharpens the softmax as contexts grow.

    ``positive``: for a rotation by the positive angle, (a cos - b sin, b cos +
    a sin) of a pair (a, b), as the RoFormer paper and most published weights
    have it; the kernels' own is the negative one, (a cos + b sin, b cos - a sin),
    so that the sines come negated.  Weights serve the direction that they were
    trained in only."""
    if rotary_dim < 2 or rotary_dim % 2 or rows < 0:
        raise ValueError(f"rotary_dim={rotary_dim} must be even and positive, rows={rows} not "
                         "negative")
    if not (math.isfinite(base) and base > 0):
        raise ValueError(f"base={base!r} must be positive and finite")
    if scaling is None:
        if factor != 1.0:
            raise ValueError(f"factor={factor!r} needs a scaling ({', '.join(SCALINGS)})")
    elif scaling not in SCALINGS:
        raise ValueError(f"scaling={scaling!r} is none of {', '.join(SCALINGS)}")
    if not (math.isfinite(factor) and factor >= 1.0):
        raise ValueError(f"factor={factor!r} must be at least 1 and finite")
    if scaling == "base" and rotary_dim < 4:
        raise ValueError('scaling="base" needs rotary_dim of 4 or more')
    if scaling == "by_parts" and not (original_len > 0 and 0 <= slow < fast
                                      and math.isfinite(fast)):
        raise ValueError(f'scaling="by_parts" needs original_len > 0 and 0 <= slow < fast, got '
                         f"{original_len}, {slow!r}, {fast!r}")
    if magnitude is None:
        magnitude = 1.0 + 0.1 * math.log(factor) if scaling == "by_parts" else 1.0
    if not math.isfinite(magnitude):
        raise ValueError(f"magnitude={magnitude!r} must be finite")
    device = _where(device)
    key = ("rotary", rotary_dim, rows, float(base), scaling, float(factor), original_len,
           float(fast), float(slow), float(magnitude), bool(positive), str(device))

    def make():
        ang = _rotary_angles(rotary_dim, rows, base, scaling, factor, original_len, fast, slow)
        turn = -magnitude if positive else magnitude
        return (ang.cos() * magnitude).float().to(device), (ang.sin() * turn).float().to(device)
    return _tables(key, make)


@dataclass(frozen=True)
class RotaryForm:
    """A module's form of the rotary embedding: the ``fraction`` of the head that
    rotates (its first dimensions), the pairs' layout, and the tables' base,
    scaling, magnitude and direction (rotary_tables; ``positive`` for weights
    trained with the published rotation)."""
    fraction: float = 1.0
    interleaved: bool = False
    base: float = 10000.0
    scaling: Optional[str] = None
    factor: float = 1.0
    original_len: int = 0
    positive: bool = False
    fast: float = 32.0
    slow: float = 1.0
    magnitude: Optional[float] = None

    def dims(self, head_dim: int) -> int:
        """Rotated dimensions of a head of head_dim."""
        R = round(self.fraction * head_dim)
        if not 16 <= R <= head_dim or R % 16:
            raise ValueError(f"fraction={self.fraction!r} of head_dim={head_dim} is {R} rotated "
                             "dimensions (a multiple of 16 up to head_dim)")
        return R

    def tables(self, head_dim: int, rows: int, device):
        return rotary_tables(self.dims(head_dim), rows, device, self.base, self.scaling,
                             self.factor, self.original_len, self.fast, self.slow,
                             self.magnitude, self.positive)


def _split_dims(qkv: torch.Tensor, num_heads: int):
    if qkv.dim() != 3:
        raise ValueError(f"qkv must be [B, T, 3 C], got shape {tuple(qkv.shape)}")
    B, T, C3 = qkv.shape
    if C3 % (3 * num_heads) != 0:
        raise ValueError(f"last dim {C3} is not 3 * num_heads * head_dim (num_heads={num_heads})")
    return B, T, C3 // (3 * num_heads)


def _qkv_rope_impl(qkv, cos, sin, num_heads, pos0):
    return _lib.host().qkv_rope(qkv, cos, sin, num_heads, pos0)


def _qkv_rope_bwd_impl(dq, dk, dv, cos, sin, pos0):
    return _lib.host().qkv_rope_backward(dq, dk, dv, cos, sin, pos0)


@torch.library.custom_op("t2t::qkv_rope", mutates_args=())
def qkv_rope_op(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
                pos0: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(q, k, v) [B, H, T, D] from qkv [B, T, 3 H D]; q and k rotated."""
    return _qkv_rope_impl(qkv, cos, sin, num_heads, pos0)


@qkv_rope_op.register_fake
def _qkv_rope_fake(qkv, cos, sin, num_heads, pos0):
    B, T, D = _split_dims(qkv, num_heads)
    return tuple(qkv.new_empty((B, num_heads, T, D)) for _ in range(3))


@torch.library.custom_op("t2t::qkv_rope_backward", mutates_args=())
def qkv_rope_backward_op(dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, cos: torch.Tensor,
                         sin: torch.Tensor, pos0: int) -> torch.Tensor:
    """dqkv [B, T, 3 H D]: transposed rotation of dq, dk; dv copied."""
    return _qkv_rope_bwd_impl(dq, dk, dv, cos, sin, pos0)


@qkv_rope_backward_op.register_fake
def _qkv_rope_backward_fake(dq, dk, dv, cos, sin, pos0):
    B, H, T, D = dq.shape
    return dq.new_empty((B, T, 3 * H * D))


def _qkv_rope_setup(ctx, inputs, output):
    _, cos, sin, _, pos0 = inputs
    ctx.save_for_backward(cos, sin)
    ctx.pos0 = pos0


def _qkv_rope_bwd(ctx, dq, dk, dv):
    # Unused outputs arrive as materialised zero gradients.
    cos, sin = ctx.saved_tensors
    return qkv_rope_backward_op(dq, dk, dv, cos, sin, ctx.pos0), None, None, None, None


qkv_rope_op.register_autograd(_qkv_rope_bwd, setup_context=_qkv_rope_setup)


class QKVRopeFn(torch.autograd.Function):
    """The same kernels as t2t::qkv_rope for eager execution (a plain
    autograd.Function has a fraction of the host cost of the custom op's
    registered autograd; compiled graphs trace the custom op)."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, num_heads, pos0):
        ctx.save_for_backward(cos, sin)
        ctx.pos0 = pos0
        return _qkv_rope_impl(qkv, cos, sin, num_heads, pos0)

    @staticmethod
    def backward(ctx, dq, dk, dv):
        cos, sin = ctx.saved_tensors
        return _qkv_rope_bwd_impl(dq, dk, dv, cos, sin, ctx.pos0), None, None, None, None


def qkv_rope_torch(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
                   pos0: int = 0):
    """The same split and rotation composed from torch ops in qkv's dtype, for
    modules whose dtype the prologue kernel does not take (float32)."""
    B, T, D = _split_dims(qkv, num_heads)
    x = qkv.view(B, T, 3, num_heads, D).permute(2, 0, 3, 1, 4)  # [3, B, H, T, D]
    c = cos[pos0:pos0 + T].to(qkv.dtype)
    s = sin[pos0:pos0 + T].to(qkv.dtype)
    h = D // 2

    def rot(t):
        t1, t2 = t[..., :h], t[..., h:]
        return torch.cat((t1 * c + t2 * s, t2 * c - t1 * s), dim=-1)

    return rot(x[0]).contiguous(), rot(x[1]).contiguous(), x[2].contiguous()


def qkv_rope(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
             pos0: int = 0):
    """Split qkv [B, T, 3 C] into rotated q, k and v, each [B, H, T, D]
    (contiguous), with positions pos0 .. pos0 + T - 1 (table rows); the pair
    (a, b) = (x[i], x[i + D/2]) becomes (a cos + b sin, b cos - a sin).  bf16 runs
    the kernel; float32 (module not cast to bf16) the torch composition."""
    if qkv.dtype == torch.float32:
        return qkv_rope_torch(qkv, cos, sin, num_heads, pos0)
    if torch.compiler.is_compiling():
        return qkv_rope_op(qkv, cos, sin, int(num_heads), int(pos0))
    if _lib.unwatched(qkv, cos, sin):
        return _qkv_rope_impl(qkv, cos, sin, int(num_heads), int(pos0))
    return QKVRopeFn.apply(qkv, cos, sin, int(num_heads), int(pos0))


# ---- with norms of queries and keys

def _qk_norm_dims(qkv: torch.Tensor, num_heads: int, num_kv_heads: int):
    B, T, W = qkv.shape
    return B, T, W // (num_heads + 2 * num_kv_heads)


@torch.library.custom_op("t2t::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                    cos: torch.Tensor, sin: torch.Tensor, num_heads: int, num_kv_heads: int,
                    pos0: int, eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q [B, H, T, D] and k, v [B, Hkv, T, D] from qkv [B, T, (H + 2 Hkv) D];
    q and k normed per head and rotated."""
    return _lib.host().qk_norm_rope(qkv, q_weight, k_weight, cos, sin, num_heads, num_kv_heads,
                                    pos0, eps)


@qk_norm_rope_op.register_fake
def _qk_norm_rope_fake(qkv, q_weight, k_weight, cos, sin, num_heads, num_kv_heads, pos0, eps):
    B, T, D = _qk_norm_dims(qkv, num_heads, num_kv_heads)
    return tuple(qkv.new_empty((B, h, T, D)) for h in (num_heads, num_kv_heads, num_kv_heads))


@torch.library.custom_op("t2t::qk_norm_rope_backward", mutates_args=())
def qk_norm_rope_backward_op(
        dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor, qkv: torch.Tensor,
        q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
        num_heads: int, num_kv_heads: int, pos0: int,
        eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dqkv, dq_weight, dk_weight)."""
    return _lib.host().qk_norm_rope_backward(dq, dk, dv, qkv, q_weight, k_weight, cos, sin,
                                             num_heads, num_kv_heads, pos0, eps)


@qk_norm_rope_backward_op.register_fake
def _qk_norm_rope_backward_fake(dq, dk, dv, qkv, q_weight, k_weight, cos, sin, num_heads,
                                num_kv_heads, pos0, eps):
    return (qkv.new_empty(qkv.shape), q_weight.new_empty(q_weight.shape),
            k_weight.new_empty(k_weight.shape))


def _qk_norm_rope_setup(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:5])
    ctx.args = inputs[5:]


def _qk_norm_rope_bwd(ctx, dq, dk, dv):
    dqkv, dqw, dkw = qk_norm_rope_backward_op(dq, dk, dv, *ctx.saved_tensors, *ctx.args)
    return dqkv, dqw, dkw, None, None, None, None, None, None


qk_norm_rope_op.register_autograd(_qk_norm_rope_bwd, setup_context=_qk_norm_rope_setup)


class QKNormRopeFn(torch.autograd.Function):
    """The same kernels as t2t::qk_norm_rope for eager calls that something
    besides autograd watches (the others are recorded by the host module)."""

    @staticmethod
    def forward(ctx, qkv, q_weight, k_weight, cos, sin, *args):
        ctx.save_for_backward(qkv, q_weight, k_weight, cos, sin)
        ctx.args = args
        return _lib.host().qk_norm_rope(qkv, q_weight, k_weight, cos, sin, *args)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk, dv):
        got = _lib.host().qk_norm_rope_backward(dq, dk, dv, *ctx.saved_tensors, *ctx.args)
        return (*got, None, None, None, None, None, None)


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
                 num_kv_heads: Optional[int] = None, pos0: int = 0, eps: float = 1e-6):
    """Split qkv [B, T, (H + 2 Hkv) D] (query heads, key heads, value heads;
    Hkv = H unless ``num_kv_heads`` is given) into q [B, H, T, D] and k, v
    [B, Hkv, T, D] (contiguous): every query and key row RMS-normalised with
    q_weight / k_weight [D] and then rotated at positions pos0 .. pos0 + T - 1
    (table rows), value rows copied.  bf16 or float32 rows, head_dim a
    multiple of 16 up to 512, bf16 or float32 weights; fp32 arithmetic with one
    rounding.  Gradients for qkv and the weights."""
    if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("the rotary tables get no gradient: detach cos and sin")
    args = (int(num_heads), int(num_heads if num_kv_heads is None else num_kv_heads), int(pos0),
            float(eps))
    if torch.compiler.is_compiling():
        return qk_norm_rope_op(qkv, q_weight, k_weight, cos, sin, *args)
    if _lib.unwatched(qkv, q_weight, k_weight, cos, sin):
        return _lib.host().qk_norm_rope(qkv, q_weight, k_weight, cos, sin, *args)
    if _lib.only_recorded(qkv, q_weight, k_weight, cos, sin):
        return _lib.host().qk_norm_rope_ad(qkv, q_weight, k_weight, cos, sin, *args)
    return QKNormRopeFn.apply(qkv, q_weight, k_weight, cos, sin, *args)


@torch.library.custom_op("t2t::qk_norm_rope_append", mutates_args=("k_cache", "v_cache"))
def qk_norm_rope_append_op(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                           cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
                           pos: Optional[torch.Tensor], pos0: int, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, eps: float) -> torch.Tensor:
    """The append for traces: q, with rows of the caches overwritten."""
    return _lib.host().qk_norm_rope_append(qkv, q_weight, k_weight, cos, sin, num_heads, pos, pos0,
                                           k_cache, v_cache, eps)


@qk_norm_rope_append_op.register_fake
def _qk_norm_rope_append_fake(qkv, q_weight, k_weight, cos, sin, num_heads, pos, pos0, k_cache,
                              v_cache, eps):
    return qkv.new_empty((qkv.shape[0], num_heads, qkv.shape[1], q_weight.shape[0]))


def qk_norm_rope_append(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                        cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
                        pos: Union[int, torch.Tensor], k_cache: torch.Tensor,
                        v_cache: torch.Tensor, eps: float = 1e-6) -> torch.Tensor:
    """``qk_norm_rope`` of M new tokens' rows qkv [B, M, (H + 2 Hkv) D] with
    the keys and values written into k_cache / v_cache [B, Hkv, capacity, D]
    at their positions; returns q [B, H, M, D].  Every other cache row is left
    as it is.

    pos: the first token's position (rows at pos .. pos + M - 1), or a device
    int64 tensor [M] or [B, M] of positions, read by the kernel (M at most 8).
    A device position outside the tables or the cache stores nothing and gives
    a query row of zeros; of rows at the same position the last is stored.
    No gradient: for rows that autograd records, use ``qk_norm_rope``; caches
    that require one are refused too, except under torch.no_grad()."""
    rows = (qkv, q_weight, k_weight, cos, sin)
    tensors = (*rows, k_cache, v_cache)
    if (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)
            or forward_ad._current_level >= 0
            and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)):
        raise RuntimeError("qk_norm_rope_append has no gradient: call it under torch.no_grad()")
    at, pos0 = (pos, 0) if isinstance(pos, torch.Tensor) else (None, int(pos))
    args = (*rows, int(num_heads), at, pos0, k_cache, v_cache, float(eps))
    watched = tensors if at is None else (*tensors, at)
    if torch.compiler.is_compiling() or not _lib.only_recorded(*watched):
        return qk_norm_rope_append_op(*args)
    return _lib.host().qk_norm_rope_append(*args)


# ---- any rotary form

@torch.library.custom_op("t2t::qkv_rotary", mutates_args=())
def qkv_rotary_op(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
                  num_kv_heads: int, pos: Optional[torch.Tensor], pos0: int,
                  interleaved: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q [B, H, T, D] and k, v [B, Hkv, T, D] from qkv [B, T, (H + 2 Hkv) D]."""
    return _lib.host().qkv_rotary(qkv, cos, sin, num_heads, num_kv_heads, pos, pos0, interleaved)


@qkv_rotary_op.register_fake
def _qkv_rotary_fake(qkv, cos, sin, num_heads, num_kv_heads, pos, pos0, interleaved):
    B, T, D = _qk_norm_dims(qkv, num_heads, num_kv_heads)
    return tuple(qkv.new_empty((B, h, T, D)) for h in (num_heads, num_kv_heads, num_kv_heads))


@torch.library.custom_op("t2t::qkv_rotary_backward", mutates_args=())
def qkv_rotary_backward_op(dq: torch.Tensor, dk: torch.Tensor, dv: torch.Tensor,
                           cos: torch.Tensor, sin: torch.Tensor, pos: Optional[torch.Tensor],
                           pos0: int, interleaved: bool) -> torch.Tensor:
    """dqkv [B, T, (H + 2 Hkv) D]."""
    return _lib.host().qkv_rotary_backward(dq, dk, dv, cos, sin, pos, pos0, interleaved)


@qkv_rotary_backward_op.register_fake
def _qkv_rotary_backward_fake(dq, dk, dv, cos, sin, pos, pos0, interleaved):
    B, H, T, D = dq.shape
    return dq.new_empty((B, T, (H + 2 * dk.shape[1]) * D))


# The rotation is linear, so each direction's gradient is the other one.
def _qkv_rotary_setup(ctx, inputs, output):
    _, cos, sin, ctx.heads, ctx.kv_heads, pos, ctx.pos0, ctx.interleaved = inputs
    ctx.save_for_backward(cos, sin, pos)


def _qkv_rotary_bwd(ctx, dq, dk, dv):
    cos, sin, pos = ctx.saved_tensors
    d = qkv_rotary_backward_op(dq, dk, dv, cos, sin, pos, ctx.pos0, ctx.interleaved)
    return d, None, None, None, None, None, None, None


def _qkv_rotary_backward_setup(ctx, inputs, output):
    dq, dk, _, cos, sin, pos, ctx.pos0, ctx.interleaved = inputs
    ctx.heads, ctx.kv_heads = dq.shape[1], dk.shape[1]
    ctx.save_for_backward(cos, sin, pos)


def _qkv_rotary_backward_bwd(ctx, d):
    cos, sin, pos = ctx.saved_tensors
    got = qkv_rotary_op(d, cos, sin, ctx.heads, ctx.kv_heads, pos, ctx.pos0, ctx.interleaved)
    return *got, None, None, None, None, None


qkv_rotary_op.register_autograd(_qkv_rotary_bwd, setup_context=_qkv_rotary_setup)
qkv_rotary_backward_op.register_autograd(_qkv_rotary_backward_bwd,
                                         setup_context=_qkv_rotary_backward_setup)


def qkv_rotary(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, num_heads: int,
               num_kv_heads: Optional[int] = None, pos: Union[int, torch.Tensor] = 0,
               interleaved: bool = False):
    """Split qkv [B, T, (H + 2 Hkv) D] (query heads, key heads, value heads;
    Hkv = H unless ``num_kv_heads`` is given) into q [B, H, T, D] and k, v
    [B, Hkv, T, D] (contiguous), the first R dimensions of every query and key
    head rotated by tables cos, sin float32 [rows, R / 2] and the others copied.
    A pair (a, b) becomes (a cos + b sin, b cos - a sin), as in qkv_rope: it turns
    by the tables' negative angle (rotary_tables' ``positive`` for the other way).

    ``interleaved``: pairs of neighbouring dimensions (x[2i], x[2i + 1]) instead
    of (x[i], x[i + R/2]).  ``pos``: the first token's position, or a device
    int64 tensor [T] or [B, T] of positions (read by the kernel, any order,
    repeats too); one without a table row gives query and key rows of zeros and
    no gradient.  bf16 or float32 rows, head_dim a multiple of 16 up to 512, R a
    multiple of 16; fp32 arithmetic with one rounding.  Gradient for qkv."""
    if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("the rotary tables get no gradient: detach cos and sin")
    at, pos0 = (pos, 0) if isinstance(pos, torch.Tensor) else (None, index(pos))
    args = (qkv, cos, sin, index(num_heads),
            index(num_heads if num_kv_heads is None else num_kv_heads), at, pos0, bool(interleaved))
    watched = (qkv, cos, sin) if at is None else (qkv, cos, sin, at)
    if not torch.compiler.is_compiling():
        if _lib.unwatched(*watched):
            return _lib.host().qkv_rotary(*args)
        if _lib.only_recorded(*watched):
            return _lib.host().qkv_rotary_ad(*args)
    return qkv_rotary_op(*args)  # a compiler, or something besides autograd watches
