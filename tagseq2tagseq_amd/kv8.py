"""A key/value cache held in 8 bits, with a scale for each block of 64 positions
and head, and the attention of new rows over it: half of the bf16 cache's
bytes, which are what a generated token's attention waits for.

A value is an e4m3 code times its block's scale, a power of two (keys and
values have their own).  Per sequence, kv head and block the codes are one run:

    k_codes  float8_e4m3fn [B, Hkv, blocks, 64, D]
    v_codes  float8_e4m3fn [B, Hkv, blocks, D, 64]     (positions last)
    k_scale, v_scale  float32 [B, Hkv, blocks]

    kv8_append(k, v, pos, k_codes, v_codes, k_scale, v_scale)
    o, lse2 = attn_decode_kv8(q, k_codes, v_codes, k_scale, v_scale, n_keys, key_doc, key_bits,
                              q_pos, q_doc, q_bits)

``KV8Cache`` holds the four buffers and makes the calls.  No counterpart in the
reference, which keeps no keys or values between tokens
(model/generation_loop.py:90-92).  Kernels: libt2t_attn.so ``t2t_kv8_append``
and ``t2t_kv8_attend``.
"""
from __future__ import annotations

import math
from operator import index
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad

from . import _lib
from .block_mask import check_window

BLOCK = 64      # positions that share a scale
MAX_ROWS = 16   # (Hq / Hkv) * Tq per call


def _refuse_grad(what: str, *tensors) -> None:
    if (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)
            or forward_ad._current_level >= 0
            and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")


@torch.library.custom_op("t2t::kv8_append", mutates_args=("k_codes", "v_codes", "k_scale",
                                                          "v_scale"))
def kv8_append_op(k: torch.Tensor, v: torch.Tensor, pos: Optional[torch.Tensor], pos0: int,
                  k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, capacity: int) -> None:
    """The append for traces."""
    _lib.host().kv8_append(k, v, pos, pos0, k_codes, v_codes, k_scale, v_scale, capacity)


@kv8_append_op.register_fake
def _kv8_append_fake(k, v, pos, pos0, k_codes, v_codes, k_scale, v_scale, capacity):
    return None


def kv8_append(k: torch.Tensor, v: torch.Tensor, pos: Union[int, torch.Tensor],
               k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor,
               v_scale: torch.Tensor, capacity: Optional[int] = None) -> None:
    """Store M new tokens' keys and values k, v [B, Hkv, M, D] (bf16 or float32)
    at positions pos .. pos + M - 1 of every sequence; pos is an int, or a
    device int64 tensor of one position or one for each sequence, read by the
    kernel.  ``capacity``: positions that may be written (default: all blocks).

    The tokens end their sequence: what stands behind them is no longer part of
    it (its codes stay as they were).  A block's scale grows to what its new
    tokens need, and its positions before pos are written again where it did;
    a block that pos begins starts from its new tokens.  A token whose key or
    value is not finite makes every row that reads it NaN.  What the codes hold
    where nothing was stored is never looked at, nor are the scales of blocks
    that no token is in; a block that pos begins inside keeps the scale it has,
    so scales start out as zeros (KV8Cache's do) where positions may be left out.
    A device position below 0 or above capacity - M stores nothing.  No
    gradient."""
    at, pos0 = (pos, 0) if isinstance(pos, torch.Tensor) else (None, index(pos))
    if capacity is not None and capacity < 0:
        raise ValueError(f"capacity={capacity} is negative")
    args = (k, v, at, pos0, k_codes, v_codes, k_scale, v_scale,
            -1 if capacity is None else index(capacity))
    tensors = (k, v, k_codes, v_codes, k_scale, v_scale)
    if (not torch.compiler.is_compiling()
            and _lib.unwatched(*(tensors if at is None else (*tensors, at)))):
        _lib.host().kv8_append(*args)
        return
    _refuse_grad("kv8_append", *tensors)
    kv8_append_op(*args)  # a compiler, or something besides autograd watches


@torch.library.custom_op("t2t::kv8_attend", mutates_args=())
def kv8_attend_op(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                  k_scale: torch.Tensor, v_scale: torch.Tensor, n_keys: int,
                  key_doc: torch.Tensor, key_bits: Optional[torch.Tensor], q_pos: torch.Tensor,
                  q_doc: torch.Tensor, q_bits: Optional[torch.Tensor], scale: float, window: int,
                  sinks: int,
                  q_start: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """The attention for traces (window 0: none)."""
    return _lib.host().kv8_attend(q, k_codes, v_codes, k_scale, v_scale, n_keys, key_doc,
                                  key_bits, q_pos, q_doc, q_bits, scale, window, sinks, q_start)


@kv8_attend_op.register_fake
def _kv8_attend_fake(q, k_codes, v_codes, k_scale, v_scale, n_keys, key_doc, key_bits, q_pos,
                     q_doc, q_bits, scale, window, sinks, q_start):
    return q.new_empty(q.shape), q.new_empty(q.shape[:3], dtype=torch.float32)


def attn_decode_kv8(q: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, n_keys: int,
                    key_doc: torch.Tensor, key_bits: Optional[torch.Tensor], q_pos: torch.Tensor,
                    q_doc: torch.Tensor, q_bits: Optional[torch.Tensor],
                    scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0,
                    q_start: Optional[torch.Tensor] = None):
    """``decode.attn_decode`` over an 8-bit cache: attention of the new rows q
    [B, Hq, Tq, D] (bf16) over positions 0 .. n_keys - 1; the mask's arguments,
    the window and what is returned are as there.  Rows without an allowed key
    give o = 0 and lse2 = -inf.  (Hq / Hkv) * Tq must be at most 16.  No
    gradient."""
    window, sinks = check_window(window, sinks)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    args = (q, k_codes, v_codes, k_scale, v_scale, index(n_keys), key_doc, key_bits, q_pos, q_doc,
            q_bits, float(scale), window or 0, sinks, q_start)
    if (not torch.compiler.is_compiling()
            and _lib.unwatched(*[t for t in args if isinstance(t, torch.Tensor)])):
        return _lib.host().kv8_attend(*args)
    _refuse_grad("attn_decode_kv8", q, k_codes, v_codes, k_scale, v_scale)
    return kv8_attend_op(*args)  # a compiler, or something besides autograd watches


class KV8Cache:
    """The 8-bit cache of ``capacity`` positions of B sequences with Hkv key /
    value heads of head_dim (64 or 128), all zeros."""

    def __init__(self, B: int, Hkv: int, capacity: int, head_dim: int, device):
        if B < 0 or Hkv < 1 or capacity < 1 or head_dim not in (64, 128):
            raise ValueError(f"B={B}, Hkv={Hkv}, capacity={capacity}, head_dim={head_dim}: no "
                             "cache (head_dim 64 or 128)")
        blocks = -(-capacity // BLOCK)
        self.capacity = capacity
        self.k_codes = torch.zeros((B, Hkv, blocks, BLOCK, head_dim), dtype=torch.uint8,
                                   device=device).view(torch.float8_e4m3fn)
        self.v_codes = torch.zeros((B, Hkv, blocks, head_dim, BLOCK), dtype=torch.uint8,
                                   device=device).view(torch.float8_e4m3fn)
        self.k_scale = torch.zeros((B, Hkv, blocks), dtype=torch.float32, device=device)
        self.v_scale = torch.zeros((B, Hkv, blocks), dtype=torch.float32, device=device)

    def buffers(self):
        return self.k_codes, self.v_codes, self.k_scale, self.v_scale

    def append(self, k: torch.Tensor, v: torch.Tensor, pos: Union[int, torch.Tensor]) -> None:
        """kv8_append of the cache."""
        kv8_append(k, v, pos, *self.buffers(), capacity=self.capacity)

    def attend(self, q: torch.Tensor, n_keys: int, key_doc: torch.Tensor,
               key_bits: Optional[torch.Tensor], q_pos: torch.Tensor, q_doc: torch.Tensor,
               q_bits: Optional[torch.Tensor], **kwargs):
        """attn_decode_kv8 of the cache."""
        return attn_decode_kv8(q, *self.buffers(), n_keys, key_doc, key_bits, q_pos, q_doc,
                               q_bits, **kwargs)

    def values(self, dtype: torch.dtype = torch.bfloat16):
        """(k, v) [B, Hkv, capacity, D]: the numbers the cache holds, exact in
        bf16 and float32 alike (in torch operations; for looking at a cache)."""
        k = self.k_codes.float() * self.k_scale[..., None, None]
        v = self.v_codes.float().transpose(3, 4) * self.v_scale[..., None, None]
        return tuple(t.flatten(2, 3)[:, :, :self.capacity].to(dtype) for t in (k, v))
