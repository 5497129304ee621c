"""Decode-step attention on the gfx950 kernels: a few new query rows against
a key/value cache, the mask evaluated per key from the per-token mask inputs
(doc ids and q / kv words, the layout ``T2TBlockMask`` carries).

Replaces, for generation, the full recompute the reference does per token
(model/generation_loop.py:90-92 -> TS2TSModel.forward_inference,
model/model.py:214-237).  Kernels: libt2t_attn.so ``t2t_attn_decode`` and, with
a sliding window, ``t2t_attn_decode_window``.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from .block_mask import check_window

MAX_ROWS = 8  # (Hq / Hkv) * Tq per call


def attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, n_keys: int,
                key_doc: torch.Tensor, key_bits: Optional[torch.Tensor], q_pos: torch.Tensor,
                q_doc: torch.Tensor, q_bits: Optional[torch.Tensor],
                scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                window: Optional[int] = None, sinks: int = 0,
                q_start: Optional[torch.Tensor] = None):
    """Attention of the new rows q [B, Hq, Tq, D] over cache positions
    0 .. n_keys - 1 of k_cache / v_cache [B, Hkv, cap, D].

    key_doc int32 [Bm, cap], key_bits int64 [Bm, W, cap] (or None for W = 0);
    q_pos / q_doc int32 [Bm, Tq], q_bits int64 [Bm, W, Tq].  Key j is allowed
    for row t iff j <= q_pos[t] and (key_doc[j] == q_doc[t] or the rows share a
    word bit).  With ``window``, a key of the row's own document is allowed only
    within the last ``window`` positions, q_pos[t] - j < window, or among the
    first ``sinks`` of the document, 0 <= j - q_start[t] < sinks (q_start int32
    [Bm, Tq], its first position).  Returns (o [B, Hq, Tq, D] bf16, lse2 float32
    [B, Hq, Tq], log2 domain).  (Hq / Hkv) * Tq must be at most 8."""
    window, sinks = check_window(window, sinks)
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return _lib.host().attn_decode(q, k_cache, v_cache, n_keys, key_doc, key_bits, q_pos, q_doc,
                                   q_bits, scale, out, window or 0, sinks, q_start)
