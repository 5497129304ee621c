"""Inference wrapper with the reference's ``TS2TSModel`` interface, plus a
cached forward for generation.

Mirrors (reference file:line):
  * ``TS2TSModel.__init__`` / ``from_config`` / ``eval`` / ``train`` / ``to``
    (model/model.py:17-211): backbone, embedding / LM-head weights (tied by
    default), final norm, mask creator;
  * ``forward_inference(tokens, doc_spans, **kwargs)`` (model/model.py:214-237):
    mask, embedding, backbone, norm, LM head over the whole sequence.

Added for generation: ``forward_inference_last`` returns the logits of the
last position only -- the single row the generation loop reads
(model/generation_loop.py:90-97) -- and reuses the keys / values of every
position whose inputs are unchanged since the previous call (``KVCache``).
The reusable prefix is the longest one over which the token ids and all mask
inputs (doc id, q words, kv words) agree: a position's hidden states depend
only on the positions before it and on its own mask row, so they are exact
for that prefix.  The cache also records the weights it was filled with --
each parameter's storage address and version counter, and the train / eval
mode -- and is dropped when any of them changes (an optimizer step,
load_state_dict, an in-place edit, train() / eval()).  Writes through a
parameter's ``.data`` bypass its version counter; call ``reset_cache()`` after
such an edit.  New rows go through each layer with the decode-step kernel
(``t2t_attn_decode``, up to 8 rows per kv head per launch, over the 8-bit
cache ``t2t_kv8_attend``, up to 16); when more than
``prefill_rows`` rows are new, the whole sequence is recomputed through the
block-mask kernels and the cache refilled.

``kv_bits = 8`` holds the cache in 8 bits (kv8.py): half of its memory and of
what a token's attention reads; rows that are recomputed as a whole sequence
attend to the keys and values before their rounding.  A mask creator with a
sliding window (mask_creators.SlidingWindowMaskCreator) limits the cached rows
as it limits the whole sequence.
"""
from __future__ import annotations

import ctypes
from typing import Any, Callable, List, Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from .attention import flex_attention
from .block_mask import T2TBlockMask, build_block_mask
from .decode import MAX_ROWS, attn_decode
from .embedding import embedding
from .kv8 import MAX_ROWS as MAX_ROWS_8
from .kv8 import KV8Cache
from .modules import RMSNorm, TS2TSBackbone
from .rope import qk_norm_rope_append
from .rows import applies as rows_apply, rows_linear, rows_qkv_rope


class KVCache:
    """Keys and values of every layer for the cached positions of one
    sequence (batch 1), with the token ids and mask inputs they were computed
    under.  Storage: k, v bf16 [L][1][H][cap][D], or with bits = 8 a KV8Cache a
    layer; doc int32 [1][cap]; q / kv words int64 [1][W][cap]; with a sliding
    window's sinks the documents' starts, int32 [1][cap].  Made outside of inference
    mode, so that calls in and out of it may fill one cache in turn."""

    @torch.inference_mode(False)
    def __init__(self, num_layers: int, num_heads: int, head_dim: int, capacity: int,
                 words: int, device, dtype=torch.bfloat16, bits: int = 16,
                 window: Optional[int] = None, sinks: int = 0):
        self.bits, self.window, self.sinks = bits, window, sinks
        # new rows a launch of attend (one query head per kv head in this model)
        self.max_rows = MAX_ROWS_8 if bits == 8 else MAX_ROWS
        if bits == 8:
            self.layers8 = [KV8Cache(1, num_heads, capacity, head_dim, device)
                            for _ in range(num_layers)]
        else:
            shape = (num_layers, 1, num_heads, capacity, head_dim)
            self.k = torch.empty(shape, dtype=dtype, device=device)
            self.v = torch.empty(shape, dtype=dtype, device=device)
        self.start = (torch.zeros((1, capacity), dtype=torch.int32, device=device) if sinks else
                      None)
        self.tokens = torch.full((1, capacity), -1, dtype=torch.int64, device=device)
        self.doc = torch.empty((1, capacity), dtype=torch.int32, device=device)
        self.q_bits = torch.zeros((1, words, capacity), dtype=torch.int64, device=device)
        self.kv_bits = torch.zeros((1, words, capacity), dtype=torch.int64, device=device)
        self.capacity = capacity
        self.words = words
        self.length = 0

    def fits(self, bm, bits: int) -> bool:
        """Whether rows of the mask inputs ``bm`` belong into this cache."""
        return ((self.words, self.window, self.sinks, self.bits)
                == (bm.words, getattr(bm, "window", None), getattr(bm, "sinks", 0), bits))

    def store(self, i: int, k: torch.Tensor, v: torch.Tensor, pos) -> None:
        """Layer i's keys and values k, v [1, H, n, D] at positions pos .. pos +
        n - 1 (pos an int, or for one row a device int64 tensor [1])."""
        if self.bits == 8:
            self.layers8[i].append(k, v, pos)
        elif isinstance(pos, torch.Tensor):
            self.k[i].index_copy_(2, pos, k)
            self.v[i].index_copy_(2, pos, v)
        else:
            self.k[i, :, :, pos:pos + k.shape[2]] = k
            self.v[i, :, :, pos:pos + k.shape[2]] = v

    def attend(self, i: int, q: torch.Tensor, n_keys: int, q_pos, q_doc, q_bits, q_start,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention rows [1, H, n, D] of layer i's new rows q over the positions
        before n_keys (in ``out`` where it is given)."""
        mask = (n_keys, self.doc, self.kv_bits if self.words else None, q_pos, q_doc, q_bits)
        limits = dict(window=self.window, sinks=self.sinks, q_start=q_start)
        if self.bits == 8:
            y = self.layers8[i].attend(q, *mask, **limits)[0]
            return y if out is None else out.copy_(y)
        return attn_decode(q, self.k[i], self.v[i], *mask, out=out, **limits)[0]

    def first_diff(self, tokens: torch.Tensor, bm, n: int) -> torch.Tensor:
        """Device int32 [1]: the first of positions 0 .. n - 1 whose token id
        or mask inputs (doc id, q / kv words) differ from the cached ones, or n
        (``t2t_first_input_diff`` lowering a fill of n; no host sync)."""
        out = torch.full((1,), n, dtype=torch.int32, device=self.tokens.device)

        def row(t):
            t = t[0]
            return t if t.stride(-1) == 1 else t.contiguous()

        tok, doc = row(tokens.to(torch.int64)), row(bm.doc_ids.to(torch.int32))
        qa = ka = qb = kb = None
        if self.words:
            qa, ka, qb, kb = (row(t) for t in (self.q_bits, self.kv_bits, bm.q_bits, bm.kv_bits))
            if qb.stride(0) != kb.stride(0):
                qb, kb = qb.contiguous(), kb.contiguous()
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        with torch.cuda.device(out.device):
            rc = _lib.lib().t2t_first_input_diff(
                self.tokens.data_ptr(), tok.data_ptr(), self.doc.data_ptr(), doc.data_ptr(),
                ptr(qa), ptr(qb), ptr(ka), ptr(kb), qa.stride(0) if qa is not None else 0,
                qb.stride(0) if qb is not None else 0, self.words, n, out.data_ptr(),
                ctypes.c_void_p(torch.cuda.current_stream(out.device).cuda_stream))
        _lib.check(rc, "t2t_first_input_diff")
        return out

    def reusable_prefix(self, tokens: torch.Tensor, bm) -> int:
        """Length of the longest prefix whose token ids and mask inputs match."""
        n = min(self.length, tokens.shape[1])
        return int(self.first_diff(tokens, bm, n).item()) if n else 0

    def store_inputs(self, tokens: torch.Tensor, bm, p0: int, p1: int) -> None:
        self.tokens[0, p0:p1] = tokens[0, p0:p1]
        self.doc[0, p0:p1] = bm.doc_ids[0, p0:p1]
        if self.sinks:
            self.start[0, p0:p1] = bm.doc_start[0, p0:p1]
        if self.words:
            self.q_bits[0, :, p0:p1] = bm.q_bits[0, :, p0:p1]
            self.kv_bits[0, :, p0:p1] = bm.kv_bits[0, :, p0:p1]


class TS2TSModel:
    """model/model.py:17-237 (generation / evaluation helpers that need the
    absent tokenizer stack are not provided)."""

    def __init__(self, backbone: TS2TSBackbone, embedding_weight: torch.Tensor,
                 lm_head_weight: torch.Tensor, norm: nn.Module, block_mask_creator: Callable,
                 vocab_size: int, ignore_index: int = -100, tokenizer=None, link_detector=None,
                 layout_policy=None, embedding_scale: Optional[float] = None):
        self.backbone = backbone
        self.embedding_weight = embedding_weight
        self.lm_head_weight = lm_head_weight
        self.norm = norm
        self.block_mask_creator = block_mask_creator
        self.vocab_size = vocab_size
        self.ignore_index = ignore_index
        self.tokenizer = tokenizer
        self.link_detector = link_detector
        self.layout_policy = layout_policy
        self.embedding_scale = embedding_scale  # factor on the embedding's rows, or None
        self.kv_cache: Optional[KVCache] = None
        self.prefill_rows = 64
        self.kv_bits = 16  # of the key/value cache: 16 (bf16) or 8
        self.use_graphs = True
        self.fuse_rows = True  # few-row steps on the fused row kernels (rows.py)
        self._graph: Optional[_DecodeGraph] = None
        self._weights_seen = None  # _weights_state() the cache was filled under
        self._param_slots = None   # (module, name) of every backbone / norm parameter

    @classmethod
    def from_config(cls, vocab_size: int, num_layers: int, model_dim: int, num_heads: int,
                    max_seq_len: int, dropout: float, drop_path_rate: float,
                    block_mask_creator: Callable, fp8: bool = False, weight_tying: bool = True,
                    ignore_index: int = -100, tokenizer=None, link_detector=None,
                    layout_policy=None, qk_norm: bool = False,
                    embedding_scale: Optional[float] = None, rotary=None) -> "TS2TSModel":
        backbone = TS2TSBackbone(num_layers=num_layers, model_dim=model_dim, num_heads=num_heads,
                                 max_seq_len=max_seq_len, dropout=dropout,
                                 drop_path_rate=drop_path_rate, fp8=fp8, qk_norm=qk_norm,
                                 rotary=rotary)
        table = nn.Embedding(vocab_size, model_dim)
        norm = RMSNorm(model_dim)
        if weight_tying:
            lm_head_weight = table.weight
        else:
            lm_head_weight = nn.Parameter(torch.empty(vocab_size, model_dim))
            nn.init.normal_(lm_head_weight, mean=0.0, std=0.02)
        return cls(backbone, table.weight, lm_head_weight, norm, block_mask_creator,
                   vocab_size, ignore_index, tokenizer, link_detector, layout_policy,
                   embedding_scale)

    def eval(self):
        self.backbone.eval()
        return self

    def train(self, mode: bool = True):
        self.backbone.train(mode)
        return self

    def to(self, device, dtype=None):
        self.backbone.to(device, dtype)
        self.norm.to(device, dtype)
        tied = self.lm_head_weight is self.embedding_weight
        self.embedding_weight = self.embedding_weight.to(device=device, dtype=dtype)
        self.lm_head_weight = (self.embedding_weight if tied else
                               self.lm_head_weight.to(device=device, dtype=dtype))
        self.kv_cache = None
        self._graph = None
        return self

    def reset_cache(self) -> None:
        self.kv_cache = None
        self._graph = None
        self._weights_seen = None
        self._param_slots = None

    def _weights_state(self):
        """What the cached keys / values depend on besides the inputs: the mode
        and, per parameter, its storage address and version counter (bumped by
        every in-place write through the parameter, optimizer steps and
        load_state_dict included).  The (module, attribute) slots that hold
        the parameters are listed once (walking the module tree per token cost
        ~0.2 ms of host time before each step); each call reads the slots
        again, so a parameter assigned anew is seen.  Submodules replaced
        after the first cached call need reset_cache()."""
        if self._param_slots is None:
            self._param_slots = [(m, name) for owner in (self.backbone, self.norm)
                                 for m in owner.modules()
                                 for name, prm in m._parameters.items() if prm is not None]
        params = [m._parameters.get(name) for m, name in self._param_slots]
        params += (self.embedding_weight, self.lm_head_weight)
        return (self.backbone.training, self.embedding_scale,
                tuple(None if p is None else (p.data_ptr(), p._version)
                      for p in params))

    @torch.no_grad()
    def forward_inference(self, tokens: torch.Tensor, doc_spans: Optional[List[Any]] = None,
                          **kwargs) -> torch.Tensor:
        """model/model.py:214-237: logits [1, T, V] over the whole sequence."""
        block_mask = self.block_mask_creator(tokens=tokens, doc_spans=doc_spans or [], **kwargs)
        x = self._embed(tokens)
        x = self.backbone(x, block_mask=block_mask)
        x = self.norm(x)
        return F.linear(x, self.lm_head_weight)

    def _embed(self, tokens: torch.Tensor) -> torch.Tensor:
        if self.embedding_scale is None:
            return F.embedding(tokens, self.embedding_weight)
        return embedding(tokens, self.embedding_weight, self.embedding_scale)

    # -- cached path -------------------------------------------------------

    def _layers(self):
        return self.backbone.layers

    def _new_cache(self, bm, device) -> KVCache:
        attn = self._layers()[0].attn
        return KVCache(len(self._layers()), attn.num_heads, attn.head_dim,
                       self._layers()[0].attn.rotary.max_seq_len, bm.words, device,
                       self.embedding_weight.dtype, self.kv_bits, getattr(bm, "window", None),
                       getattr(bm, "sinks", 0))

    @torch.no_grad()
    def forward_inference_last(self, tokens: torch.Tensor,
                               doc_spans: Optional[List[Any]] = None, **kwargs) -> torch.Tensor:
        """Logits [1, 1, V] of the last position of ``tokens`` [1, T]; equal
        (to bf16 rounding) to ``forward_inference(tokens, doc_spans)[:, -1:]``."""
        if tokens.shape[0] != 1:
            raise ValueError("the cached path serves one sequence (batch 1)")
        if self.embedding_weight.dtype != torch.bfloat16:
            # The key/value cache and the decode kernel are bf16; a float32
            # model recomputes the sequence on the float32 attention kernels.
            return self.forward_inference(tokens, doc_spans, **kwargs)[:, -1:]
        if self.kv_bits not in (8, 16):
            raise ValueError(f"kv_bits={self.kv_bits!r}: the cache holds 16 or 8 bits")
        # Per-token mask inputs only; the tile tables are built below if the
        # whole sequence has to be recomputed.
        bm = self.block_mask_creator(tokens=tokens, doc_spans=doc_spans or [], inputs_only=True,
                                     **kwargs)
        T = tokens.shape[1]
        state = self._weights_state()
        if state != self._weights_seen:
            self.reset_cache()
            self._weights_seen = state
        cache = self.kv_cache
        if cache is None or not cache.fits(bm, self.kv_bits) or T > cache.capacity:
            cache = self.kv_cache = self._new_cache(bm, tokens.device)
            self._graph = None
        p = T - 1
        if self.use_graphs and p >= 1 and cache.length >= p:
            # The generation case: the cached prefix covers every position but
            # the last.  Launch the single-row step at once and check the
            # prefix on the device beside it; the check is read back after the
            # step's launches, so the step costs one host synchronisation.
            cache.store_inputs(tokens, bm, p, T)
            logits = self._graph_step(cache, tokens, bm, p)
            first = cache.first_diff(tokens, bm, p)  # reads positions < p only
            if int(first.item()) == p:
                cache.length = T
                return logits
            # an earlier input changed: recompute from the first difference
            cache.length = int(first.item())
        p0 = min(cache.reusable_prefix(tokens, bm), T - 1)
        full = T - p0 > self.prefill_rows
        if full:
            p0 = 0
            if not isinstance(bm, T2TBlockMask):
                bm = build_block_mask(bm.doc_ids, bm.q_bits, bm.kv_bits, window=cache.window,
                                      sinks=cache.sinks)
        cache.length = p0  # positions >= p0 are rewritten below
        cache.store_inputs(tokens, bm, p0, T)
        if self.use_graphs and not full and T - p0 == 1:
            logits = self._graph_step(cache, tokens, bm, p0)
            cache.length = T
            return logits
        x = self._embed(tokens[:, p0:])
        x = self._backbone_rows(x, bm, cache, p0, full)
        cache.length = T
        x = x[:, -1:]
        if self._rows_fusable(x):
            return rows_linear(x, self.lm_head_weight, norm=self.norm)
        return F.linear(self.norm(x), self.lm_head_weight)

    def _graph_step(self, cache: KVCache, tokens: torch.Tensor, bm, p: int) -> torch.Tensor:
        """One new row at position p through the captured decode step."""
        if (self._graph is None or self._graph.cache is not cache
                or self._graph.fused != self.fuse_rows):
            self._graph = _DecodeGraph(self, cache)
        return self._graph.run(p)

    def _step_body(self, cache: KVCache, buf: "_DecodeGraph") -> torch.Tensor:
        """The single-row step over static buffers (no host values in any
        launch): embedding, every layer with its cache write and decode
        attention over the whole cache capacity (slots past the new row are
        excluded by the causal test), final norm and LM head."""
        # The new row's token id and mask inputs, written into the cache at
        # position pos before every replay, are gathered inside the graph.
        tok = cache.tokens.index_select(1, buf.pos)
        qdoc = cache.doc.index_select(1, buf.pos)
        qbits = cache.q_bits.index_select(2, buf.pos) if cache.words else None
        qstart = cache.start.index_select(1, buf.pos) if cache.sinks else None
        qpos = buf.pos.to(torch.int32).view(1, 1)
        x = self._embed(tok)
        fused = self._rows_fusable(x)
        bb = self.backbone
        skips = []
        n_skip = len(bb.skip_weights)
        carried = False  # this layer's skip add was folded into the previous layer
        for i, layer in enumerate(bb.layers):
            if i >= n_skip and skips and not carried:
                x = x + bb.skip_weights[i - n_skip] * skips.pop()
            C = x.shape[-1]
            nxt = self._next_skip(i, skips) if fused else None
            q, _, _ = self._new_rows(i, layer, x, fused, cache, buf.pos)
            y = cache.attend(i, q, cache.capacity, qpos, qdoc, qbits, qstart)
            x = self._layer_tail(layer, y.transpose(1, 2).reshape(1, 1, C), x, fused, nxt)
            carried = nxt is not None
            if i < n_skip and not carried:
                skips.append(x)
        if fused:
            return rows_linear(x, self.lm_head_weight, norm=self.norm)
        return F.linear(self.norm(x), self.lm_head_weight)

    @staticmethod
    def _new_rows(i: int, layer, x, fused: bool, cache: KVCache, pos):
        """Query rows of layer i for the rows x at positions pos .. (an int, or
        for one row a device int64 tensor [1]), their keys and values put into the
        cache; also these as the kernels left them, [1, H, n, D] (None, None
        where they went to the cache alone)."""
        attn = layer.attn
        cos, sin = attn.rotary.tables(x.device)
        if cache.bits == 16 and fused and attn.rotary.whole_halves and not attn.qk_norm:
            return rows_qkv_rope(x, attn.qkv.weight, attn.num_heads, cos, sin, pos, cache.k[i],
                                 cache.v[i], norm=layer.ln_1), None, None
        h = (rows_linear(x, attn.qkv.weight, norm=layer.ln_1) if fused else
             attn.qkv(layer.ln_1(x)))
        if cache.bits == 16 and attn.qk_norm:
            return qk_norm_rope_append(h, attn.q_norm, attn.k_norm, cos, sin, attn.num_heads, pos,
                                       cache.k[i], cache.v[i], eps=attn.NORM_EPS), None, None
        q, k, v = attn.heads(h, pos)
        cache.store(i, k, v, pos)
        return q, k, v

    def _rows_fusable(self, x) -> bool:
        """Whether the layers of a few-row step can run on the fused row
        kernels (rows.py): bf16 rows and weights on the GPU, at most 8 rows,
        SwiGLU GLUs, and dropout / drop-path that are the identity."""
        if (not self.fuse_rows or not rows_apply(x, self.lm_head_weight)
                or not self.lm_head_weight.is_contiguous()):
            return False
        for layer in self._layers():
            mlp = layer.mlp
            if (mlp.act is not F.silu or not isinstance(layer.ln_1, RMSNorm)
                    or not isinstance(layer.ln_2, RMSNorm)):
                return False
            if layer.training and (layer.drop_path.p > 0 or mlp.dropout.p > 0):
                return False
            ws = (layer.attn.qkv.weight, layer.attn.proj.weight, mlp.gate_up.weight,
                  mlp.down.weight)
            if not all(w.dtype == torch.bfloat16 and w.is_contiguous() for w in ws):
                return False
            if mlp.down.weight.shape[1] > 4096:
                return False
        return isinstance(self.norm, RMSNorm)

    def _next_skip(self, i: int, skips: list):
        """The skip add that starts layer i + 1 (model/modules/backbone.py:93-104:
        x + skip_weights[j - n_skip] * skips.pop() for layers j >= n_skip),
        to be folded into layer i's down-projection: (rows, weight), rows None
        when layer i + 1 pops layer i's own output; None when layer i + 1 adds
        nothing."""
        bb = self.backbone
        n_skip, j = len(bb.skip_weights), i + 1
        if j >= len(bb.layers) or j < n_skip:
            return None
        if i == n_skip - 1:
            return None, bb.skip_weights[0]
        if not skips:
            return None
        return skips.pop(), bb.skip_weights[j - n_skip]

    @staticmethod
    def _layer_tail(layer, y, x, fused: bool, skip=None):
        """Out-projection + residual, norm + GLU + residual of Layer.forward
        (model/modules/layer.py:33-34) on the attention rows y; ``skip``: the
        next layer's skip add, folded into the last product (fused only)."""
        if fused:
            mlp = layer.mlp
            x = rows_linear(y, layer.attn.proj.weight, epilogue="add", res=x)
            h = rows_linear(x, mlp.gate_up.weight, norm=layer.ln_2, epilogue="swiglu")
            return rows_linear(h, mlp.down.weight, epilogue="add", res=x, skip=skip)
        x = x + layer.drop_path(layer.attn.proj(y))
        return x + layer.drop_path(layer.mlp(layer.ln_2(x)))

    def _backbone_rows(self, x, bm, cache: KVCache, p0: int, full: bool):
        """TS2TSBackbone.forward (skip wiring of model/modules/backbone.py:93-104)
        over rows p0 .. T - 1 with cached attention."""
        bb = self.backbone
        skips = []
        n_skip = len(bb.skip_weights)
        fused = not full and self._rows_fusable(x)
        carried = False  # this layer's skip add was folded into the previous layer
        for i, layer in enumerate(bb.layers):
            if i >= n_skip and skips and not carried:
                x = x + bb.skip_weights[i - n_skip] * skips.pop()
            nxt = self._next_skip(i, skips) if fused else None
            x = self._layer_rows(i, layer, x, bm, cache, p0, full, fused, nxt)
            carried = nxt is not None
            if i < n_skip and not carried:
                skips.append(x)
        return x

    def _layer_rows(self, i: int, layer, x, bm, cache: KVCache, p0: int, full: bool,
                    fused: bool, skip=None):
        """Layer.forward (model/modules/layer.py:32-35) over the new rows."""
        B, n, C = x.shape
        T = p0 + n
        q, k, v = self._new_rows(i, layer, x, fused, cache, p0)
        if full:
            if k is None:
                k, v = cache.k[i, :, :, p0:T], cache.v[i, :, :, p0:T]
            y = flex_attention(q, k, v, block_mask=bm)
        else:
            y = torch.empty_like(q)
            rows = cache.max_rows
            pos = torch.arange(p0, T, dtype=torch.int32, device=x.device)[None]
            for c0 in range(0, n, rows):
                c1 = min(n, c0 + rows)
                at = slice(p0 + c0, p0 + c1)
                cache.attend(i, q[:, :, c0:c1], p0 + c1, pos[:, c0:c1].contiguous(),
                             bm.doc_ids[:, at].contiguous(),
                             bm.q_bits[:, :, at].contiguous() if bm.words else None,
                             bm.doc_start[:, at].contiguous() if cache.sinks else None,
                             out=y[:, :, c0:c1])
        return self._layer_tail(layer, y.transpose(1, 2).reshape(B, n, C), x, fused, skip)


class _DecodeGraph:
    """The single-row decode step of a TS2TSModel captured as a HIP graph
    (torch.cuda.graph) over one static buffer, the row's position: the step
    gathers the row's token id and mask inputs from the cache, where
    ``store_inputs`` has written them before the replay.  Replays cost two
    launches from the host (the position and the graph) instead of the
    launches of the eager step (six per layer on the fused row kernels, ~15
    without them); the recorded kernels (the row kernels and the decode
    kernels, or hipBLASLt GEMMs, torch elementwise / reduction kernels and
    the prologue kernel) write no memset nodes of their own."""

    @torch.inference_mode(False)  # (as the cache)
    def __init__(self, model: TS2TSModel, cache: KVCache):
        self.cache = cache
        self.pos = torch.zeros((1,), dtype=torch.int64, device=cache.tokens.device)
        self.model = model
        self.fused = model.fuse_rows
        self.graph = None
        self.logits = None

    @torch.inference_mode(False)  # (torch keeps tensors of its own from a first capture too)
    @torch.no_grad()
    def _capture(self):
        """Warm up on a side stream (default priority), then capture.  The
        buffers already hold the first step's values, so the warm-up run writes
        exactly what the first replay writes."""
        dev = self.pos.device
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            self.model._step_body(self.cache, self)
        torch.cuda.current_stream(dev).wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.logits = self.model._step_body(self.cache, self)

    def run(self, p: int) -> torch.Tensor:
        """Logits of the row at position p, whose inputs are in the cache."""
        self.pos.fill_(p)
        if self.graph is None:
            self._capture()
        self.graph.replay()
        return self.logits.clone()

