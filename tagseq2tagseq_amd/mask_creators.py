"""Mask creators with the reference's signatures, returning ``T2TBlockMask``.

Mirrors model/graph_traversal/block_mask_creator.py and cross_doc_mask.py:

* ``create_doc_causal_block_mask(tokens, doc_spans, **kw)``   -- :87-141
* ``create_causal_block_mask(tokens, doc_spans, **kw)``       -- :144-… (one
  document covering the row; causal only)
* ``CrossDocLinkMaskCreator(link_detector, max_grants, ...)`` -- cross_doc_mask.py:25-369
  (same link matching, DAG rule, grant bitmask construction and cosine
  max-grants warm-up)
* ``create_doc_link_block_mask(tokens, doc_spans, doc_links)`` -- the doc x doc
  link-bitmask form of the cross_doc_link mask (lower-triangular rows with the
  diagonal set), expressed in the same (q_bitmask, kv_bitmask) encoding
* ``SlidingWindowMaskCreator(creator, window, sinks)`` -- any of them with a
  sliding window (no counterpart in the reference); the creators' own keywords
  ``window=`` and ``sinks=`` give the same mask
* ``MASK_CREATORS`` / ``get_mask_creator`` / ``list_mask_creators`` /
  ``make_mask_creator_callable_from`` / ``make_mask_creator_callable`` -- :252-334

Per-token inputs (document ids, grant words) are built on the GPU from the
span and grant lists by t2t_token_inputs, replacing the reference's
per-span / per-grant device slice loops; only the O(#spans + #grants) lists
travel from the host.  Tile classification and the index tables are then
computed on the GPU by the metadata kernel.
"""
from __future__ import annotations

import logging
import math
from typing import Any, Dict, List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import _lib
from .block_mask import T2TBlockMask, build_block_mask, check_window, mask_inputs

logger = logging.getLogger(__name__)


def _device_of(tokens: torch.Tensor) -> torch.device:
    if not tokens.is_cuda:
        raise RuntimeError("mask creators need `tokens` on a ROCm GPU device "
                           "(the masked-attention path has no CPU implementation)")
    return tokens.device


def _clip_i32(x: int, T: int) -> int:
    """A span / grant bound clipped to [-1, T + 1] (same coverage of [0, T))."""
    return int(min(max(int(x), -1), T + 1))


class TokenLists:
    """Span / grant / link lists of B mask rows, resident on the device, from
    which ``build()`` makes the per-token inputs of the metadata pass with one
    t2t_token_inputs launch.

    ``span_rows[b]``: the row's spans in order (later ones overwrite earlier
    ones, as in block_mask_creator.py:107-117).  ``grant_rows[b]``: (bit,
    q_start, q_end, kv_start, kv_end) entries (cross_doc_mask.py:282-289).
    ``link_rows[b]``: uint64 [n_spans, words] doc x doc link rows.  Only these
    lists travel from the host (one int32 upload plus the link rows).
    """

    def __init__(self, seq_len: int, span_rows: Sequence[Sequence], device: torch.device,
                 words: int = 0,
                 grant_rows: Optional[Sequence[Sequence[Tuple[int, int, int, int, int]]]] = None,
                 link_rows: Optional[Sequence[np.ndarray]] = None):
        T = int(seq_len)
        B = len(span_rows)
        ms = max(1, max((len(r) for r in span_rows), default=0))
        mg = max(1, max((len(r) for r in grant_rows), default=0)) if grant_rows is not None else 1
        sp = np.zeros((B, ms, 3), dtype=np.int32)
        gr = np.zeros((B, mg, 5), dtype=np.int32)
        cnt = np.zeros((2, B), dtype=np.int32)
        for b, row in enumerate(span_rows):
            if row:
                try:  # one array per row; bounds beyond int64 take the scalar path
                    a = np.array([(s.start, s.end, s.doc_id) for s in row], dtype=np.int64)
                    sp[b, :len(row), :2] = np.clip(a[:, :2], -1, T + 1)
                    sp[b, :len(row), 2] = a[:, 2].astype(np.int32)
                except OverflowError:
                    for i, s in enumerate(row):
                        sp[b, i] = (_clip_i32(s.start, T), _clip_i32(s.end, T),
                                    np.int64(s.doc_id).astype(np.int32))
            cnt[0, b] = len(row)
        if grant_rows is not None:
            for b, row in enumerate(grant_rows):
                if len(row):
                    try:
                        a = np.array(row, dtype=np.int64).reshape(-1, 5)
                        gr[b, :len(row), 0] = a[:, 0]
                        gr[b, :len(row), 1:] = np.clip(a[:, 1:], -1, T + 1)
                    except OverflowError:
                        for i, (bit, qs, qe, ks, ke) in enumerate(row):
                            gr[b, i] = (bit, _clip_i32(qs, T), _clip_i32(qe, T),
                                        _clip_i32(ks, T), _clip_i32(ke, T))
                cnt[1, b] = len(row)
        parts = [sp.ravel(), gr.ravel(), cnt.ravel()]
        n = sum(p.size for p in parts)
        self._links = -1  # int32 offset of the link rows behind the lists (8-byte aligned)
        if link_rows is not None:
            la = np.zeros((B, ms, words), dtype=np.uint64)
            for b, rows in enumerate(link_rows):
                r = np.asarray(rows, dtype=np.uint64).reshape(-1, words)
                la[b, :r.shape[0]] = r
            self._links = n + n % 2
            parts += [np.zeros(n % 2, dtype=np.int32), la.ravel().view(np.int32)]
        both = torch.from_numpy(np.concatenate(parts)).to(device)  # one upload
        self.lists = both[:n]
        self.links = None if link_rows is None else both[self._links:].view(torch.int64).view(
            B, ms, words)
        self.device, self.B, self.T, self.words = device, B, T, words
        self.max_spans, self.max_grants = ms, mg
        self.has_grants = grant_rows is not None
        self._off = (sp.size, sp.size + gr.size)

    def build(self, out=None):
        """(doc int32 [B, T], q_bits, kv_bits int64 [B, words, T] or None).
        ``out``: a previous result to overwrite instead of allocating."""
        grants, counts = self._off
        given = [] if out is None else [x for x in out if x is not None]
        t = _lib.host().token_inputs(
            self.lists, grants, counts, self._links, self.B, self.T, self.words, self.max_spans,
            self.max_grants, self.has_grants, given)
        if out is not None:
            return tuple(out)
        return tuple(t) if self.words > 0 else (t[0], None, None)


def token_inputs(seq_len: int, doc_spans: Sequence, device: torch.device, words: int = 0,
                 grants: Optional[Sequence[Tuple[int, int, int, int, int]]] = None,
                 links: Optional[np.ndarray] = None):
    """Per-token inputs of one mask row (the reference's B=None masks) built
    on the device; see TokenLists."""
    return TokenLists(seq_len, [doc_spans], device, words,
                      None if grants is None else [grants],
                      None if links is None else [links]).build()


def document_ids_host(seq_len: int, doc_spans: Sequence) -> np.ndarray:
    """Doc-id map of block_mask_creator.py:107-117 (-1 = not covered; later
    spans overwrite earlier ones)."""
    ids = np.full(seq_len, -1, dtype=np.int32)
    for span in doc_spans:
        start = max(0, span.start)
        end = min(seq_len, span.end)
        if start < end:
            ids[start:end] = span.doc_id
    return ids


def _finish(doc, qb, kb, kwargs):
    """The creators' result: the BlockMask, or with ``inputs_only=True`` just
    its per-token inputs (what the cached generation path reads).  ``window``
    and ``sinks``: of a sliding window (block_mask.build_block_mask)."""
    limits = dict(window=kwargs.get("window"), sinks=kwargs.get("sinks", 0))
    if kwargs.get("inputs_only"):
        return mask_inputs(doc, qb, kb, **limits)
    return build_block_mask(doc, qb, kb, **limits)


def create_doc_causal_block_mask(tokens: torch.Tensor, doc_spans: List[Any], **kwargs) -> T2TBlockMask:
    """block_mask_creator.py:87-141: causal & same document."""
    device = _device_of(tokens)
    doc, _, _ = token_inputs(tokens.shape[-1], doc_spans, device)
    return _finish(doc, None, None, kwargs)


def create_causal_block_mask(tokens: torch.Tensor, doc_spans: List[Any], **kwargs) -> T2TBlockMask:
    """Plain causal mask (every token in one document)."""
    device = _device_of(tokens)
    seq_len = tokens.shape[-1]
    return _finish(torch.zeros(seq_len, dtype=torch.int32, device=device), None, None, kwargs)


def create_doc_link_block_mask(tokens: torch.Tensor, doc_spans: List[Any],
                               doc_links: np.ndarray, **kwargs) -> T2TBlockMask:
    """cross_doc_link mask from a per-sequence doc x doc link bitmask.

    ``doc_links``: uint64 [n_docs, W]; bit j of row i lets document i (the i-th
    span) read document j (j <= i; the diagonal is implied by same-document
    attention).  Grant bit j is "target document j": kv_bits[t] = 1 << doc(t),
    q_bits[t] = doc_links[doc(t)], so (q_bits & kv_bits) != 0 exactly when the
    query's document links the key's document -- the mask_mod of
    cross_doc_mask.py:348-357 on these words.
    """
    device = _device_of(tokens)
    T = tokens.shape[-1]
    links = np.asarray(doc_links, dtype=np.uint64)
    if links.ndim != 2 or links.shape[0] != len(doc_spans):
        raise ValueError(f"doc_links must be [n_docs={len(doc_spans)}, W], got {links.shape}")
    W = links.shape[1]
    if W * 64 < len(doc_spans):
        raise ValueError(f"{len(doc_spans)} documents need {math.ceil(len(doc_spans) / 64)} words, got {W}")
    doc, qb, kb = token_inputs(T, doc_spans, device, words=W, links=links)
    return _finish(doc, qb, kb, kwargs)


class CrossDocLinkMaskCreator:
    """cross_doc_mask.py:25-369 with the device-side metadata pass.

    ``link_detector`` is any object with ``detect_links(input_ids) ->
    List[LinkInfo]`` (``link_end_pos``, ``target_str``) and
    ``index_doc_span(span) -> str`` (model/graph_traversal/link_detector.py:15-84).
    """

    def __init__(self, link_detector, max_grants: int = 64,
                 max_grants_start: Optional[int] = None, max_grants_warmup_steps: int = 0):
        self.link_detector = link_detector
        self.max_grants = max_grants
        self._max_grants_start = max_grants_start if max_grants_start is not None else max_grants
        self._max_grants_warmup_steps = max_grants_warmup_steps
        self._step = 0
        # sized for the final max_grants so the kernel inputs keep one shape (:67)
        self._n_chunks = max(1, (max_grants + 63) // 64)

    def _current_max_grants(self) -> int:
        """Grant budget of the current step (:76-85): max_grants_start rising to
        max_grants along half a cosine period over the warm-up steps, rounded
        with Python's round(); max_grants once the warm-up is over."""
        steps = self._max_grants_warmup_steps
        if steps <= 0 or self._step >= steps:
            return self.max_grants
        ramp = (1.0 - math.cos(math.pi * (self._step / steps))) * 0.5
        lo, hi = self._max_grants_start, self.max_grants
        return round(lo + (hi - lo) * ramp)

    def _match_links_to_docs(self, links, doc_spans) -> Dict[int, List[int]]:
        """{link_end_pos: [target doc ids in link order]} for the links whose
        target is a span of this pack that starts before the link (:87-149).
        When two spans index to the same key, the later one wins."""
        key_of = self.link_detector.index_doc_span
        where = {key_of(sp): (sp.doc_id, sp.start) for sp in doc_spans}
        grouped: Dict[int, List[int]] = {}
        for link in links:
            pos = link.link_end_pos
            found = where.get(link.target_str)
            if found is not None and found[1] < pos:  # targets must precede the link
                grouped.setdefault(pos, []).append(found[0])
        return grouped

    def _grant_ranges(self, seq_len: int, doc_spans, link_to_target,
                      max_grants_cap: Optional[int] = None) -> List[Tuple[int, int, int, int, int]]:
        """The grants of :210-300 as (bit, q_start, q_end, kv_start, kv_end).

        Links are visited by position, each link's targets in order.  A grant
        lets the queries from the link position to the end of the span holding
        the link (the first span s with s.start < pos <= s.end) read the first
        span carrying the target doc id, both ranges clipped to the sequence.
        Grants are numbered in visiting order (bit k = bit k % 64 of word
        k // 64); a link outside every span, an unknown target or an empty
        range consumes no number, and numbering stops at the cap."""
        limit = self.max_grants if max_grants_cap is None else max_grants_cap
        first_span_of_doc: Dict[int, Any] = {}
        for sp in doc_spans:
            first_span_of_doc.setdefault(sp.doc_id, sp)
        out: List[Tuple[int, int, int, int, int]] = []
        pending = [(pos, tgt) for pos in sorted(link_to_target) for tgt in link_to_target[pos]]
        for pos, tgt in pending:
            if len(out) >= limit:
                logger.warning("grant budget of %d reached; the pack's remaining links get no grant",
                               limit)
                break
            holder = next((sp for sp in doc_spans if sp.start < pos <= sp.end), None)
            target = first_span_of_doc.get(tgt)
            if holder is None or target is None:
                continue
            q_rng = (pos, min(seq_len, holder.end))
            kv_rng = (max(0, target.start), min(seq_len, target.end))
            if q_rng[0] < q_rng[1] and kv_rng[0] < kv_rng[1]:
                out.append((len(out),) + q_rng + kv_rng)
        return out

    def _build_grant_bitmasks(self, seq_len: int, doc_spans, link_to_target,
                              max_grants_cap: Optional[int] = None, device=None):
        """Grant words of :210-300 built on the device: (q_bits, kv_bits int64
        [1, W, T], number of grants)."""
        grants = self._grant_ranges(seq_len, doc_spans, link_to_target, max_grants_cap)
        device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        _, qb, kb = token_inputs(seq_len, doc_spans, device, words=self._n_chunks, grants=grants)
        return qb, kb, len(grants)

    def __call__(self, tokens: torch.Tensor, doc_spans: List[Any], **kwargs) -> T2TBlockMask:
        device = _device_of(tokens)
        seq_len = tokens.shape[-1]
        links = self.link_detector.detect_links(tokens[0])
        link_to_target = self._match_links_to_docs(links, doc_spans)
        cap = self._current_max_grants()
        self._step += 1
        grants = self._grant_ranges(seq_len, doc_spans, link_to_target, max_grants_cap=cap)
        doc, qb, kb = token_inputs(seq_len, doc_spans, device, words=self._n_chunks, grants=grants)
        return _finish(doc, qb, kb, kwargs)


class SlidingWindowMaskCreator:
    """The masks of ``creator`` (a ``(tokens, doc_spans, **kw)`` creator of this
    module, or one that hands its keywords on to one) with a sliding window: a
    token reads of its own document the last ``window`` tokens, itself among
    them, and the first ``sinks`` ones; granted documents are read whole."""

    def __init__(self, creator, window: int, sinks: int = 0):
        if window is None:
            raise ValueError("a sliding window needs a number of tokens")
        self.creator = creator
        self.window, self.sinks = check_window(window, sinks)

    def __call__(self, tokens: torch.Tensor, doc_spans: List[Any], **kwargs):
        bm = self.creator(tokens, doc_spans, **{**kwargs, "window": self.window,
                                                "sinks": self.sinks})
        if (getattr(bm, "window", None), getattr(bm, "sinks", 0)) != (self.window, self.sinks):
            raise TypeError(f"{self.creator!r} does not take window= and sinks=")
        return bm


# Named creators; cross_doc_link is built from a link detector instead
# (CrossDocLinkMaskCreator, wrapped with make_mask_creator_callable_from).
MASK_CREATORS = dict(doc_causal=create_doc_causal_block_mask, causal=create_causal_block_mask)


def get_mask_creator(name: str):
    """The creator registered under ``name`` (ValueError for other names)."""
    try:
        return MASK_CREATORS[name]
    except KeyError:
        raise ValueError(f"no mask creator is registered as {name!r} "
                         f"(registered: {sorted(MASK_CREATORS)})") from None


def list_mask_creators() -> List[str]:
    return [*MASK_CREATORS]


class _BatchMaskCreator:
    """A ``(tokens, doc_spans, **kw)`` creator called with a batch dict, the
    interface of block_mask_creator.py:288-317: ``tokens`` is required,
    ``doc_spans`` defaults to no spans, every other key is passed through."""

    def __init__(self, creator):
        self.creator = creator

    @torch._dynamo.disable
    def __call__(self, **batch):
        if batch.get("tokens") is None:
            raise ValueError("the batch has no 'tokens' entry to build a mask for")
        rest = dict(batch)
        tokens = rest.pop("tokens")
        spans = rest.pop("doc_spans", [])
        return self.creator(tokens, spans, **rest)


def make_mask_creator_callable_from(creator):
    """(**batch) -> mask wrapper of any creator."""
    return _BatchMaskCreator(creator)


def make_mask_creator_callable(mask_type: str, window: Optional[int] = None, sinks: int = 0):
    """The named creator as a (**batch) -> mask callable, with a sliding window
    where one is given."""
    creator = get_mask_creator(mask_type)
    window, sinks = check_window(window, sinks)
    if window is not None:
        creator = SlidingWindowMaskCreator(creator, window, sinks)
    return _BatchMaskCreator(creator)
