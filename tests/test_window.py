"""Refusals of the sliding-window calls that need no GPU: the C entries reject
bad arguments before any launch, the Python layer bad windows and CPU tensors."""
import ctypes

import pytest
import torch

from tagseq2tagseq_amd import _lib
from tagseq2tagseq_amd.block_mask import build_block_mask, check_window, doc_starts, mask_inputs
from tagseq2tagseq_amd.decode import attn_decode
from tagseq2tagseq_amd.mask_creators import (SlidingWindowMaskCreator, create_causal_block_mask,
                                             make_mask_creator_callable)

no_gpu = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="placeholder-pointer checks run on CPU-only hosts")
P = ctypes.c_void_p(0x1000)
L = _lib.lib()


def _err():
    return L.t2t_last_error().decode()


def _tables(T=256, Bm=1, slots=None):
    nt = -(-T // 128)
    m = _lib.T2TBlockMaskC(Bm, nt, *[0x1000] * 13, Bm * nt * (nt + 1) // 2 if slots is None else slots)
    return ctypes.byref(m)


def _meta(**kw):
    a = dict(doc=P, qb=None, kb=None, start=P, Bm=1, T=256, words=0, window=5, sinks=2, cls=P,
             out=_tables())
    a.update(kw)
    return L.t2t_mask_meta_window(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(window=0), -1, "window=0"), (dict(window=-1), -1, "window=-1"),
    (dict(sinks=-1), -1, "sinks=-1"), (dict(start=None), -1, "doc_start"),
    (dict(T=-1), -1, "negative"), (dict(Bm=-1), -1, "negative"), (dict(words=9), -2, "words"),
    (dict(words=1), -1, "NULL"), (dict(doc=None), -1, "NULL"), (dict(cls=None), -1, "NULL"),
    (dict(out=None), -1, "out is NULL"), (dict(Bm=2), -1, "describes"),
    (dict(out=_tables(slots=2)), -1, "slots"),
])
def test_metadata_entry_refuses(kw, rc, text):
    assert _meta(**kw) == rc and text in _err()


@no_gpu
def test_doc_starts_entry_refuses():
    assert L.t2t_doc_starts(P, -1, 5, P, None) == -1 and "negative" in _err()
    assert L.t2t_doc_starts(P, 1, -5, P, None) == -1 and "negative" in _err()
    assert L.t2t_doc_starts(None, 1, 5, P, None) == -1 and "NULL" in _err()
    assert L.t2t_doc_starts(P, 1, 5, None, None) == -1 and "NULL" in _err()
    assert L.t2t_doc_starts(P, 70000, 5, P, None) == -2 and "one launch" in _err()
    assert L.t2t_doc_starts(P, 1, 2 ** 31 - 1, P, None) == -2 and "one launch" in _err()
    assert L.t2t_doc_starts(None, 0, 5, None, None) == 0
    assert L.t2t_doc_starts(None, 1, 0, None, None) == 0


def _view(**kw):
    f = dict(data=0x1000, stride_b=0, stride_h=64, stride_t=64)
    f.update(kw)
    return ctypes.byref(_lib.T2TTensor(*f.values()))


def _decode(**kw):
    a = dict(q=_view(), k=_view(), v=_view(), o=_view(), lse2=P, key_doc=P, key_bits=None,
             key_stride=1000, q_pos=P, q_doc=P, q_bits=None, Bm=1, words=0, B=1, Hq=2, Hkv=2, Tq=1,
             Tkv=1000, D=64, dtype=0, scale=0.125, window=9, sinks=1, q_start=P, ws=P,
             ws_bytes=1 << 30)
    a.update(kw)
    return L.t2t_attn_decode_window(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(window=0), -1, "window=0"), (dict(sinks=-2), -1, "sinks=-2"),
    (dict(q_start=None), -1, "q_start"), (dict(Hq=9), -1, "multiple"),
    (dict(Tq=9), -2, "exceeds 8"), (dict(D=80), -2, "head dim"), (dict(dtype=1), -2, "bf16"),
    (dict(scale=0.0), -1, "scale"), (dict(key_stride=999), -1, "key_stride"),
    (dict(Bm=2), -1, "broadcast"), (dict(ws_bytes=4), -1, "workspace"),
    (dict(q_pos=None), -1, "NULL"), (dict(words=1), -1, "NULL"), (dict(k=_view(stride_t=60)), -1, "view"),
])
def test_decode_entry_refuses(kw, rc, text):
    assert _decode(**kw) == rc and text in _err()


@no_gpu
def test_nothing_to_do_is_no_error():
    assert _meta(T=0, window=0, doc=None) == 0
    assert _decode(Tq=0, window=0) == 0


def _backward(**kw):
    v = _view(stride_h=128, stride_t=128)
    a = dict(q=v, k=v, v=v, o=v, rest=v, do=v, lse2=P, delta=P, dq=v, dk=v, dv=v, B=1, Hq=2, Hkv=1, T=256,
             D=128, dtype=0, scale=0.1, mask=_tables(), ws=P, ws_bytes=1 << 40)
    a.update(kw)
    return L.t2t_attn_bwd_uneven(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(ws=None), -1, "workspace"), (dict(ws=ctypes.c_void_p(0x1008)), -1, "16-byte"),
    (dict(ws_bytes=1000), -1, "workspace"), (dict(D=96), -2, "head dim"), (dict(Hq=3, Hkv=2), -1, "GQA"),
    (dict(scale=-1.0), -1, "scale"), (dict(lse2=None), -1, "lse2"), (dict(mask=None), -1, "mask"),
    (dict(dk=None), -1, "view"), (dict(dtype=1), -2, "o_rest"),
    (dict(rest=_view(data=None)), -1, "view"),
])
def test_backward_entry_refuses(kw, rc, text):
    assert _backward(**kw) == rc and text in _err()


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(rest=None), -1, "o_rest"), (dict(dtype=1), -2, "not bf16"), (dict(lse2=None), -1, "lse2"),
    (dict(rest=_view(data=None)), -1, "view"), (dict(D=96), -2, "head dim"), (dict(mask=None), -1, "mask"),
])
def test_forward_entry_refuses(kw, rc, text):
    v = _view(stride_h=128, stride_t=128)
    a = dict(q=v, k=v, v=v, o=v, rest=v, lse2=P, B=1, Hq=2, Hkv=1, T=256, D=128, dtype=0,
             scale=0.1, mask=_tables())
    a.update(kw)
    assert L.t2t_attn_fwd_rest(*a.values(), None) == rc and text in _err()


def test_backward_workspace():
    w = L.t2t_attn_bwd_uneven_workspace
    piece = 2 * 128 * 128 * 4
    assert w(1, 1, 256, 128, 0) == 2 * 4 * piece          # two columns, four parts each
    assert w(2, 4, 4001, 128, 0) == 2 * 4 * 32 * 4 * piece
    assert w(1, 12, 16384, 128, 0) == 0                    # many columns: as t2t_attn_bwd
    assert w(1, 1, 256, 64, 0) == 0 and w(1, 1, 256, 128, 1) == 0
    assert w(0, 1, 256, 128, 0) == 0 and w(1, 1, 0, 128, 0) == 0 and w(-1, 1, 5, 128, 0) == 0
    for B, H, T in ((1, 512, 128), (512, 1, 100), (4, 4, 4096), (1, 2, 32768)):
        assert 0 < w(B, H, T, 128, 0) <= 256 << 20


@pytest.mark.parametrize("window,sinks,match", [
    (0, 0, "at least 1"), (-4, 0, "at least 1"), (1.5, 0, "at least 1"), (None, 2, "without"),
    (5, -1, "number of tokens"), (5, 0.5, "number of tokens"),
])
def test_bad_windows(window, sinks, match):
    with pytest.raises(ValueError, match=match):
        check_window(window, sinks)
    with pytest.raises(ValueError, match=match):
        mask_inputs(torch.zeros(4, dtype=torch.int32), window=window, sinks=sinks)
    with pytest.raises(ValueError, match=match):
        make_mask_creator_callable("causal", window=window, sinks=sinks)


def test_window_creators_need_a_window_and_a_gpu():
    with pytest.raises(ValueError, match="number of tokens"):
        SlidingWindowMaskCreator(create_causal_block_mask, None)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        SlidingWindowMaskCreator(create_causal_block_mask, 5)(torch.zeros(1, 4, dtype=torch.long), [])
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        build_block_mask(torch.zeros(4, dtype=torch.int32), window=3)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        doc_starts(torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU tensors"):
        mask_inputs(torch.zeros(4, dtype=torch.int32), window=3, sinks=1)
    t = mask_inputs(torch.zeros(4, dtype=torch.int32), window=3)  # (no device work)
    assert (t.window, t.sinks, t.doc_start) == (3, 0, None)
    k = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    one = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        attn_decode(k[:, :, :1], k, k, 4, one.repeat(1, 4), None, one, one, None, window=2)


def test_columns_are_shared_only_where_one_can_be_long():
    """A column has at most (Hq / Hkv) ceil(T / 128) items, a work-group takes 32."""
    w = L.t2t_attn_bwd_uneven_pieces
    assert w(4, 4, 4, 4096, 128, 0) == 1 and w(1, 8, 8, 100, 128, 0) == 1   # 32 items; 1
    assert w(4, 4, 4, 4097, 128, 0) == 1                                     # 528 columns
    assert w(1, 4, 4, 4097, 128, 0) == 2 and w(1, 8, 4, 2304, 128, 0) == 2   # 33; 36
    assert w(1, 8, 2, 2304, 128, 0) == 3 and w(2, 16, 4, 4001, 128, 0) == 4  # 72; 128
    assert w(1, 64, 1, 32768, 128, 0) == 4
    assert w(1, 64, 1, 32768, 64, 0) == 1 and w(1, 64, 1, 32768, 128, 1) == 1
    assert w(0, 1, 1, 9, 128, 0) == 1 and w(1, 0, 1, 9, 128, 0) == 1 and w(1, 1, 0, 9, 128, 0) == 1
    assert w(1, 1, 1, 2 ** 31 - 1, 128, 0) == 1 and w(1, 1, 1, -5, 128, 0) == 1


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(D=96), -2, "head dim"), (dict(Hq=3, Hkv=2), -1, "GQA"), (dict(scale=-1.0), -1, "scale"),
    (dict(lse2=None), -1, "lse2"), (dict(mask=None), -1, "mask"), (dict(dk=None), -1, "view"),
    (dict(dtype=1), -2, "o_rest"), (dict(rest=_view(data=None)), -1, "view"),
])
def test_backward_entry_without_a_workspace_refuses(kw, rc, text):
    v = _view(stride_h=128, stride_t=128)
    a = dict(q=v, k=v, v=v, o=v, rest=v, do=v, lse2=P, delta=P, dq=v, dk=v, dv=v, B=1, Hq=2, Hkv=1,
             T=256, D=128, dtype=0, scale=0.1, mask=_tables())
    a.update(kw)
    assert L.t2t_attn_bwd_rest(*a.values(), None) == rc and text in _err()
