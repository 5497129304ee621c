"""Refusals of the 8-bit key/value cache that need no GPU: the C entries reject
bad arguments before any launch, the Python layer CPU tensors."""
import ctypes

import pytest
import torch

from tagseq2tagseq_amd import _lib
from tagseq2tagseq_amd.kv8 import KV8Cache, attn_decode_kv8, kv8_append

no_gpu = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="placeholder-pointer checks run on CPU-only hosts")
P = ctypes.c_void_p(0x1000)
V = ctypes.c_void_p(0x2000)
ODD = ctypes.c_void_p(0x1008)
L = _lib.lib()


def _err():
    return L.t2t_last_error().decode()


def _view(**kw):
    f = dict(data=0x1000, stride_b=0, stride_h=64, stride_t=64)
    f.update(kw)
    return ctypes.byref(_lib.T2TTensor(*f.values()))


def _append(**kw):
    a = dict(k=_view(), v=_view(), B=1, Hkv=2, M=3, D=64, dtype=0, pos=None, pos_stride=0, pos0=0,
             kc=P, vc=V, ks=P, vs=V, blocks=2, capacity=100)
    a.update(kw)
    return L.t2t_kv8_append(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(B=-1), -1, "negative"), (dict(M=-1), -1, "negative"), (dict(blocks=-1), -1, "negative"),
    (dict(D=32), -2, "head dim"), (dict(dtype=2), -2, "dtype"), (dict(B=70000), -2, "one launch"),
    (dict(Hkv=70000), -2, "one launch"), (dict(capacity=129), -1, "exceeds the 2 blocks"),
    (dict(capacity=2 ** 31 - 1, blocks=2 ** 40), -1, "exceeds"),
    (dict(pos0=-1), -1, "positions"), (dict(pos0=98), -1, "positions"),
    (dict(M=101), -1, "positions"), (dict(pos0=2 ** 62), -1, "positions"),
    (dict(pos=P, M=101), -1, "exceed capacity"), (dict(pos=ctypes.c_void_p(0x1004)), -1, "misaligned"),
    (dict(pos=P, pos_stride=-1), -1, "negative stride"),
    (dict(k=None), -1, "view"), (dict(v=_view(stride_t=60)), -1, "view"),
    (dict(k=_view(data=0)), -1, "view"), (dict(kc=None), -1, "codes"), (dict(vc=ODD), -1, "codes"),
    (dict(vc=P), -1, "are one"), (dict(ks=None), -1, "scales"), (dict(vs=P), -1, "are one"),
])
def test_append_entry_refuses(kw, rc, text):
    assert _append(**kw) == rc and text in _err()


def _attend(**kw):
    a = dict(q=_view(), kc=P, vc=V, ks=P, vs=V, blocks=20, o=_view(), lse2=P, key_doc=P,
             key_bits=None, key_stride=1280, q_pos=P, q_doc=P, q_bits=None, Bm=1, words=0, B=1, Hq=4,
             Hkv=2, Tq=1, Tkv=1280, D=64, dtype=0, scale=0.125, window=0, sinks=0, q_start=None,
             ws=P, ws_bytes=1 << 30)
    a.update(kw)
    return L.t2t_kv8_attend(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(B=-1), -1, "negative"), (dict(Tkv=-1), -1, "negative"), (dict(blocks=-1), -1, "negative"),
    (dict(dtype=1), -2, "bf16"), (dict(D=80), -2, "head dim"), (dict(words=9), -2, "words"),
    (dict(scale=0.0), -1, "scale"), (dict(scale=float("nan")), -1, "scale"),
    (dict(window=-1), -1, "window=-1"), (dict(sinks=1), -1, "without a window"),
    (dict(window=5, sinks=1), -1, "q_start"), (dict(window=5, sinks=-1), -1, "sinks=-1"),
    (dict(Hq=3), -1, "multiple"), (dict(Hkv=0), -1, "multiple"), (dict(Tq=9), -2, "exceeds 16"),
    (dict(Bm=3), -1, "broadcast"), (dict(key_stride=1279), -1, "key_stride"),
    (dict(blocks=19), -1, "blocks"), (dict(q=None), -1, "view"), (dict(o=_view(stride_t=4)), -1, "view"),
    (dict(kc=ODD), -1, "codes"), (dict(vc=P), -1, "are one"), (dict(lse2=None), -1, "NULL"),
    (dict(key_doc=None), -1, "NULL"), (dict(words=1), -1, "NULL"),
    (dict(ws=None), -1, "workspace"), (dict(ws_bytes=8), -1, "workspace"),
    (dict(ws=ODD), -1, "16-byte"),
    (dict(B=70000, Bm=1), -2, "one launch"),
])
def test_attend_entry_refuses(kw, rc, text):
    assert _attend(**kw) == rc and text in _err()


@no_gpu
def test_nothing_to_do_is_no_error():
    assert _append(M=0, k=None) == 0 and _append(B=0, kc=None) == 0
    assert _append(M=0, pos0=100, k=None) == 0
    assert _attend(Tq=0, q=None) == 0 and _attend(B=0, lse2=None) == 0


def test_workspace():
    w = L.t2t_kv8_attend_workspace
    assert w(1, 12, 12, 1, 1024, 64) == 0 and w(1, 8, 8, 1, 512, 128) == 0     # one pass
    assert w(1, 12, 12, 1, 1025, 64) == 12 * 5 * 66 * 4                        # five chunks
    assert w(1, 12, 12, 1, 32768, 64) == 12 * 64 * 66 * 4                      # at most 64
    assert w(2048, 8, 8, 1, 32768, 64) == 0                                    # enough rows
    assert w(0, 1, 1, 1, 9, 64) == 0 and w(1, 1, 0, 1, 9, 64) == 0 and w(1, 1, 1, 1, -1, 64) == 0


def test_python_layer_refuses_host_memory():
    cache = KV8Cache(1, 2, 100, 64, "cpu")
    assert [tuple(t.shape) for t in cache.buffers()] == [(1, 2, 2, 64, 64)] * 2 + [(1, 2, 2)] * 2
    k = torch.zeros(1, 2, 3, 64)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        cache.append(k, k, 0)
    one = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        cache.attend(k[:, :, :1].bfloat16(), 1, one, None, one, one, None)
    ks, vs = cache.values(torch.float32)
    assert ks.shape == vs.shape == (1, 2, 100, 64) and not ks.any()


@pytest.mark.parametrize("args", [(-1, 1, 8, 64), (1, 0, 8, 64), (1, 1, 0, 64), (1, 1, 8, 96)])
def test_no_cache_of_such_sizes(args):
    with pytest.raises(ValueError, match="no cache"):
        KV8Cache(*args, "cpu")


def test_positions_that_are_no_whole_numbers_are_refused():
    none = torch.zeros(1)
    with pytest.raises(TypeError):
        kv8_append(none, none, 3.0, none, none, none, none)
    with pytest.raises(TypeError):
        kv8_append(none, none, 3, none, none, none, none, capacity=64.5)
    with pytest.raises(TypeError):
        attn_decode_kv8(none, none, none, none, none, 2.5, none, None, none, none, None)
