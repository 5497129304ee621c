"""Refusals of the prologue with per-head norms that need no GPU: the C entries
reject bad arguments before any launch, the Python layer CPU tensors and bad
shapes."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch._subclasses.fake_tensor import FakeTensorMode

from tagseq2tagseq_amd import _lib
from tagseq2tagseq_amd.attention import FlexSelfAttention
from tagseq2tagseq_amd.rope import qk_norm_rope, qk_norm_rope_append

no_gpu = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="placeholder-pointer checks run on CPU-only hosts")
P = ctypes.c_void_p(0x1000)


def _err():
    return _lib.lib().t2t_last_error().decode()


def _view(**kw):
    f = dict(data=0x1000, stride_b=0, stride_h=64, stride_t=64)
    f.update(kw)
    return ctypes.byref(_lib.T2TTensor(*f.values()))


def _forward(**kw):
    a = dict(qkv=P, sb=0, st=256, B=1, T=4, Hq=2, Hkv=1, D=64, dtype=0, qw=P, kw=P, wdt=0,
             eps=1e-6, cos=P, sin=P, rows=16, pos0=0, q=_view(), k=_view(), v=_view())
    a.update(kw)
    return _lib.lib().t2t_qk_norm_rope(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(B=-1), -1, "B=-1"), (dict(Hq=0), -1, "Hq=0"), (dict(Hkv=0), -1, "Hkv=0"),
    (dict(D=24), -2, "head dim"), (dict(D=528), -2, "head dim"), (dict(D=0), -2, "head dim"),
    (dict(dtype=2), -2, "dtype"), (dict(wdt=7), -2, "dtype"),
    (dict(eps=-1e-6), -1, "eps"), (dict(eps=float("nan")), -1, "eps"),
    (dict(eps=float("inf")), -1, "eps"),
    (dict(B=1 << 20, T=1 << 20), -2, "more tokens"),
    (dict(B=2, T=1 << 30, rows=2 ** 31 - 1), -2, "more tokens"),
    (dict(Hq=1 << 20, st=1 << 30), -2, "more tokens or heads"),
    (dict(qw=None), -1, "norm weights"), (dict(kw=ctypes.c_void_p(0x1008)), -1, "norm weights"),
    (dict(qkv=None), -1, "16-byte"), (dict(qkv=ctypes.c_void_p(0x1008)), -1, "16-byte"),
    (dict(st=257), -1, "16-byte"), (dict(sb=-8), -1, "16-byte"),
    (dict(cos=None), -1, "cos"), (dict(sin=ctypes.c_void_p(0x1004)), -1, "cos"),
    (dict(rows=3), -1, "exceed"), (dict(pos0=-1), -1, "positions"), (dict(pos0=13), -1, "exceed"),
    (dict(q=None), -1, "view"), (dict(k=_view(stride_t=60)), -1, "view"),
    (dict(v=_view(data=0)), -1, "view"),
])
def test_forward_entry_refuses(kw, rc, text):
    assert _forward(**kw) == rc and text in _err()


@no_gpu
def test_nothing_to_do_is_no_error():
    assert _forward(T=0, qkv=None, q=None) == 0
    assert _forward(B=0, cos=None) == 0


def _append(**kw):
    a = dict(qkv=P, sb=0, st=256, B=1, M=4, Hq=2, Hkv=1, D=64, dtype=0, qw=P, kw=P, wdt=0,
             eps=1e-6, cos=P, sin=P, rows=16, pos=None, pos_sb=0, pos0=0, q=_view(), k=_view(),
             v=_view(data=0x2000), cache=16)
    a.update(kw)
    return _lib.lib().t2t_qk_norm_rope_append(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(pos=P, M=9), -2, "at most 8"), (dict(pos=ctypes.c_void_p(0x1004)), -1, "misaligned"),
    (dict(pos=P, pos_sb=-4), -1, "stride"), (dict(pos0=-1), -1, "positions"),
    (dict(pos0=13), -1, "exceed"), (dict(cache=3), -1, "exceed"), (dict(cache=-1), -1, "cache"),
    (dict(k=_view(stride_t=0)), -1, "overlap"), (dict(B=2), -1, "overlap"),
    (dict(v=_view()), -1, "are one"),
    (dict(Hkv=2, k=_view(stride_h=0)), -1, "overlap"), (dict(D=20), -2, "head dim"),
])
def test_append_entry_refuses(kw, rc, text):
    assert _append(**kw) == rc and text in _err()


def _backward(**kw):
    a = dict(dq=_view(), dk=_view(), dv=_view(), qkv=P, sb=0, st=256, B=1, T=4, Hq=2, Hkv=1, D=64,
             dtype=0, qw=P, kw=P, wdt=0, eps=1e-6, cos=P, sin=P, rows=16, pos0=0, dqkv=P, dqw=P,
             dkw=P, ws=P, bytes=1 << 20)
    a.update(kw)
    return _lib.lib().t2t_qk_norm_rope_backward(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(dq=None), -1, "view"), (dict(dqkv=None), -1, "dqkv"),
    (dict(dqkv=ctypes.c_void_p(0x1008)), -1, "dqkv"), (dict(dqw=None), -1, "weight"),
    (dict(ws=None), -1, "workspace"), (dict(bytes=4), -1, "workspace"),
    (dict(pos0=15), -1, "exceed"), (dict(D=8), -2, "head dim"),
])
def test_backward_entry_refuses(kw, rc, text):
    assert _backward(**kw) == rc and text in _err()


def test_workspace_sizes():
    ws = _lib.lib().t2t_qk_norm_rope_backward_workspace
    assert ws(0, 5, 2, 2, 64) == ws(1, 5, 2, 2, 20) == ws(1, 5, 0, 2, 64) == 0
    assert ws(1, 1, 1, 1, 64) == 2 * 64 * 4
    assert 0 < ws(8, 1 << 20, 16, 16, 128) <= 1024 * 128 * 4  # bounded


def _cpu(H=2, Hkv=2, D=64, dt=torch.bfloat16, T=3):
    return (torch.zeros(1, T, (H + 2 * Hkv) * D, dtype=dt), torch.ones(D), torch.ones(D),
            torch.zeros(8, D // 2), torch.zeros(8, D // 2))


def test_python_layer_refuses():
    a = _cpu()
    with pytest.raises(RuntimeError, match="GPU"):
        qk_norm_rope(*a, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        qk_norm_rope_append(*a, 2, 0, torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16),
                            torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError, match="dtype"):
        qk_norm_rope(a[0].half(), *a[1:], 2)
    for heads, kv in ((0, 1), (1, 0), (-1, 2), (5, 5), (2 ** 62, 2 ** 62)):
        with pytest.raises(ValueError, match="num_heads|head_dim"):
            qk_norm_rope(*a, heads, num_kv_heads=kv)
    with pytest.raises(ValueError, match="qkv must be"):
        qk_norm_rope(a[0][0], *a[1:], 2)
    with pytest.raises(ValueError, match="weight"):
        qk_norm_rope(a[0], torch.ones(32), *a[2:], 2)
    with pytest.raises(ValueError, match="cos"):
        qk_norm_rope(*a[:3], a[3][:, :16], a[4][:, :16], 2)
    with pytest.raises(ValueError, match="cos"):
        qk_norm_rope(*a[:3], a[3].double(), a[4].double(), 2)
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rope(*a, 2, eps=-1.0)
    for i in (3, 4):
        b = list(a)
        b[i] = b[i].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="tables get no gradient"):
            qk_norm_rope(*b, 2)
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
            qk_norm_rope(*b, 2)
    caches = [torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16) for _ in range(2)]
    for i in range(5):
        b = list(a)
        b[i] = b[i].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="append has no gradient"):
            qk_norm_rope_append(*b, 2, 0, *caches)
    with fwad.dual_level(), pytest.raises(RuntimeError, match="append has no gradient"):
        qk_norm_rope_append(fwad.make_dual(a[0], a[0].clone()), *a[1:], 2, 0, *caches)
    with pytest.raises(ValueError, match="caches"):
        qk_norm_rope_append(*a, 2, 0, torch.zeros(1, 2, 8, 64), torch.zeros(1, 2, 9, 64))


def test_shapes_of_the_traced_op():
    with FakeTensorMode():
        a = _cpu(H=4, Hkv=2, D=32, T=7)
        q, k, v = torch.ops.t2t.qk_norm_rope(*a, 4, 2, 0, 1e-6)
        assert q.shape == (1, 4, 7, 32) and k.shape == v.shape == (1, 2, 7, 32)
        cache = torch.zeros(1, 2, 8, 32, dtype=torch.bfloat16)
        q = torch.ops.t2t.qk_norm_rope_append(*a, 4, None, 1, cache, cache.clone(), 1e-6)
        assert q.shape == (1, 4, 7, 32)


def test_module_parameters():
    plain = FlexSelfAttention(128, 2, 16)
    normed = FlexSelfAttention(128, 2, 16, qk_norm=True)
    extra = set(normed.state_dict()) - set(plain.state_dict())
    assert extra == {"q_norm", "k_norm"} and set(plain.state_dict()) == {"qkv.weight",
                                                                         "proj.weight"}
    assert normed.q_norm.shape == normed.k_norm.shape == (64,)
