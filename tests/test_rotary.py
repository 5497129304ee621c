"""The prologue with any rotary form where no GPU is needed: refusals of the C
entries and of the Python layer, the tables' scalings, and the modules' forms."""
import ctypes
import inspect
import math

import pytest
import torch

from tagseq2tagseq_amd import _lib
from tagseq2tagseq_amd.attention import FlexSelfAttention
from tagseq2tagseq_amd.rope import RotaryForm, qkv_rotary, rope_tables, rotary_tables

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
    a = dict(qkv=P, sb=0, st=256, B=1, T=4, Hq=2, Hkv=1, D=64, R=32, inter=0, dtype=0, cos=P,
             sin=P, rows=16, pos=None, pos_sb=0, pos0=0, q=_view(), k=_view(), v=_view())
    a.update(kw)
    return _lib.lib().t2t_qkv_rotary(*a.values(), None)


def _backward(**kw):
    a = dict(q=_view(), k=_view(), v=_view(), dqkv=P, sb=0, st=256, B=1, T=4, Hq=2, Hkv=1, D=64,
             R=32, inter=0, dtype=0, cos=P, sin=P, rows=16, pos=None, pos_sb=0, pos0=0)
    a.update(kw)
    return _lib.lib().t2t_qkv_rotary_backward(*a.values(), None)


BAD = [
    (dict(B=-1), -1, "B=-1"), (dict(T=-1), -1, "T=-1"), (dict(Hq=0), -1, "Hq=0"),
    (dict(Hkv=0), -1, "Hkv=0"),
    (dict(D=24), -2, "head dim"), (dict(D=528), -2, "head dim"), (dict(D=0), -2, "head dim"),
    (dict(R=0), -2, "rotated"), (dict(R=24), -2, "rotated"), (dict(R=80), -2, "rotated"),
    (dict(R=-16), -2, "rotated"), (dict(dtype=2), -2, "dtype"),
    (dict(B=1 << 20, T=1 << 20), -2, "more tokens"), (dict(Hq=1 << 20), -2, "more tokens or heads"),
    (dict(rows=-1), -1, "table_rows"), (dict(rows=3), -1, "exceed"), (dict(pos0=-1), -1, "exceed"),
    (dict(pos0=13), -1, "exceed"), (dict(pos=ctypes.c_void_p(0x1004)), -1, "pos misaligned"),
    (dict(pos=P, pos_sb=-4), -1, "negative stride"),
    (dict(st=257), -1, "16-byte"), (dict(sb=-8), -1, "16-byte"),
    (dict(cos=None), -1, "cos"), (dict(sin=ctypes.c_void_p(0x1004)), -1, "cos"),
    (dict(q=None), -1, "view"), (dict(k=_view(stride_t=60)), -1, "view"),
    (dict(v=_view(data=0)), -1, "view"),
]


@no_gpu
@pytest.mark.parametrize("kw,rc,text", BAD + [
    (dict(qkv=None), -1, "16-byte"), (dict(qkv=ctypes.c_void_p(0x1008)), -1, "16-byte"),
    (dict(q=_view(stride_h=0)), -1, "overlap"), (dict(k=_view(stride_t=0)), -1, "overlap"),
    (dict(B=2), -1, "overlap"),
])
def test_forward_entry_refuses(kw, rc, text):
    assert _forward(**kw) == rc and text in _err()


@no_gpu
@pytest.mark.parametrize("kw,rc,text", BAD + [
    (dict(dqkv=None), -1, "16-byte"), (dict(dqkv=ctypes.c_void_p(0x1008)), -1, "16-byte"),
    (dict(st=0), -1, "overlap"), (dict(B=2), -1, "overlap"),
])
def test_backward_entry_refuses(kw, rc, text):
    assert _backward(**kw) == rc and text in _err()


@no_gpu
def test_nothing_to_do_is_no_error():
    assert _forward(T=0, qkv=None, q=None) == 0
    assert _backward(B=0, cos=None) == 0


@pytest.mark.parametrize("change,error,match", [
    (dict(), RuntimeError, "ROCm GPU tensors"),
    (dict(qkv=torch.zeros(4, 256)), ValueError, r"must be \[B, T"),
    (dict(heads=0), ValueError, "positive"), (dict(kv=-1), ValueError, "positive"),
    (dict(heads=3), ValueError, "last dim"), (dict(heads=2 ** 62), ValueError, "last dim"),
    (dict(qkv=torch.zeros(1, 4, 256, dtype=torch.float16)), NotImplementedError, "dtype Half"),
    (dict(cos=torch.zeros(8, 33)), ValueError, "must be float32"),
    (dict(cos=torch.zeros(8, 40), sin=torch.zeros(8, 40)), ValueError, "head_dim=64"),
    (dict(cos=torch.zeros(8, 0), sin=torch.zeros(8, 0)), ValueError, "must be float32"),
    (dict(sin=torch.zeros(8, 32, dtype=torch.bfloat16)), ValueError, "must be float32"),
])
def test_python_layer_refuses(change, error, match):
    a = dict(qkv=torch.zeros(1, 4, 256), cos=torch.zeros(8, 32), sin=torch.zeros(8, 32), heads=2,
             kv=1)
    a.update(change)
    with pytest.raises(error, match=match):
        qkv_rotary(*a.values())


def test_tables_get_no_gradient():
    c = torch.zeros(8, 32, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        qkv_rotary(torch.zeros(1, 4, 256), c, c.detach(), 2, 1)


def test_unscaled_tables():
    cos, sin = rotary_tables(64, 40, "cpu")
    want = rope_tables(64, 40, "cpu")
    # rope_tables rounds inverse frequencies and angles to float32: 40 * 2^-23
    assert torch.allclose(cos, want[0], atol=5e-6) and torch.allclose(sin, want[1], atol=5e-6)


def test_far_positions_keep_their_angle():
    """The angle is rounded after sine and cosine, not before."""
    rows = 300001
    cos, sin = rotary_tables(16, rows, "cpu")
    for p in (131071, 300000):
        for i in (0, 3, 7):
            ang = p * 10000.0 ** (-2 * i / 16)
            # float64 angles of up to 3e5: 3e5 * 2^-52, then the float32 rounding
            assert abs(float(cos[p, i]) - math.cos(ang)) < 2 ** -24 + 1e-9
            assert abs(float(sin[p, i]) - math.sin(ang)) < 2 ** -24 + 1e-9


def _angles(dim, p, **kw):
    cos, sin = rotary_tables(dim, p + 1, "cpu", magnitude=1.0, **kw)
    return torch.atan2(sin[p].double(), cos[p].double())


def test_scalings():
    plain = _angles(64, 1)
    assert torch.allclose(_angles(64, 1, scaling="linear", factor=4.0), plain / 4, atol=1e-6)
    by_base = _angles(64, 1, scaling="base", factor=4.0)
    assert abs(by_base[0] - plain[0]) < 1e-6
    assert abs(by_base[-1] - plain[-1] / 4) < 1e-6 * 4
    parts = _angles(64, 1, scaling="by_parts", factor=4.0, original_len=2048)
    turns = 2048 * plain / (2 * math.pi)
    assert torch.allclose(parts[turns > 32], plain[turns > 32], atol=1e-6)
    assert torch.allclose(parts[turns < 1], plain[turns < 1] / 4, atol=1e-6)
    mid = (turns > 1) & (turns < 32)
    keep = (turns[mid] - 1) / 31
    assert int(mid.sum()) > 4
    assert torch.allclose(parts[mid], plain[mid] * (keep + (1 - keep) / 4), atol=1e-6)
    cos, sin = rotary_tables(64, 9, "cpu", scaling="by_parts", factor=4.0, original_len=2048)
    size = 1 + 0.1 * math.log(4.0)
    assert torch.allclose(cos * cos + sin * sin, torch.full_like(cos, size * size), atol=1e-6)


@pytest.mark.parametrize("kw,match", [
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"),
    (dict(rows=-1), "rows"), (dict(base=0.0), "base"), (dict(base=float("inf")), "base"),
    (dict(factor=2.0), "needs a scaling"), (dict(scaling="cubic"), "none of"),
    (dict(scaling="linear", factor=0.5), "factor"),
    (dict(scaling="linear", factor=float("nan")), "factor"),
    (dict(scaling="base", factor=2.0, rotary_dim=2), "4 or more"),
    (dict(scaling="by_parts", factor=2.0), "original_len"),
    (dict(scaling="by_parts", factor=2.0, original_len=9, fast=1.0), "fast"),
    (dict(magnitude=float("nan")), "magnitude"),
])
def test_tables_refuse(kw, match):
    a = dict(rotary_dim=64, rows=4, device="cpu")
    a.update(kw)
    with pytest.raises(ValueError, match=match):
        rotary_tables(**a)


def test_module_forms():
    for fraction in (0.0, 0.1, 1.5, 0.3):
        with pytest.raises(ValueError, match="fraction"):
            FlexSelfAttention(128, 2, 32, rotary=RotaryForm(fraction=fraction))
    with pytest.raises(ValueError, match="whole heads"):
        FlexSelfAttention(128, 2, 32, qk_norm=True, rotary=RotaryForm(interleaved=True))
    FlexSelfAttention(128, 2, 32, qk_norm=True, rotary=RotaryForm(scaling="linear", factor=2.0))
    part = FlexSelfAttention(128, 2, 32, rotary=RotaryForm(fraction=0.5, interleaved=True))
    assert not part.rotary.whole_halves and part.rotary.tables("cpu")[0].shape == (32, 16)
    plain = FlexSelfAttention(128, 2, 32)
    assert plain.rotary.whole_halves and plain.rotary.form is None


@pytest.mark.parametrize("change", [dict(pos=1.0), dict(num_heads=2.0), dict(num_kv_heads=1.5)])
def test_numbers_that_are_not_whole_are_refused(change):
    cs = torch.zeros(8, 16)
    with pytest.raises(TypeError):
        qkv_rotary(torch.zeros(1, 4, 192), cs, cs, **{"num_heads": 1, **change})


# every test its own row count: the tables are kept by their arguments
def _made_under(mode, rows):
    with mode:
        first = [*rope_tables(32, rows, "cpu"), *rotary_tables(32, rows, "cpu")]
    return first, [*rope_tables(32, rows, "cpu"), *rotary_tables(32, rows, "cpu")]


def test_tables_made_in_inference_mode_serve_training():
    for t in _made_under(torch.inference_mode(), 101)[1]:
        assert not t.is_inference()
        x = torch.ones(101, 16, requires_grad=True)
        (x * t).sum().backward()  # (saves the table)
        assert torch.equal(x.grad, t)


def test_tables_of_fake_tensors_are_not_kept():
    from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
    first, later = _made_under(FakeTensorMode(), 102)
    assert all(isinstance(t, FakeTensor) for t in first)
    assert all(type(t) is torch.Tensor for t in later)


def test_tables_of_a_function_transform_are_not_kept():
    def f(x):
        cos, sin = rotary_tables(32, 103, "cpu")
        c2, s2 = rope_tables(32, 103, "cpu")
        return (x * (cos + sin + c2 + s2)).sum()
    torch.func.grad(f)(torch.ones(103, 16))
    for t in (*rope_tables(32, 103, "cpu"), *rotary_tables(32, 103, "cpu")):
        assert t.data_ptr() != 0 and float(t[0].abs().max()) in (0.0, 1.0)


@pytest.mark.parametrize("tables", [rope_tables, rotary_tables])
@pytest.mark.parametrize("inference", [False, True])
def test_tables_made_while_compiling(tables, inference):
    rows = 104 + inference

    @torch.compile(backend="eager", fullgraph=True)
    def f(x):
        cos, sin = tables(32, rows, x.device)
        return x * cos + sin
    x = torch.ones(rows, 16)
    with torch.inference_mode(inference):
        got = f(x)
    cos, sin = tables(32, rows, "cpu")
    assert torch.equal(got, cos + sin) and not cos.is_inference()
    assert tables(32, rows, "cpu")[0] is cos


@pytest.mark.parametrize("tables", [rope_tables, rotary_tables])
def test_a_device_without_an_index_is_the_current_one(tables, monkeypatch):
    """Kept by the device that the call means, not by its name."""
    from tagseq2tagseq_amd import rope
    now = [0]
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    keys = []
    monkeypatch.setattr(rope, "_tables", lambda key, make: keys.append(key))
    tables(32, 106, "cuda")
    now[0] = 1
    tables(32, 106, "cuda")
    tables(32, 106, torch.device("cuda", 1))
    tables(32, 106, "cuda:0")
    assert keys[0] != keys[1] == keys[2] and keys[0] == keys[3]


def test_the_tables_turn_either_way():
    """A pair (a, b) becomes (a cos + b sin, b cos - a sin) of the tables: by the
    negative angle, or with positive=True by the published rotation's."""
    for kw in (dict(), dict(scaling="by_parts", factor=4.0, original_len=16)):
        cos, sin = rotary_tables(32, 40, "cpu", **kw)
        c2, s2 = rotary_tables(32, 40, "cpu", positive=True, **kw)
        assert torch.equal(c2, cos) and torch.equal(s2, -sin)
    form = RotaryForm(fraction=0.5, interleaved=True, base=500.0, positive=True)
    cos, sin = form.tables(64, 9, "cpu")
    want = rotary_tables(32, 9, "cpu", base=500.0, positive=True)
    assert torch.equal(cos, want[0]) and torch.equal(sin, want[1])
    i = torch.arange(16, dtype=torch.float64)
    ang = torch.outer(torch.arange(9, dtype=torch.float64), 500.0 ** (-i / 16))
    # published: (a cos - b sin, a sin + b cos), here with s = -sin
    assert torch.allclose(sin.double(), -ang.sin(), atol=2 ** -24)


def test_a_form_hands_on_every_argument_of_the_tables():
    kw = dict(scaling="by_parts", factor=4.0, original_len=64, fast=8.0, slow=2.0, magnitude=1.5,
              base=300.0, positive=True)
    for a, b in zip(RotaryForm(**kw).tables(64, 50, "cpu"), rotary_tables(64, 50, "cpu", **kw)):
        assert torch.equal(a, b)
    names = set(RotaryForm.__dataclass_fields__) - {"fraction", "interleaved"}
    assert names == set(kw) == set(inspect.signature(rotary_tables).parameters) - {
        "rotary_dim", "rows", "device"}
