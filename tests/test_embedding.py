"""Refusals and shapes of the scaled embedding that need no GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tagseq2tagseq_amd import _lib
from tagseq2tagseq_amd.embedding import ScaledEmbedding, embedding
from tagseq2tagseq_amd.modules import TS2TSTrainingModule

no_gpu = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="placeholder-pointer checks run on CPU-only hosts")
P = ctypes.c_void_p(0x1000)


def _err():
    return _lib.lib().t2t_last_error().decode()


def _forward(**kw):
    a = dict(tokens=P, N=4, w=P, ws=64, V=10, C=64, dtype=0, scale=1.0, out=P)
    a.update(kw)
    return _lib.lib().t2t_embedding(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(N=-1), -1, "N=-1"), (dict(V=0), -1, "V=0"), (dict(C=0), -1, "C=0"),
    (dict(dtype=2), -2, "dtype"), (dict(V=(1 << 20) + 1), -2, "one launch"),
    (dict(N=1 << 31), -2, "one launch"), (dict(C=(1 << 20) + 1, ws=1 << 21), -2, "one launch"), (dict(N=1 << 30, C=1 << 10), -2, "one launch"),
    (dict(tokens=None), -1, "tokens"), (dict(tokens=ctypes.c_void_p(0x1004)), -1, "tokens"),
    (dict(w=None), -1, "weight"), (dict(out=ctypes.c_void_p(0x1001)), -1, "misaligned"),
    (dict(ws=63), -1, "stride"),
])
def test_forward_entry_refuses(kw, rc, text):
    assert _forward(**kw) == rc and text in _err()


def _backward(**kw):
    a = dict(tokens=P, N=4, dy=P, ds=64, V=10, C=64, dtype=0, scale=1.0, pad=-1, dw=P, ws=P,
             bytes=1 << 20)
    a.update(kw)
    return _lib.lib().t2t_embedding_backward(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(pad=-2), -1, "padding"), (dict(pad=10), -1, "padding"), (dict(dw=None), -1, "dweight"),
    (dict(dy=None), -1, "dy"), (dict(dw=ctypes.c_void_p(0x1008)), -1, "16-byte"), (dict(ds=-1), -1, "stride"), (dict(ws=None), -1, "workspace"),
    (dict(bytes=16), -1, "workspace"), (dict(ws=ctypes.c_void_p(0x1008)), -1, "workspace"),
    (dict(V=1 << 21), -2, "one launch"),
])
def test_backward_entry_refuses(kw, rc, text):
    assert _backward(**kw) == rc and text in _err()



@no_gpu
@pytest.mark.parametrize("kw", [
    dict(N=1 << 26, C=2049), dict(N=1 << 26, C=2049, dtype=1),
    dict(N=1 << 26, C=2048, dy=ctypes.c_void_p(0x1002)),
    dict(N=(1 << 30) + 64, C=255),
])
def test_backward_entry_refuses_what_a_launch_does_not_number(kw):
    """A thread a column and piece of 32 positions: 2^32 of them and more, before
    the first launch."""
    assert _backward(ds=0, bytes=1 << 50, **kw) == -2 and "one launch" in _err()


@no_gpu
@pytest.mark.parametrize("kw", [
    dict(N=1 << 26, C=2048), dict(N=(1 << 26) - 32, C=2048, dy=ctypes.c_void_p(0x1002)),
    dict(N=1 << 30, C=127), dict(N=(1 << 31) - 4097, C=1),
    dict(N=1 << 28, C=1 << 10, dtype=1),
])
def test_backward_entry_takes_what_a_launch_numbers(kw):
    """(Refused for its workspace, which is checked behind the sizes.)"""
    assert _backward(ds=0, bytes=0, **kw) == -1 and "workspace" in _err()


def test_workspace_sizes():
    ws = _lib.lib().t2t_embedding_backward_workspace
    assert ws(-1, 5, 5) == ws(5, 0, 5) == ws(5, 5, 0) == ws(5, 1 << 21, 5) == 0
    assert 0 < ws(0, 5, 5) == ws(2048, 5, 5) < ws(2049, 5, 5) < ws(1 << 20, 50257, 768) < 1 << 30


def test_python_layer_refuses():
    w = torch.zeros(10, 8)
    t = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        embedding(t, w)
    for scale in (float("nan"), float("inf"), -1e39):
        with pytest.raises(ValueError, match="finite"):
            embedding(t, w, scale)
    for pad in (10, -11):
        with pytest.raises(ValueError, match="padding_idx"):
            embedding(t, w, padding_idx=pad)
    with pytest.raises(ValueError, match="weight"):
        embedding(t, w[0])


def test_shapes_of_the_traced_op():
    with FakeTensorMode():
        out = torch.ops.t2t.embedding(torch.zeros(2, 3, dtype=torch.int64), torch.zeros(9, 4), 2.0,
                                      -1)
        assert out.shape == (2, 3, 4)



def test_module_from_a_table():
    """nn.Embedding's constructor from a table, with the factor."""
    w = torch.randn(7, 4)
    m = ScaledEmbedding.from_pretrained(w, scale=3.0, padding_idx=-1)
    t = torch.tensor([[1, 6], [0, 2]])
    assert m.weight.data_ptr() == w.data_ptr() and not m.weight.requires_grad
    assert (m.num_embeddings, m.embedding_dim, m.padding_idx, m.scale) == (7, 4, 6, 3.0)
    assert torch.equal(m(t), w[t] * 3.0)
    free = ScaledEmbedding.from_pretrained(w, freeze=False)
    assert free.weight.requires_grad and free.scale == 1.0 and free.padding_idx is None
    with pytest.raises(ValueError, match="V, C"):
        ScaledEmbedding.from_pretrained(w[0])


def test_module_on_the_cpu_and_in_the_training_module():
    m = ScaledEmbedding(7, 4, scale=3.0)
    t = torch.tensor([[1, 6], [0, 2]])
    assert torch.equal(m(t), m.weight[t] * 3.0)
    assert set(m.state_dict()) == {"weight"}
    kw = dict(vocab_size=32, num_layers=1, model_dim=64, num_heads=1, max_seq_len=8, dropout=0.0,
              drop_path_rate=0.0, block_mask_creator=lambda **_: None)
    assert type(TS2TSTrainingModule.from_config(**kw).embedding) is torch.nn.Embedding
    scaled = TS2TSTrainingModule.from_config(embedding_scale=8.0, **kw)
    assert isinstance(scaled.embedding, ScaledEmbedding) and scaled.embedding.scale == 8.0
    assert scaled.loss_fn.weight is scaled.embedding.weight
