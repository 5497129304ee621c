"""Refusals and shapes of the distillation loss that need no GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from tagseq2tagseq_amd import _lib
from tagseq2tagseq_amd.distill import LinearDistillLoss, distill_loss, head_distill
from tagseq2tagseq_amd.modules import LinearCELoss, TS2TSTrainingModule

no_gpu = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="placeholder-pointer checks run on CPU-only hosts")
P, P8 = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1001)


def _err():
    return _lib.lib().t2t_last_error().decode()


def _rows(**kw):
    a = dict(z=P, ld=100, rows=4, V=100, dt=0, idx=P, ib=8, ildx=5, t=P, tdt=1, tld=5, K=5,
             target=P, ignore=-100, temp=2.0, alpha=0.5, scale=1.0, sd=None, g=None, gs=0,
             unless=0, loss=P, grad=P, gld=100)
    a.update(kw)
    return _lib.lib().t2t_distill_rows(*a.values(), None)


@no_gpu
@pytest.mark.parametrize("kw,rc,text", [
    (dict(rows=-1), -1, "rows=-1"), (dict(V=0), -1, "V=0"), (dict(K=-1), -1, "K=-1"),
    (dict(K=1025), -2, "at most 1024"), (dict(V=(1 << 28) + 1, ld=1 << 29, gld=1 << 29), -2, "2^28"), (dict(dt=2), -2, "dtype"), (dict(tdt=3), -2, "dtype"),
    (dict(ib=2), -2, "indices"), (dict(temp=0.0), -1, "temperature"),
    (dict(temp=-1.0), -1, "temperature"), (dict(temp=float("nan")), -1, "temperature"),
    (dict(temp=100.5), -1, "temperature"), (dict(alpha=-0.1), -1, "alpha"),
    (dict(alpha=1.1), -1, "alpha"), (dict(alpha=float("nan")), -1, "alpha"),
    (dict(target=None), -1, "targets"), (dict(ld=99), -1, "stride"),
    (dict(gld=99), -1, "stride"), (dict(unless=1), -1, "unless_one"),
    (dict(unless=1, g=P, gs=1), -1, "unless_one"), (dict(rows=1 << 31), -2, "one launch"),
    (dict(z=None), -1, "logits"), (dict(z=P8), -1, "off its type"),
    (dict(grad=P8), -1, "off its type"), (dict(loss=None, grad=None), -1, "nothing to write"),
    (dict(grad=P, gld=101), -1, "over the logits"), (dict(idx=None), -1, "idx"),
    (dict(t=P8), -1, "misaligned"), (dict(ildx=-1), -1, "stride"),
])
def test_rows_entry_refuses(kw, rc, text):
    assert _rows(**kw) == rc and text in _err()


@no_gpu
def test_count_and_mean_entries_refuse():
    lib = _lib.lib()
    assert lib.t2t_distill_count(None, 3, -100, P, None) == -1 and "NULL" in _err()
    assert lib.t2t_distill_count(P, -1, -100, P, None) == -1
    assert lib.t2t_distill_mean(None, 3, None, 1.0, P, None) == -1
    assert lib.t2t_distill_mean(P, 3, None, 1.0, None, None) == -1
    assert _rows(rows=0, z=None, idx=None) == 0


def _cpu():
    return (torch.zeros(3, 10), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2),
            torch.zeros(3, dtype=torch.int64))


def test_python_layer_refuses():
    z, idx, t, target = _cpu()
    with pytest.raises(RuntimeError, match="GPU"):
        distill_loss(z, idx, t, target)
    with pytest.raises(ValueError, match="reduction"):
        distill_loss(z, idx, t, target, reduction="batchmean")
    for temp in (0.0, -1.0, 0.009, 101.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            distill_loss(z, idx, t, target, temperature=temp)
    for alpha in (-0.5, 1.5, float("nan")):
        with pytest.raises(ValueError, match="alpha"):
            distill_loss(z, idx, t, target, alpha=alpha)
    with pytest.raises(ValueError, match="targets"):
        distill_loss(z, idx, t, alpha=0.5)
    for bad in (idx[:2], idx[:, :1], idx.view(1, 3, 2)):
        with pytest.raises(ValueError, match="teacher_idx"):
            distill_loss(z, bad, t, target)
    for k in (1025, 1 << 32):  # (also where 32 bits hold none of it)
        with pytest.raises(NotImplementedError, match="at most 1024"):
            distill_loss(z, idx[:, :1].expand(3, k), t[:, :1].expand(3, k), target)
    with pytest.raises(ValueError, match="teacher_idx must"):
        distill_loss(z, idx.float(), t, target)
    with pytest.raises(NotImplementedError, match="dtype"):
        distill_loss(z, idx, t.double(), target)
    with pytest.raises(RuntimeError, match="detach"):
        distill_loss(z, idx, t.clone().requires_grad_(True), target)
    with pytest.raises(RuntimeError, match="bf16 rows"):
        head_distill(z, z, idx, t)
    # (rows that the chunks would not reach)
    m = LinearDistillLoss(4, 10)
    x = torch.zeros(2, 4)
    for bad in ((target, idx[:2], t[:2]), (target[:2], idx, t[:2]), (target[:2], idx[:2], t)):
        with pytest.raises(RuntimeError, match="shape"):
            m(x, *bad)


def test_shapes_of_the_traced_op():
    with FakeTensorMode():
        z, idx, t, target = _cpu()
        op = torch.ops.t2t.distill_loss
        assert op(z, idx, t, target, 1.0, 0.5, -100, 2).shape == ()
        rows = op(z.bfloat16(), idx, t, None, 1.0, 1.0, -100, 0)
        assert rows.shape == (3,) and rows.dtype == torch.float32


def test_training_module_takes_a_teacher():
    kw = dict(vocab_size=32, num_layers=1, model_dim=64, num_heads=1, max_seq_len=8, dropout=0.0,
              drop_path_rate=0.0)
    seen = {}

    def creator(tokens, **rest):
        seen.update(rest)

    plain = TS2TSTrainingModule.from_config(block_mask_creator=creator, **kw)
    assert type(plain.loss_fn) is LinearCELoss
    m = TS2TSTrainingModule.from_config(block_mask_creator=creator, distill_alpha=0.5,
                                        distill_temperature=2.0, **kw)
    assert isinstance(m.loss_fn, LinearDistillLoss)
    assert (m.loss_fn.alpha, m.loss_fn.temperature) == (0.5, 2.0)
    assert m.loss_fn.weight is m.embedding.weight
    m.backbone.forward = lambda x, block_mask: x
    got = {}
    m.loss_fn.forward = lambda x, y, i=None, t=None: got.update(y=y, i=i, t=t)
    tokens = torch.randint(0, 32, (1, 9))
    batch = dict(tokens=tokens, doc_spans=["a"], teacher_idx="i", teacher_logits="t")
    m(batch)
    # the mask creator sees the batch without the teacher, which stays in the batch
    assert seen == {"doc_spans": ["a"]} and got["i"] == "i" and got["t"] == "t"
    assert "teacher_idx" in batch and torch.equal(got["y"], tokens[:, 1:])
    m(dict(tokens=tokens, doc_spans=["a"]))
    assert got["i"] is None and got["t"] is None
    for missing in ("teacher_idx", "teacher_logits"):
        with pytest.raises(ValueError, match="together"):
            m({k: v for k, v in batch.items() if k != missing})
    with pytest.raises(ValueError, match="distill_alpha"):
        plain(batch)
