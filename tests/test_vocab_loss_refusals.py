"""What the losses over a vocabulary refuse, on the host."""
import ctypes
import math

import pytest
import torch

from moc_amd import MoCConfig, _native as N, build_model, losses as L

BF, F32 = torch.bfloat16, torch.float32


def good():
    return dict(hidden=torch.zeros(2, 3, 8), weight=torch.zeros(10, 8), labels=torch.zeros(2, 3, dtype=torch.int64))


def teacher():
    return dict(hidden=torch.zeros(2, 3, 8), weight=torch.zeros(10, 8), teacher_ids=torch.zeros(2, 3, 4, dtype=torch.int32),
                teacher_logits=torch.zeros(2, 3, 4))


@pytest.mark.parametrize("change,says", [
    (dict(reduction="max"), "reduction"),
    (dict(labels=torch.zeros(2, 3, dtype=torch.int32)), "int64"),
    (dict(labels=torch.zeros(6, dtype=torch.int64)), "int64"),
    (dict(hidden=torch.zeros(2, 3, 8, dtype=torch.float16)), "bf16 or f32"),
    (dict(hidden=torch.zeros(2, 3, 8, dtype=BF)), "one type"),
    (dict(weight=torch.zeros(10, 9)), "weight is"),
    (dict(weight=torch.zeros(0, 8)), "weight is"),
    (dict(weight=torch.zeros(10)), "weight is"),
    (dict(row_weight=torch.ones(2, 3, dtype=torch.float64)), "row_weight"),
    (dict(row_weight=torch.ones(6)), "row_weight"),
    (dict(row_weight=torch.ones(2, 3, requires_grad=True)), "no gradient"),
    (dict(weight=torch.zeros(1, 8).expand((1 << 21) + 1, 8)), "2\\^21"),
    (dict(hidden=torch.zeros(2, 3, 512, dtype=BF), weight=torch.zeros(1, 512, dtype=BF).expand(1 << 21, 512)), "2 GiB"),
    (dict(), "device tensors"),
])
def test_cross_entropy(change, says):
    with pytest.raises(ValueError, match=says):
        L.linear_cross_entropy(**{**good(), **change})


@pytest.mark.parametrize("change,says", [
    (dict(temperature=0.0), "temperature"),
    (dict(temperature=math.inf), "temperature"),
    (dict(temperature=math.nan), "temperature"),
    (dict(teacher_ids=torch.zeros(2, 3, 4)), "int32 or int64"),
    (dict(teacher_logits=torch.zeros(2, 3, 4, dtype=torch.float16)), "bf16 or f32"),
    (dict(teacher_logits=torch.zeros(2, 3, 5)), "words"),
    (dict(teacher_ids=torch.zeros(6, 4, dtype=torch.int32), teacher_logits=torch.zeros(6, 4)), "words"),
    (dict(teacher_ids=torch.zeros(2, 3, 0, dtype=torch.int32), teacher_logits=torch.zeros(2, 3, 0)), "1 to 1024"),
    (dict(teacher_ids=torch.zeros(2, 3, 1025, dtype=torch.int32), teacher_logits=torch.zeros(2, 3, 1025)), "1 to 1024"),
    (dict(teacher_logits=torch.zeros(2, 3, 4, requires_grad=True)), "no gradient"),
    (dict(reduction=None), "reduction"),
    (dict(), "device tensors"),
])
def test_distillation(change, says):
    args = {**teacher(), **change}
    with pytest.raises(ValueError, match=says):
        L.linear_distillation(**args)
    args["logits"] = torch.zeros(2, 3, 10)
    del args["hidden"], args["weight"]
    with pytest.raises(ValueError, match=says):
        L.distillation_loss(**args)


def test_entry_points_refuse():
    """The library's own checks, before any device work: none of these pointers is read."""
    lib = N.load()
    p = ctypes.c_void_p(4096)
    bad = [
        ("moc_label_targets", (None, 4, 10, -100, None, 1, None, p, None)),
        ("moc_label_targets", (p, 4, 10, -100, None, 1, None, None, None)),
        ("moc_label_targets", (p, 4, 0, -100, None, 1, None, p, None)),
        ("moc_label_targets", (p, 4, (1 << 21) + 1, -100, None, 1, None, p, None)),
        ("moc_label_targets", (p, (1 << 24) + 1, 10, -100, None, 1, None, p, None)),
        ("moc_teacher_targets", (p, 1, 4, p, 1, 4, 3, 0, 10, 1.0, None, 1, None, p, None)),
        ("moc_teacher_targets", (p, 1, 4, p, 1, 4, 3, 1025, 10, 1.0, None, 1, None, p, None)),
        ("moc_teacher_targets", (p, 0, 4, p, 1, 4, 3, 4, 10, 1.0, None, 1, None, p, None)),
        ("moc_teacher_targets", (p, 1, 4, p, 2, 4, 3, 4, 10, 1.0, None, 1, None, p, None)),
        ("moc_teacher_targets", (p, 1, 3, p, 1, 4, 3, 4, 10, 1.0, None, 1, None, p, None)),
        ("moc_teacher_targets", (p, 1, 4, p, 1, 4, 3, 4, 10, 0.0, None, 1, None, p, None)),
        ("moc_teacher_targets", (p, 1, 4, p, 1, 4, 3, 4, 10, math.nan, None, 1, None, p, None)),
        ("moc_logits_loss", (2, p, 3, 10, 10, p, 4, 1.0, p, p, p, 10, None)),
        ("moc_logits_loss", (0, p, 3, 10, 9, p, 4, 1.0, p, p, p, 10, None)),
        ("moc_logits_loss", (0, p, 3, 10, 10, p, 4, 1.0, p, p, p, 9, None)),
        ("moc_logits_loss", (0, None, 3, 10, 10, p, 4, 1.0, p, p, p, 10, None)),
        ("moc_logits_loss", (0, p, 3, 10, 10, p, 4, -1.0, p, p, p, 10, None)),
        ("moc_linear_loss", (0, p, 3, 8, 8, p, 10, 8, p, 0, 1.0, p, p, p, 0, p, 0, p, 64, None, 0, None)),  # workspace
        ("moc_linear_loss", (0, p, 3, 8, 12, p, 10, 8, p, 0, 1.0, p, p, None, 0, None, 0, p, 1 << 40, None, 0, None)),
        ("moc_linear_loss", (1, p, 3, 8, 8, p, 10, 8, p, 0, 1.0, p, p, p, 0, None, 0, p, 1 << 40, None, 0, None)),
        ("moc_linear_loss", (0, p, 3, 0, 8, p, 10, 8, p, 0, 1.0, p, p, None, 0, None, 0, p, 1 << 40, None, 0, None)),
        ("moc_linear_loss", (0, p, 3, 512, 512, p, 1 << 21, 512, p, 0, 1.0, p, p, None, 0, None, 0, p, 1 << 40, None, 0,
                             None)),
        ("moc_scale_inplace", (5, p, 8, 0, None, 0, p, None)),
        ("moc_scale_inplace", (0, None, 8, 0, None, 0, p, None)),
        ("moc_scale_inplace", (0, p, 8, 0, None, 8, p, None)),
        ("moc_scale_inplace", (0, p, 8, 0, None, 0, None, None)),
    ]
    for name, args in bad:
        assert getattr(lib, name)(*args) == N.MOC_ERR_INVALID, (name, args)
        assert name.split("_")[1] in N.last_error() or "moc_" in N.last_error()


def test_model_off_the_device():
    """loss() is forward's; distill() says what it takes."""
    torch.manual_seed(0)
    model = build_model(MoCConfig(hidden_size=32, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2,
                                  vocab_size=50, max_seq_len=16), "dense")
    ids = torch.randint(0, 50, (2, 9))
    labels = torch.where(torch.rand(2, 9) < 0.3, -100, ids)
    # the same f32 terms in another order of summation, 16 of them
    assert torch.allclose(model.loss(ids, labels), model(ids, labels)[1], rtol=16 * 2.0 ** -24, atol=0)
    weight = torch.rand(2, 9)
    on = labels[:, 1:] != -100
    each = torch.nn.functional.cross_entropy(model(ids)[:, :-1].flatten(0, 1).double(), labels[:, 1:].flatten(),
                                             reduction="none", ignore_index=-100)
    w = torch.where(on, weight[:, :-1], 0.0).flatten().double()
    # f32 logits, exponentials and sums over 50 words: 2^-20 of the loss
    assert torch.allclose(model.loss(ids, labels, weight).double(), (each * w).sum() / w.sum(), rtol=2.0 ** -20, atol=0)
    with pytest.raises(ValueError, match="plain LM head"):
        model.distill(ids, ids[..., None].int(), torch.zeros(2, 9, 1))
