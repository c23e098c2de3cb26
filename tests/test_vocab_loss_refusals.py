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
    null, teacher = (None, 1, 0, None, 1, 0), (p, 1, 4, p, 1, 4)  # ids, dtype, ld, top, dtype, ld

    def logits(dtype=0, x=p, rows=3, vocab=10, ld=10, by=teacher, words=4, heat=1.0, ldd=10, ws=p, size=1 << 40,
               counters=p):
        return "moc_logits_loss", (dtype, x, rows, vocab, ld, *by, words, heat, None, 1, None, None, p, p, ldd, ws, size,
                                   counters, None)

    def linear(dtype=0, h=p, rows=3, d=8, ldh=8, w=p, vocab=10, ldw=8, labels=p, by=null, words=0, heat=1.0, dh=p,
               dh_dtype=0, ws=p, size=1 << 40, gws=p, gsize=1 << 30):
        return "moc_linear_loss", (dtype, h, rows, d, ldh, w, vocab, ldw, labels, -100, *by, words, heat, None, 1, None,
                                   None, p, dh, dh_dtype, None, 0, ws, size, gws, gsize, None)

    bad = [
        logits(dtype=2), logits(x=None), logits(rows=(1 << 24) + 1), logits(vocab=0), logits(vocab=(1 << 21) + 1),
        logits(ld=9), logits(ldd=9), logits(words=0), logits(words=1025), logits(heat=0.0), logits(heat=math.nan),
        logits(heat=-1.0), logits(heat=math.inf), logits(by=(p, 0, 4, p, 1, 4)), logits(by=(p, 1, 4, p, 2, 4)),
        logits(by=(p, 1, 3, p, 1, 4)), logits(by=(p, 1, 4, p, 1, 3)), logits(by=(None, 1, 4, p, 1, 4)),
        logits(by=(p, 1, 4, None, 1, 4)), logits(ws=None), logits(size=64), logits(counters=None),
        linear(dtype=2), linear(h=None), linear(w=None), linear(labels=None), linear(d=0), linear(d=(1 << 20) + 1),
        linear(rows=(1 << 24) + 1), linear(vocab=(1 << 21) + 1), linear(vocab=0), linear(ldh=12), linear(ldw=4),
        linear(h=ctypes.c_void_p(4100)), linear(heat=2.0), linear(words=4, by=teacher, heat=0.0),
        linear(words=4, by=(p, 1, 3, p, 1, 4)), linear(words=1025, by=teacher), linear(dtype=1, dh_dtype=0),
        linear(dh_dtype=5), linear(size=64), linear(ws=None), linear(gws=None), linear(gsize=64),
        linear(d=512, ldh=512, vocab=1 << 21, ldw=512),
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
