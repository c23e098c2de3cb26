"""Losses over a vocabulary at the ends of what they take."""
import pytest
import torch

from moc_amd import losses as L
from test_gpu_vocab_loss import check, labels_of, logit_error, operands, rand, reference, shares, teacher_of

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.mark.parametrize("op", ["entropy", "teacher"])
def test_few_rows_in_two_pieces(op):
    """A hidden size of which a piece has fewer rows than dhidden comes from gradients in
    two parts.  All but 64 columns are zeros, whose products and sums are exact."""
    rows, d, wide, vocab = 300, 64, 1 << 19, 70
    small = operands(rows, d, vocab, BF)
    cols = torch.arange(d, device="cuda") * (wide // d) + 5
    h, w = (torch.zeros(t.shape[0], wide, dtype=BF, device="cuda").index_copy(1, cols, t).requires_grad_() for t in small)
    ids, top = teacher_of(rows, vocab, 5, True)
    y = labels_of(rows, vocab, 0.2)
    weight = rand(rows, seed=4).abs() + 0.5
    out = L.linear_cross_entropy(h, w, y, weight) if op == "entropy" else L.linear_distillation(h, w, ids, top, weight)
    got = torch.autograd.grad(out, (h, w))
    hd, wd = (t.to(F64) for t in small)
    if op == "entropy":
        q, some = torch.zeros(rows, vocab, dtype=F64, device="cuda"), y != -100
        q[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    else:
        q, some = shares(ids, top, vocab, 1.0)
    want, dz, c = reference(hd @ wd.t(), q, some, weight.to(F64), 1.0, "mean")
    check(out.detach(), want, [t[:, cols] for t in got], (hd, wd), dz, c, q, logit_error(hd, wd), 1.0, 1.0, weight)
    for t in got:
        assert not t.index_fill(1, cols, 0).any()


@pytest.mark.parametrize("d", [8, 17, 24])
def test_few_rows_of_a_weight_up_to_its_segments_end(d):
    """Hidden sizes of less than a step of the operand registers: the last word's row
    ends the weight's memory."""
    vocab = 1 << 21
    h, w = operands(3, d, vocab, BF)
    y = torch.tensor([vocab - 1, 5, -100], device="cuda")
    hd, wd = h.to(F64), w.to(F64)
    z = hd @ wd.t()
    label = torch.zeros(3, vocab, dtype=F64, device="cuda")
    label[torch.arange(3, device="cuda"), y.clamp(min=0)] = 1
    one = torch.ones(3, dtype=F64, device="cuda")
    want, _, _ = reference(z, label, y != -100, one, 1.0, "none")
    check(L.linear_cross_entropy(h, w, y, reduction="none"), want, (None, None), (hd, wd), z, z, label, logit_error(hd, wd),
          1.0, 1.0, one)
