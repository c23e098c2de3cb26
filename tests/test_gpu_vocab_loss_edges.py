"""Losses over a vocabulary at the ends of what they take, and rows
that count for nothing where a gradient has a graph of its own."""
import math

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


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_rows_that_do_not_count_in_a_graph(op, reduction):
    """create_graph: ignored rows, rows without words and rows of weight 0 hold NaN,
    which reaches no gradient, as in the ones that the kernels compute."""
    rows, d, vocab = 12, 32, 100
    h, w = operands(rows, d, vocab, F32)
    ids, top = teacher_of(rows, vocab, 6, False)
    y = labels_of(rows, vocab, 0.0)
    x = 2 * rand(rows, vocab, seed=1)
    weight = rand(rows, seed=4).abs() + 0.5
    dead = torch.tensor([1, 2, 7], device="cuda")
    y[1], ids[1] = -100, -1
    weight[2] = weight[7] = 0
    top[7, 2] = math.nan
    h[dead] = math.nan
    x[dead] = math.nan
    if op == "kept":
        leaves = (x,)
        run = lambda: L.distillation_loss(x, ids, top, weight, reduction=reduction)  # noqa: E731
    else:
        leaves = (h, w)
        run = (lambda: L.linear_cross_entropy(h, w, y, weight, reduction=reduction)) if op == "entropy" else (
            lambda: L.linear_distillation(h, w, ids, top, weight, reduction=reduction))
    for t in leaves:
        t.requires_grad_()
    g = torch.tensor(0.5, device="cuda")
    if reduction == "none":
        g = rand(rows, seed=9).index_fill(0, dead, math.nan)
    want = torch.autograd.grad(run(), leaves, g)
    got = torch.autograd.grad(run(), leaves, g, create_graph=True)
    for a, b in zip(got, want):
        assert a.requires_grad and torch.isfinite(a).all() and torch.isfinite(b).all()
        # two f32 computations of sums of up to 100 terms below the largest
        assert (a - b).abs().max() <= 2 * 100 * 2.0 ** -23 * b.abs().max()
    assert (got[0][dead] == 0).all()
    again = torch.autograd.grad(sum((t * t).sum() for t in got), leaves)
    assert all(torch.isfinite(t).all() for t in again) and (again[0][dead] == 0).all()


@pytest.mark.parametrize("weighted", [False, True])
def test_unknown_label_in_a_graph(weighted):
    """create_graph: a label outside the vocabulary gives NaN gradients, to its own
    hidden row alone, and nothing where its row's weight is 0."""
    h, w = operands(6, 64, 300, F32)
    y = labels_of(6, 300, 0.0)
    y[2], y[4] = 300, -5
    weight = torch.ones(6, device="cuda")
    weight[4] = 0
    h.requires_grad_()
    for graph in (False, True):
        g = torch.autograd.grad(L.linear_cross_entropy(h, w, y, weight if weighted else None), h, create_graph=graph)[0]
        # the mean of NaN losses sends finite factors to all rows
        assert torch.isnan(g).all(1).tolist() == [i == 2 or (i == 4 and not weighted) for i in range(6)]
        assert torch.isnan(g).any(1).tolist() == torch.isnan(g).all(1).tolist()


@pytest.mark.parametrize("words", [3, 0])
def test_2_24_rows(words):
    """As many rows as are taken, more than one launch has workgroups of 256 threads."""
    rows, vocab = 1 << 24, 8
    block = 1 << 12
    g = torch.Generator().manual_seed(1)
    if words:
        x = torch.randn(block, vocab, generator=g).to(BF).cuda().repeat(rows // block, 1).requires_grad_()
        ids = torch.randint(0, vocab, (block, words), generator=g).int().cuda().repeat(rows // block, 1)
        top = torch.randn(block, words, generator=g).to(BF).cuda().repeat(rows // block, 1)
        run = lambda n: L.distillation_loss(x[:n], ids[:n], top[:n], reduction="none")  # noqa: E731
    else:
        x = torch.randn(block, vocab, generator=g).cuda().repeat(rows // block, 1).requires_grad_()
        w = torch.randn(5, vocab, generator=g).cuda()
        y = torch.randint(0, 5, (block,), generator=g).cuda().repeat(rows // block)
        run = lambda n: L.linear_cross_entropy(x[:n], w, y[:n], reduction="none")  # noqa: E731
    each, few = run(rows), run(block)
    assert torch.equal(each.view(-1, block), few.expand(rows // block, block))
    up = rand(block, seed=3)
    got = torch.autograd.grad(each, x, up.repeat(rows // block))[0].view(-1, block, vocab)
    want = torch.autograd.grad(few, x, up)[0][:block]
    assert torch.equal(got, want.expand_as(got))


@pytest.mark.parametrize("op", ["kept", "linear"])
def test_many_rows_of_many_words(op):
    """Rows of more than 256 words of a teacher, in more than one launch."""
    rows, block, vocab, words = (1 << 20) + 5, 1 << 10, 300, 257
    ids, top = teacher_of(block, vocab, words, True, top_dtype=BF)
    full = lambda t: torch.cat([t.repeat(rows // block, 1), t[:rows % block]])  # noqa: E731
    if op == "kept":
        x = (2 * rand(block, vocab, seed=1)).to(BF)
        run = lambda x, ids, top: L.distillation_loss(x, ids, top, reduction="none")  # noqa: E731
    else:
        x, w = operands(block, 16, vocab, BF)
        run = lambda x, ids, top: L.linear_distillation(x, w, ids, top, reduction="none")  # noqa: E731
    few = run(x, ids, top)
    each = run(full(x), full(ids), full(top))
    assert torch.equal(each, full(few[:, None])[:, 0])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_infinite_factor_of_one_row(op, dtype, value):
    """An infinite upstream gradient of one row leaves the others' gradients as they are."""
    h, w = operands(40, 64, 900, dtype)
    ids, top = teacher_of(40, 900, 5, False)
    y = labels_of(40, 900, 0.2)
    x = (3 * rand(40, 900, seed=1)).to(dtype).requires_grad_()
    h.requires_grad_()
    y[7] = 3
    each = L.linear_cross_entropy(h, w, y, reduction="none") if op == "entropy" else (
        L.linear_distillation(h, w, ids, top, reduction="none") if op == "teacher" else
        L.distillation_loss(x, ids, top, reduction="none"))
    g, leaf = rand(40, seed=2), x if op == "kept" else h
    others = torch.arange(40, device="cuda") != 7
    want = torch.autograd.grad(each, leaf, torch.where(others, g, 0.0), retain_graph=True)[0]
    got = torch.autograd.grad(each, leaf, torch.where(others, g, value))[0]
    assert torch.equal(got[others], want[others])
    assert not torch.isfinite(got[7]).any()


def test_hidden_rows_far_apart():
    """Views whose rows' pitch passes what the products address: copies of them."""
    d, vocab = 1 << 20, 66
    cols = torch.arange(64, device="cuda") * (d // 64)
    h, w = operands(3, 64, vocab, BF)
    y = labels_of(3, vocab, 0.0)
    wide = lambda t, pitch: torch.zeros(t.shape[0], pitch, dtype=BF, device="cuda").index_copy(1, cols, t)[:, :d]  # noqa: E731
    want = L.linear_cross_entropy(wide(h, d), wide(w, d), y, reduction="none")
    assert torch.equal(want, L.linear_cross_entropy(wide(h, 4 * d), wide(w, d), y, reduction="none"))
    assert torch.equal(want, L.linear_cross_entropy(wide(h, d), wide(w, 4 * d), y, reduction="none"))


@pytest.mark.parametrize("up", [0, 20, -30])
@pytest.mark.parametrize("rows", [40, 600])
def test_small_channels_beside_large_ones(rows, up):
    """bf16: channels down to 2^-40 of the largest.  The products for the gradients take
    hidden rows and weight as f16 under one power of two, which holds bf16 values above
    2^-19 and 2^-23 as they are (above 2^-32 of a largest that is far from 1) and rounds
    smaller ones by 2^-27 and 2^-31 (2^-39 of it) at most."""
    d, vocab = 82, 700
    h, w = operands(rows, d, vocab, BF)
    size = 2.0 ** -(torch.arange(d, device="cuda") % 41).float()
    h = (h.float() * size * 2.0 ** up).to(BF).requires_grad_()
    w = (w.float() * size.flip(0) * 2.0 ** -up).to(BF).requires_grad_()
    y = labels_of(rows, vocab, 0.2)
    out = L.linear_cross_entropy(h, w, y, reduction="sum")
    got = torch.autograd.grad(out, (h, w))
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    q = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    q[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    one = torch.ones(rows, dtype=F64, device="cuda")
    want, dz, c = reference(hd @ wd.t(), q, y != -100, one, 1.0, "sum")
    z_err = logit_error(hd, wd)
    assert abs(out.item() - want.item()) <= (2 * z_err + 2.0 ** -20 * math.log(2 * vocab)) * rows
    soft = dz.abs() + c * q
    rel = 2.01 * 2.0 ** -11 + 4 * z_err
    for g, exact, terms, other, lost in ((got[0], dz @ wd, soft, wd, 2.0 ** -31), (got[1], dz.t() @ hd, soft.t(), hd, 2.0 ** -27)):
        if up:
            lost = 2.0 ** -39 * other.abs().max().item()
        # dlogits' roundings (2^-39 of the row's factor where they are smallest), f32 sums, the operand's rounding
        tol = (rel + (4 * math.sqrt(terms.shape[1]) + 2) * 2.0 ** -24) * (terms @ other.abs())
        tol = tol + 2.0 ** -39 * other.abs().sum(0) + lost * terms.sum(1)[:, None]
        tol = tol * (1 + 2.0 ** -7) + 2.0 ** -8 * exact.abs() + 1e-38
        err = (g.to(F64) - exact).abs()
        assert (err <= tol).all(), (err / tol).max()
