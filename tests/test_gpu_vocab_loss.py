"""Losses over a vocabulary against 64 bits: linear cross entropy, linear
distillation, distillation of kept logits, with their gradients.

Tolerances.  A logit is a sum of d products that bf16 or f32 operands give without
or with one rounding of 2^-24: with S the largest sum of |h||w|, an error of 4 sqrt(d)
2^-24 S (roundings of either sign) and 2 more units for an f32 product's own.  A
row's loss differs by twice that and by f32 exponentials, logarithms and a sum over
the vocabulary, 2^-20 of its terms.  A gradient is a sum over dlogits, which are
rounded to f16 twice (2^-11 of each; 2^-39 of the row's factor where it is smallest)
or to f16 once and two bf16 parts (less),
its other operand by 2^-24 of its largest value, or stay f32 (2^-23 with the
exponential's own), behind a relative error of the logits' errors, and is rounded
itself; |dlogits| |operand| in 64 bits bounds what that comes to.  p's relative error
counts for p, not for p - q: with c the row's factor, c p <= |dlogits| + c q.  A
gradient that was computed ahead and rounded to bf16 is rounded once more by an
upstream factor that is no power of two: (1 + 2^-8)^2 - 1 < 2.01 2^-8.
"""
import math

import pytest
import torch

from moc_amd import losses as L

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SIZES = [(1, 8, 1), (1, 64, 500), (3, 100, 1003), (17, 256, 4099), (40, 2048, 8190), (256, 64, 32000), (300, 512, 2050),
         (1030, 96, 777), (129, 1000, 5000), (5, 1, 9), (2, 24, 1), (1, 7, 2), (257, 333, 700)]


def rand(*shape, seed):
    g = torch.Generator().manual_seed(seed + 7 * math.prod(shape))
    return torch.randn(*shape, generator=g).cuda()


def operands(rows, d, vocab, dtype, seed=0):
    w = (rand(vocab, d, seed=seed) * (1.5 / math.sqrt(d))).to(dtype)
    h = (rand(rows, d, seed=seed + 1) + 2 * w[torch.arange(rows, device="cuda") % vocab].float()).to(dtype)
    return h, w


def labels_of(rows, vocab, masked, seed=3):
    g = torch.Generator().manual_seed(seed + rows)
    y = torch.randint(0, vocab, (rows,), generator=g)
    y[torch.rand(rows, generator=g) < masked] = -100
    return y.cuda()


def teacher_of(rows, vocab, words, ragged, seed=5, ids_dtype=torch.int32, top_dtype=F32):
    g = torch.Generator().manual_seed(seed + rows + words)
    ids = torch.randint(0, vocab, (rows, words), generator=g)  # the same word twice now and then
    top = torch.randn(rows, words, generator=g) * 2
    if ragged:
        ids[torch.rand(rows, words, generator=g) < 0.3] = -1
        top[torch.rand(rows, words, generator=g) < 0.1] = -math.inf
        ids[torch.rand(rows, generator=g) < 0.2] = -1
        ids[rows // 2, 0], top[rows // 2, 0] = vocab - 1, 0.5
        ids[rows // 2 - 1, -1] = vocab  # outside
    return ids.to("cuda", ids_dtype), top.to("cuda", top_dtype)


def shares(ids, top, vocab, heat):
    """The teacher's distribution over the whole vocabulary, rows that have one."""
    ids, x = ids.long(), top.to(F64) / heat
    there = (ids >= 0) & (ids < vocab) & (x != -math.inf)
    some = there.any(1)
    q = torch.where(there, torch.exp(x - torch.where(there, x, -math.inf).amax(1, keepdim=True).clamp(min=-1e30)), 0.0)
    q = q / q.sum(1, keepdim=True).clamp(min=1e-300)
    return torch.zeros(ids.shape[0], vocab, dtype=F64, device="cuda").scatter_add_(1, torch.where(there, ids, 0), q), some


def reference(z, q, counts, weight, heat, reduction):
    """(loss or rows' losses, dloss / dz for an upstream gradient of 1, the rows' factors c)."""
    log_p = torch.log_softmax(z / heat, -1)
    each = heat ** 2 * torch.where(q > 0, q * (torch.log(q.clamp(min=1e-300)) - log_p), 0.0).sum(-1)
    w = torch.where(counts, weight, 0.0)
    dz = heat * (log_p.exp() - q)
    n = w.sum() if reduction == "mean" else 1.0
    each = torch.where(w != 0, each * w, 0.0)
    dz = torch.where((w != 0)[:, None], dz * (w / n)[:, None], 0.0)
    return (each if reduction == "none" else each.sum() / n), dz, (heat * w / n).abs()[:, None]


def logit_error(h, w):
    s = (h.abs() @ w.abs().t()).amax().item()
    return (4 * math.sqrt(h.shape[1]) + 2) * 2.0 ** -24 * s


def check(out, want, got, leaves, dz, c, q, z_err, heat, factor, weights):
    """Loss and gradients (None: not asked for) of the linear losses."""
    scale = (want.abs() if want.dim() else want.abs() + 1) + weights.abs().max()
    tol = (2 * z_err * heat + 2.0 ** -20 * math.log(2 * q.shape[1]) * heat ** 2) * scale
    assert ((out.to(F64) - want).abs() <= tol).all(), ((out.to(F64) - want).abs() / tol).max()
    h, w = leaves
    dz, c = dz * factor, c * abs(factor)
    soft = dz.abs() + c * q
    for got_, want_, size, i in ((got[0], dz @ w, soft @ w.abs(), 0), (got[1], dz.t() @ h, soft.t() @ h.abs(), 1)):
        if got_ is None:
            continue
        half = got_.dtype == BF
        rel = (2.01 * 2.0 ** -11 if half else 2.0 ** -22) + 4 * z_err / heat
        terms = dz.shape[1 - i]
        tol = rel * size + (4 * math.sqrt(terms) + 2) * 2.0 ** -24 * size
        if half:
            other = (w if i == 0 else h).abs()
            tol = tol + 2.0 ** -39 * c.max() * other.sum(0) + 2.0 ** -24 * other.max() * (
                soft.sum(1)[:, None] if i == 0 else soft.sum(0)[:, None])
        if got_.dtype == BF:
            tol = tol * (1 + 2.0 ** -7) + (1 if want.dim() else 2.01) * 2.0 ** -8 * want_.abs() + 1e-38
        err = (got_.to(F64) - want_).abs()
        assert (err <= tol).all(), (i, (err / tol).max(), err.max())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,d,vocab", SIZES)
@pytest.mark.parametrize("masked,weighted,reduction", [(0.0, False, "mean"), (0.4, True, "mean"), (0.9, True, "sum"),
                                                       (0.3, True, "none")])
def test_linear_cross_entropy(rows, d, vocab, dtype, masked, weighted, reduction):
    h, w = operands(rows, d, vocab, dtype)
    y = labels_of(rows, vocab, masked)
    y[rows // 2] = vocab - 1
    weight = rand(rows, seed=9) if weighted else torch.ones(rows, device="cuda")
    if weighted:
        weight[rows // 2] = 1.5 + rows  # a mean's divisor away from 0
        weight[rows // 3 + 1:rows // 3 + 2] = 0
    counts = y != -100
    h[~counts | (weight == 0)] = math.nan  # nobody looks at these
    h.requires_grad_()
    w.requires_grad_()
    out = L.linear_cross_entropy(h, w, y, weight if weighted else None, reduction=reduction)
    assert out.dtype == F32
    g = rand(rows, seed=11) if reduction == "none" else torch.tensor(0.7, device="cuda")
    got = torch.autograd.grad(out, (h, w), g)
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    hd = torch.where((counts & (weight != 0))[:, None], hd, 0.0)
    q = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    q[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    want, dz, c = reference(hd @ wd.t(), q, counts, weight.to(F64), 1.0, reduction)
    check(out.detach(), want, got, (hd, wd), dz, c, q, logit_error(hd, wd), 1.0, g.to(F64)[:, None] if reduction == "none"
          else g.to(F64), weight)
    assert (got[0][~counts] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,d,vocab", SIZES)
@pytest.mark.parametrize("words,heat,ragged,reduction", [(1, 1.0, False, "mean"), (7, 2.0, True, "mean"),
                                                         (64, 0.7, False, "sum"), (65, 1.0, True, "mean"),
                                                         (200, 1.0, True, "sum"), (300, 1.0, True, "none")])
def test_linear_distillation(rows, d, vocab, dtype, words, heat, ragged, reduction):
    h, w = operands(rows, d, vocab, dtype)
    h, w = h.requires_grad_(), w.requires_grad_()
    ids, top = teacher_of(rows, vocab, words, ragged, ids_dtype=torch.int64 if words == 7 else torch.int32,
                          top_dtype=BF if words == 64 else F32)
    out = L.linear_distillation(h, w, ids, top, temperature=heat, reduction=reduction)
    g = rand(rows, seed=11) if reduction == "none" else torch.tensor(-1.3, device="cuda")
    got = torch.autograd.grad(out, (h, w), g)
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    q, some = shares(ids, top, vocab, heat)
    one = torch.ones(rows, dtype=F64, device="cuda")
    want, dz, c = reference(hd @ wd.t(), q, some, one, heat, reduction)
    check(out.detach(), want, got, (hd, wd), dz, c, q, logit_error(hd, wd), heat,
          g.to(F64)[:, None] if reduction == "none" else g.to(F64), one)
    assert (got[0][~some] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [1, 3, 16, 17, 129])
@pytest.mark.parametrize("d,vocab", [(8, 1), (40, 63), (104, 64), (64, 65), (256, 1003), (1000, 4099), (2048, 32000),
                                     (4096, 5000), (4104, 700), (520, 128256)])
def test_losses_alone(rows, d, vocab, dtype):
    """Without gradients: rows' losses and their mean, labels and a teacher's words."""
    h, w = operands(rows, d, vocab, dtype)
    y = labels_of(rows, vocab, 0.3)
    y[rows // 2] = vocab - 1
    ids, top = teacher_of(rows, vocab, 70 if rows == 3 else 9, True)
    hd, wd = h.to(F64), w.to(F64)
    z, z_err = hd @ wd.t(), logit_error(hd, wd)
    h[y == -100] = math.nan
    label = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    label[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    weight = rand(rows, seed=9).abs() + 0.1
    want, _, _ = reference(z, label, y != -100, weight.to(F64), 1.0, "none")
    out = L.linear_cross_entropy(h, w, y, weight, reduction="none")
    check(out, want, (None, None), (hd, wd), z, z, label, z_err, 1.0, 1.0, weight)
    mean = L.linear_cross_entropy(h, w, y, weight)
    check(mean, want.sum() / torch.where(y != -100, weight.to(F64), 0.0).sum(), (None, None), (hd, wd), z, z, label, z_err,
          1.0, 1.0, weight)
    h = torch.where((y == -100)[:, None], hd.to(dtype), h)
    q, some = shares(ids, top, vocab, 1.5)
    want, _, _ = reference(z, q, some, weight.to(F64), 1.5, "none")
    check(L.linear_distillation(h, w, ids, top, weight, temperature=1.5, reduction="none"), want, (None, None), (hd, wd), z,
          z, q, z_err, 1.5, 1.0, weight)
    check(L.linear_distillation(h, w, ids, top, weight, temperature=1.5),
          want.sum() / torch.where(some, weight.to(F64), 0.0).sum(), (None, None), (hd, wd), z, z, q, z_err, 1.5, 1.0, weight)
    x = z.to(F32)
    kept = L.distillation_loss(x, ids, top, weight, temperature=1.5)
    # the f32 rounding of the logits and the scaling's, twice, on top of the sums'
    tol = (4 * 2.0 ** -24 * (z.abs().max().item() + 20) + 2.0 ** -20 * math.log(2 * vocab)) * 2.25
    mean = want.sum() / torch.where(some, weight.to(F64), 0.0).sum()
    assert abs(kept.item() - mean.item()) <= tol * (abs(mean.item()) + 1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 3), (5, 500), (33, 1003), (7, 32000), (3, 50021), (2, 128256),
                                        (2, 262147), (2, 270011), (600, 4096), (3000, 77)])
@pytest.mark.parametrize("words,heat,ragged,reduction", [(1, 1.0, False, "mean"), (20, 2.0, True, "mean"),
                                                         (101, 0.7, False, "sum"), (256, 1.0, True, "mean"),
                                                         (257, 1.0, True, "mean"), (1024, 1.0, True, "none")])
def test_distillation_loss(rows, vocab, dtype, words, heat, ragged, reduction):
    x = (3 * rand(rows, vocab, seed=2)).to(dtype)
    ids, top = teacher_of(rows, vocab, words, ragged)
    q, some = shares(ids, top, vocab, heat)
    x[~some] = math.nan
    x.requires_grad_()
    out = L.distillation_loss(x, ids, top, temperature=heat, reduction=reduction)
    g = rand(rows, seed=11) if reduction == "none" else torch.tensor(0.7, device="cuda")
    got = torch.autograd.grad(out, x, g)[0]
    z = torch.where(some[:, None], x.detach().to(F64), 0.0)
    want, dz, c = reference(z, q, some, torch.ones(rows, dtype=F64, device="cuda"), heat, reduction)
    top_z = z.abs().max().item() / heat
    # scaling a logit and subtracting two f32 numbers of its size, on top of 2^-20
    rel = 2.0 ** -20 + 4 * 2.0 ** -24 * (top_z + 20)
    tol = rel * heat ** 2 * (want.abs() / heat ** 2 + math.log(2 * vocab) + top_z)
    assert ((out.detach().to(F64) - want).abs() <= tol).all()
    factor = g.to(F64)[:, None] if reduction == "none" else g.to(F64)
    dz = dz * factor
    # two roundings: the gradient's own and the upstream factor's
    tol = 8 * rel * (dz.abs() + c * abs(factor) * q) + (2.01 * 2.0 ** -8 if dtype == BF else 2.0 ** -23) * dz.abs() + 1e-38
    err = (got.to(F64) - dz).abs()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("up", [-60, -14, -5, 9, 40])
@pytest.mark.parametrize("op", ["entropy", "teacher"])
def test_operands_of_any_size(up, op):
    """Hidden rows of another size and a weight that makes up for it; row weights of
    any size."""
    h, w = operands(70, 200, 900, BF)
    h[3, 5] = 100.0
    h, w = (h.float() * 2.0 ** up).to(BF).requires_grad_(), (w.float() * 2.0 ** -up).to(BF).requires_grad_()
    ids, top = teacher_of(70, 900, 5, True)
    y = labels_of(70, 900, 0.2)
    weight = (rand(70, seed=4).abs() + 0.5) * 2.0 ** (up / 2)
    out = L.linear_cross_entropy(h, w, y, weight, reduction="sum") if op == "entropy" else (
        L.linear_distillation(h, w, ids, top, weight, reduction="sum"))
    got = torch.autograd.grad(out, (h, w))
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    if op == "entropy":
        q, some = torch.zeros(70, 900, dtype=F64, device="cuda"), y != -100
        q[torch.arange(70, device="cuda"), y.clamp(min=0)] = 1
    else:
        q, some = shares(ids, top, 900, 1.0)
    want, dz, c = reference(hd @ wd.t(), q, some, weight.to(F64), 1.0, "sum")
    check(out.detach(), want, got, (hd, wd), dz, c, q, logit_error(hd, wd), 1.0, 1.0, weight)


def test_rows_in_pieces():
    """More logits than a piece holds: sums over the pieces."""
    rows, d, vocab = 5300, 64, 128256
    h, w = operands(rows, d, vocab, BF)
    h, w = h.requires_grad_(), w.requires_grad_()
    y = labels_of(rows, vocab, 0.2)
    out = L.linear_cross_entropy(h, w, y)
    got = torch.autograd.grad(out, (h, w))
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    q = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    q[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    one = torch.ones(rows, dtype=F64, device="cuda")
    want, dz, c = reference(hd @ wd.t(), q, y != -100, one, 1.0, "mean")
    check(out.detach(), want, got, (hd, wd), dz, c, q, logit_error(hd, wd), 1.0, 1.0, one)


def test_nothing_counts():
    h, w = operands(9, 64, 300, BF)
    h, w = h.requires_grad_(), w.requires_grad_()
    for reduction, value in (("sum", 0.0), ("mean", math.nan), ("none", 0.0)):
        out = L.linear_cross_entropy(h, w, torch.full((9,), -100, device="cuda"), reduction=reduction)
        assert ((out == value) | (torch.isnan(out) & math.isnan(value))).all()
        if reduction != "mean":
            for t in torch.autograd.grad(out.sum(), (h, w)):
                assert (t == 0).all()


def test_unknown_label_is_nan():
    h, w = operands(6, 64, 300, BF)
    y = labels_of(6, 300, 0.0)
    y[2] = 300
    each = L.linear_cross_entropy(h, w, y, reduction="none")
    assert torch.isnan(each).tolist() == [i == 2 for i in range(6)]
    h = h.requires_grad_()
    g = torch.autograd.grad(L.linear_cross_entropy(h, w, y), h)[0]
    assert torch.isnan(g).all(1).tolist() == [i == 2 for i in range(6)]


@pytest.mark.parametrize("lead", [(2, 5), (3,), (), (2, 2, 3), (0,), (2, 0)])
def test_leading_shapes_and_no_rows(lead):
    h, w = operands(max(1, math.prod(lead)), 64, 300, BF)
    h = h[:math.prod(lead)].reshape(*lead, 64).clone().requires_grad_()
    w = w.requires_grad_()
    y = labels_of(math.prod(lead), 300, 0.0).reshape(lead)
    each = L.linear_cross_entropy(h, w, y, reduction="none")
    assert each.shape == h.shape[:-1]
    flat = L.linear_cross_entropy(h.reshape(-1, 64), w, y.reshape(-1), reduction="none")
    assert torch.equal(each.reshape(-1), flat)
    total = L.linear_cross_entropy(h, w, y, reduction="sum")
    dh, dw = torch.autograd.grad(total, (h, w))
    assert dh.shape == h.shape and dw.shape == w.shape and torch.isfinite(dw).all()
    if not math.prod(lead):
        assert total == 0 and (dw == 0).all()


def test_strides_and_alignment():
    """Views with other strides and bases give what contiguous copies give."""
    base_h, base_w = operands(50, 200, 700, BF)
    y = labels_of(50, 700, 0.1)
    pad = lambda t, a: torch.zeros(t.shape[0], t.shape[1] + a, dtype=t.dtype, device="cuda")  # noqa: E731
    want = None
    for make in (lambda t: t.clone(), lambda t: pad(t, 3)[:, 1:-2].copy_(t), lambda t: pad(t, 8)[:, :-8].copy_(t),
                 lambda t: t.t().contiguous().t(), lambda t: torch.repeat_interleave(t, 2, 0)[::2]):
        h, w = make(base_h).requires_grad_(), make(base_w).requires_grad_()
        out = L.linear_cross_entropy(h, w, y)
        got = (out, *torch.autograd.grad(out, (h, w)))
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ids, top = teacher_of(50, 700, 9, True)
    x = (3 * rand(50, 700, seed=1)).to(BF)
    a = L.distillation_loss(x, ids, top)
    for make in (lambda t: pad(t, 3)[:, 1:-2].copy_(t), lambda t: t.t().contiguous().t()):
        assert torch.equal(a, L.distillation_loss(make(x), make(ids.float()).int(), make(top)))


def test_many_rows_without_gradients():
    """More hidden rows than 32-bit offsets reach: in pieces."""
    rows, d, vocab = 140000, 4096, 40
    w = operands(8, d, vocab, BF)[1]
    h = rand(1000, d, seed=1).to(BF).repeat(rows // 1000, 1)
    y = labels_of(1000, vocab, 0.2).repeat(rows // 1000)
    each = L.linear_cross_entropy(h, w, y, reduction="none")
    assert torch.equal(each[:1000].repeat(rows // 1000), each)
    assert torch.equal(each[:1000], L.linear_cross_entropy(h[:1000], w, y[:1000], reduction="none"))
    mean = L.linear_cross_entropy(h, w, y)
    # the same rows' f32 losses in 64 bits, once
    assert abs(mean.item() - each[:1000].to(F64).sum().item() / (y[:1000] != -100).sum().item()) <= 2.0 ** -23 * mean.item()


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_second_backward_and_factor(op):
    """The gradients ahead are handed out once, computed again then."""
    h, w = operands(70, 128, 900, BF)
    h, w = h.requires_grad_(), w.requires_grad_()
    ids, top = teacher_of(70, 900, 5, True)
    y = labels_of(70, 900, 0.2)
    if op == "kept":
        x = (3 * rand(70, 900, seed=1)).to(BF).requires_grad_()
        leaves, loss = (x,), L.distillation_loss(x, ids, top)
    else:
        leaves = (h, w)
        loss = L.linear_cross_entropy(h, w, y) if op == "entropy" else L.linear_distillation(h, w, ids, top)
    first = [t.clone() for t in torch.autograd.grad(loss, leaves, retain_graph=True)]
    again = torch.autograd.grad(loss, leaves, retain_graph=True)
    third = torch.autograd.grad(loss, leaves, torch.tensor(4.0, device="cuda"))
    for a, b, c in zip(first, again, third):
        assert torch.equal(a, b) and torch.equal(a * 4, c)


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_only_what_is_asked_for(op):
    h, w = operands(40, 64, 300, BF)
    ids, top = teacher_of(40, 300, 5, False)
    y = labels_of(40, 300, 0.2)
    run = (lambda a, b: L.linear_cross_entropy(a, b, y)) if op == "entropy" else (
        lambda a, b: L.linear_distillation(a, b, ids, top)) if op == "teacher" else (
        lambda a, b: L.distillation_loss(a, ids, top))
    if op == "kept":
        h = (3 * rand(40, 300, seed=1)).to(BF)
    plain = run(h, w)
    assert not plain.requires_grad
    with torch.no_grad():
        assert torch.equal(plain, run(h.clone().requires_grad_(), w.clone().requires_grad_()))
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(run(a, b), (a, b), allow_unused=op == "kept")
    assert torch.equal(torch.autograd.grad(run(a, w), a)[0], both[0])
    if op != "kept":
        assert torch.equal(torch.autograd.grad(run(h, b), b)[0], both[1])


@pytest.mark.parametrize("op", ["entropy", "teacher"])
@pytest.mark.parametrize("types", [(F32, F32), (BF, F32), (F32, BF)])
def test_autocast(op, types):
    """Under bf16 autocast: products of bf16 casts, gradients in the operands' types."""
    h, w = operands(60, 128, 900, F32)
    h, w = h.to(types[0]).requires_grad_(), w.to(types[1]).requires_grad_()
    ids, top = teacher_of(60, 900, 5, True)
    y = labels_of(60, 900, 0.2)
    hb, wb = (t.detach().to(BF).requires_grad_() for t in (h, w))
    run = (lambda a, b: L.linear_cross_entropy(a, b, y)) if op == "entropy" else (
        lambda a, b: L.linear_distillation(a, b, ids, top))
    with torch.autocast("cuda", dtype=BF):
        out = run(h, w)
    plain = run(hb, wb)
    assert torch.equal(out, plain)
    for a, b, t in zip(torch.autograd.grad(out, (h, w)), torch.autograd.grad(plain, (hb, wb)), types):
        assert a.dtype == t and torch.equal(a.to(BF), b)


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_second_derivative(op, reduction):
    """A gradient with a graph of its own, against one in 64 bits."""
    rows, d, vocab, heat = 6, 16, 40, 1.5
    h, w = operands(rows, d, vocab, F32)
    ids, top = teacher_of(rows, vocab, 4, False)
    y = labels_of(rows, vocab, 0.3)
    y[0] = 3
    v = [rand(rows, d, seed=21), rand(vocab, d, seed=22)]
    if op == "kept":
        leaves = [(2 * rand(rows, vocab, seed=1)).requires_grad_()]
        v = [rand(rows, vocab, seed=23)]
        run = lambda x: L.distillation_loss(x, ids, top, temperature=heat, reduction=reduction)  # noqa: E731
    else:
        leaves = [h.requires_grad_(), w.requires_grad_()]
        run = (lambda a, b: L.linear_cross_entropy(a, b, y, reduction=reduction)) if op == "entropy" else (
            lambda a, b: L.linear_distillation(a, b, ids, top, temperature=heat, reduction=reduction))
    grads = torch.autograd.grad(run(*leaves).sum(), leaves, create_graph=True)
    got = torch.autograd.grad(sum((a * b).sum() for a, b in zip(grads, v)), leaves)
    exact = [t.detach().to(F64).requires_grad_() for t in leaves]
    z = exact[0] if op == "kept" else exact[0] @ exact[1].t()
    log_p = torch.log_softmax(z / (1.0 if op == "entropy" else heat), -1)
    if op == "entropy":
        on = y != -100
        each = -log_p[on, y[on]]
    else:
        q, _ = shares(ids, top, vocab, heat)
        each = -heat ** 2 * (q * log_p).sum(1)
    loss = each.sum() if reduction == "none" else each.mean()
    grads = torch.autograd.grad(loss, exact, create_graph=True)
    want = torch.autograd.grad(sum((a * b.to(F64)).sum() for a, b in zip(grads, v)), exact)
    for a, b in zip(got, want):
        # f32 sums of some hundred terms of the result's size
        assert (a.to(F64) - b).abs().max() <= 1e-4 * b.abs().max()


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_gradient_by_differences(op):
    """f32 operands: the loss along a direction against the gradient."""
    rows, d, vocab = 12, 32, 200
    h, w = operands(rows, d, vocab, F32)
    ids, top = teacher_of(rows, vocab, 6, True)
    y = labels_of(rows, vocab, 0.2)
    y[0] = 3
    if op == "kept":
        leaves = [(2 * rand(rows, vocab, seed=1)).requires_grad_()]
        run = lambda x: L.distillation_loss(x, ids, top, temperature=2.0, reduction="sum")  # noqa: E731
    else:
        leaves = [h.requires_grad_(), w.requires_grad_()]
        run = (lambda a, b: L.linear_cross_entropy(a, b, y, reduction="sum")) if op == "entropy" else (
            lambda a, b: L.linear_distillation(a, b, ids, top, temperature=2.0, reduction="sum"))
    grads = torch.autograd.grad(run(*leaves), leaves)
    way = [rand(*t.shape, seed=31) for t in leaves]
    slope = sum((a.to(F64) * b.to(F64)).sum() for a, b in zip(grads, way)).item()
    step = 2.0 ** -7
    with torch.no_grad():
        up, down = (run(*[t + s * b for t, b in zip(leaves, way)]).to(F64).item() for s in (step, -step))
    # the third derivative along the way (step^2 of the slope's size times its
    # logits' cube, below 8^3 / 6 each) and f32 losses over 2 step
    size = abs(up) + 1
    assert abs((up - down) / (2 * step) - slope) <= step ** 2 * 90 * size + 2.0 ** -20 * size / step


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_captured_pass(op):
    """Forward and backward in one HIP graph, replayed on changed inputs."""
    h, w = operands(130, 128, 2000, BF)
    h, w = h.requires_grad_(), w.requires_grad_()
    ids, top = teacher_of(130, 2000, 8, True)
    y = labels_of(130, 2000, 0.2)
    x = (3 * rand(130, 2000, seed=1)).to(BF).requires_grad_()
    factor = torch.tensor(0.7, device="cuda")
    leaves = (x,) if op == "kept" else (h, w)

    def step():
        loss = L.linear_cross_entropy(h, w, y) if op == "entropy" else (
            L.linear_distillation(h, w, ids, top, temperature=2.0) if op == "teacher" else
            L.distillation_loss(x, ids, top, temperature=2.0))
        return (loss.detach(), *torch.autograd.grad(loss, leaves, factor))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for t in leaves:
                t.copy_((t.float() * (0.9 + 0.1 * i)).to(BF))
            y.copy_(labels_of(130, 2000, 0.3, seed=i))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_two_graphs_at_once(op):
    """Graphs captured on one stream, replayed beside each other on two."""
    leaves, graphs, outs = [], [], []
    ids, top = teacher_of(700, 3000, 8, True)
    y = labels_of(700, 3000, 0.2)

    def step(h, w, x):
        if op == "kept":
            loss = L.distillation_loss(x, ids, top)
            return (loss.detach(), *torch.autograd.grad(loss, x))
        loss = L.linear_cross_entropy(h, w, y) if op == "entropy" else L.linear_distillation(h, w, ids, top)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    for i in range(2):
        h, w = operands(700, 256, 3000, BF, seed=10 * i)
        leaves.append((h.requires_grad_(), w.requires_grad_(), (3 * rand(700, 3000, seed=i)).to(BF).requires_grad_()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves[0])
    torch.cuda.current_stream().wait_stream(side)
    for own in leaves:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step(*own))
        graphs.append(graph)
    want = [step(*own) for own in leaves]
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got, exact in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, exact))


def test_captured_backward_of_an_eager_forward():
    """Each replay of a captured backward gives the same gradients."""
    w = operands(30, 64, 500, BF)[1]
    y = labels_of(30, 500, 0.1)
    factor = torch.tensor(0.5, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h = operands(30, 64, 500, BF)[0].requires_grad_()
        want = torch.autograd.grad(L.linear_cross_entropy(h, w, y), h, factor)[0]
        loss = L.linear_cross_entropy(h, w, y)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(loss, h, factor)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        # 0.5 scales without rounding
        assert torch.equal(got, want)


def test_other_stream():
    h, w = operands(300, 256, 3000, BF)
    h, w = h.requires_grad_(), w.requires_grad_()
    y = labels_of(300, 3000, 0.2)
    want = L.linear_cross_entropy(h, w, y)
    want = (want, *torch.autograd.grad(want, (h, w)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = L.linear_cross_entropy(h, w, y)
        got = (out, *torch.autograd.grad(out, (h, w)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_on_the_device():
    h, w = operands(6, 64, 300, F32)
    y = labels_of(6, 300, 0.0)
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(ValueError, match="bf16"):
        L.linear_cross_entropy(h, w, y)
    with pytest.raises(ValueError, match="device"):
        L.linear_cross_entropy(h, w, y.cpu())
    with pytest.raises(ValueError, match="one type"):
        L.linear_cross_entropy(h, w.to(BF), y)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [500, 4099, 50021, 270011])
@pytest.mark.parametrize("words,heat", [(7, 1.0), (7, 0.5), (300, 2.0)])
def test_lowest_value_in_masked_places(vocab, dtype, words, heat):
    """Masks of the type's lowest value, which f32 does not hold in other units: in half
    of a row's logits, in all of them, in a word's, in some of a teacher's words, in
    all of them."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(vocab + words)
    x = (3 * torch.randn(5, vocab, generator=g)).to(dtype)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:words] for _ in range(5)])
    top = torch.randn(5, words, generator=g).to(dtype)
    masked = torch.rand(vocab, generator=g) < 0.5
    masked[ids[0]] = False
    x[0, masked] = low
    x[1] = low
    top[2, 0] = top[2].min() - 1
    x[2, ids[2, 0]] = low
    top[3, words // 2:] = low
    top[4] = low
    x, ids, top = x.cuda().requires_grad_(), ids.cuda(), top.cuda()
    out = L.distillation_loss(x, ids, top, temperature=heat, reduction="none")
    got = torch.autograd.grad(out.sum(), x)[0]
    z = x.detach().to(F64)
    q = torch.zeros(5, vocab, dtype=F64, device="cuda").scatter_(1, ids, torch.softmax(top.to(F64) / heat, 1))
    ones = torch.ones(5, dtype=F64, device="cuda")
    want, dz, c = reference(z, q, ones != 0, ones, heat, "none")
    top_z = torch.where(z < -1e30, 0.0, z).abs().max().item() / heat
    rel = 2.0 ** -20 + 4 * 2.0 ** -24 * (top_z + 20)
    tol = rel * heat ** 2 * (want.abs() / heat ** 2 + math.log(2 * vocab) + top_z)
    assert ((out.detach().to(F64) - want).abs() <= tol).all()
    tol = 8 * rel * (dz.abs() + c * q) + (2.0 ** -8 if dtype == BF else 2.0 ** -23) * dz.abs() + 1e-38
    err = (got.to(F64) - dz).abs()
    assert (err <= tol).all(), (err / tol).max()
    again = torch.autograd.grad(L.distillation_loss(x, ids, top, temperature=heat, reduction="none").sum(), x,
                                create_graph=True)[0]
    # f32 operations: z / T and their sums round like the operator's
    assert ((again.to(F64) - dz).abs() <= tol).all()


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_upstream_nan_in_rows_that_do_not_count(op):
    """A masked mean's where() sends NaN or infinity to rows of weight 0."""
    h, w = operands(40, 64, 900, BF)
    ids, top = teacher_of(40, 900, 5, True)
    y = labels_of(40, 900, 0.2)
    weight = rand(40, seed=4).abs() + 0.5
    weight[::3] = 0
    x = (3 * rand(40, 900, seed=1)).to(BF)
    leaves = (x,) if op == "kept" else (h, w)
    for t in leaves:
        t.requires_grad_()
    each = L.linear_cross_entropy(h, w, y, weight, reduction="none") if op == "entropy" else (
        L.linear_distillation(h, w, ids, top, weight, reduction="none") if op == "teacher" else
        L.distillation_loss(x, ids, top, weight, reduction="none"))
    g, dead = rand(40, seed=2), weight == 0
    want = torch.autograd.grad(each, leaves, torch.where(dead, 0.0, g), retain_graph=True)
    for value in (math.nan, math.inf):
        got = torch.autograd.grad(each, leaves, torch.where(dead, value, g), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("op", ["entropy", "kept"])
def test_forward_and_backward_in_two_graphs(op):
    """The backward's graph, replayed twice behind one replay of the forward's, gives
    the same gradients twice."""
    h, w = operands(130, 128, 2000, BF)
    ids, top = teacher_of(130, 2000, 8, True)
    y = labels_of(130, 2000, 0.2)
    x = (3 * rand(130, 2000, seed=1)).to(BF)
    factor = torch.tensor(2.0, device="cuda")
    leaves = (x,) if op == "kept" else (h, w)
    for t in leaves:
        t.requires_grad_()

    def forward():
        return L.distillation_loss(x, ids, top) if op == "kept" else L.linear_cross_entropy(h, w, y)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(forward(), leaves, factor)
        torch.cuda.synchronize()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first, stream=side):
            loss = forward()
        with torch.cuda.graph(second, pool=first.pool(), stream=side):
            got = torch.autograd.grad(loss, leaves, factor)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_((t.float() * (0.9 + 0.1 * i)).to(BF))
        want = torch.autograd.grad(forward(), leaves, factor)
        first.replay()
        for _ in range(2):
            second.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_weight_rows_far_apart():
    """A view whose rows' pitch passes what the products address: a copy of it."""
    vocab, d = 131100, 2048
    w = torch.empty(vocab, 4 * d, dtype=BF, device="cuda")[:, :d].copy_(rand(vocab, d, seed=1) / 40)
    h, y = rand(3, d, seed=2).to(BF), torch.tensor([5, vocab - 1, 70000], device="cuda")
    assert torch.equal(L.linear_cross_entropy(h, w, y, reduction="none"),
                       L.linear_cross_entropy(h, w.contiguous(), y, reduction="none"))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_that_overlap(dtype):
    """Expanded rows and windows of one buffer."""
    base = rand(400, seed=3).to(dtype)
    w = operands(1, 30, 300, dtype)[1].requires_grad_()
    y = labels_of(40, 300, 0.1)
    for h in (base[:30].expand(40, 30), base.as_strided((40, 30), (5, 1), 3), base.as_strided((40, 30), (1, 7))):
        out, same = L.linear_cross_entropy(h, w, y), L.linear_cross_entropy(h.contiguous(), w, y)
        assert torch.equal(out, same)
        assert torch.equal(*(torch.autograd.grad(t, w)[0] for t in (out, same)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [7001, 12000, 20001, 40003, 80001])
def test_distillation_loss_of_other_widths(vocab, dtype):
    """Row widths between those of test_distillation_loss: other shares of a row in
    registers and LDS."""
    test_distillation_loss(3, vocab, dtype, 20, 2.0, True, "mean")
    test_distillation_loss(3, vocab, dtype, 300, 0.7, False, "none")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [5, 1003, 50021])
def test_rows_at_any_offset(vocab, dtype):
    """Views whose rows start anywhere in a 16-byte chunk give what copies give."""
    x = (3 * rand(4, vocab, seed=1)).to(dtype)
    ids, top = teacher_of(4, vocab, 6, False)
    want = None
    for ahead in range(9):
        v = torch.zeros(4, vocab + 11, dtype=dtype, device="cuda")[:, ahead:ahead + vocab].copy_(x).requires_grad_()
        out = L.distillation_loss(v, ids, top, reduction="none")
        got = (out.detach(), torch.autograd.grad(out.sum(), v)[0])
        want = want or got
        # the sum's order goes by the chunks: 2^-20 of the terms, as everywhere here
        assert torch.allclose(got[0], want[0], rtol=2.0 ** -20, atol=2.0 ** -20 * math.log(2 * vocab))
        step = 2.0 ** -7 if dtype == BF else 2.0 ** -20  # one bf16 step where the f32 values differ
        assert ((got[1] - want[1]).abs().float() <= step * want[1].abs().float() + 2.0 ** -20 * 2).all()


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("up", [0, 64, 4096])
def test_loss_of_logits_that_all_are_large(rows, up):
    """What all of a row's logits share leaves no rounding in its loss.  Logits are exact
    here: up, and -16 to 2 in steps of 1/8."""
    vocab = 500
    h, w = torch.zeros(rows, 64, device="cuda"), torch.zeros(vocab, 64, device="cuda")
    h[:, 0], h[:, 1] = 1, 1 + torch.arange(rows, device="cuda") % 2
    w[:, 0], w[:, 1] = up, -(torch.arange(vocab, device="cuda") * 37 % 65) / 8
    w[77, 1] = 1
    y = torch.full((rows,), 77, device="cuda")
    h, w = h.to(BF), w.to(BF)
    want = -torch.log_softmax(h.to(F64) @ w.to(F64).t(), -1)[:, 77]
    # in units of log2: a logit's distance from the slab's reference, at most 18 log2(e) + 1,
    # rounded and scaled by a rounded log2(e), twice; sum, exponential and logarithm
    tol = math.log(2) * (4 * 27 * 2.0 ** -25 + 2.0 ** -21)
    out = L.linear_cross_entropy(h, w, y, reduction="none").to(F64)
    assert ((out - want).abs() <= tol).all(), (out - want).abs().max()
    mean = L.linear_cross_entropy(h.requires_grad_(), w, y)
    assert abs(mean.item() - want.mean().item()) <= tol + 2.0 ** -24 * want.max().item()


@pytest.mark.parametrize("rows", [1, 7, 16])
@pytest.mark.parametrize("d", [1, 7, 31, 100, 250, 1500, 4093])
def test_few_rows_of_any_hidden_size(rows, d):
    """Losses alone of up to 16 rows; what lies behind a row's end is NaN."""
    vocab = 1003
    h, w = operands(rows, d, vocab, BF, seed=d)
    hd, wd = h.to(F64), w.to(F64)
    wide = [torch.full((t.shape[0], -(-d // 8) * 8), math.nan, dtype=BF, device="cuda") for t in (h, w)]
    h, w = (b[:, :d].copy_(t) for b, t in zip(wide, (h, w)))
    y = labels_of(rows, vocab, 0.2)
    label = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    label[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    z, ones = hd @ wd.t(), torch.ones(rows, device="cuda")
    want, _, _ = reference(z, label, y != -100, ones.to(F64), 1.0, "none")
    out = L.linear_cross_entropy(h, w, y, reduction="none")
    check(out, want, (None, None), (hd, wd), z, z, label, logit_error(hd, wd), 1.0, 1.0, ones)
    ids, top = teacher_of(rows, vocab, 9, False)
    q, some = shares(ids, top, vocab, 1.5)
    want, _, _ = reference(z, q, some, ones.to(F64), 1.5, "none")
    check(L.linear_distillation(h, w, ids, top, temperature=1.5, reduction="none"), want, (None, None), (hd, wd), z, z, q,
          logit_error(hd, wd), 1.5, 1.0, ones)


@pytest.mark.parametrize("rows,d,vocab", [(5, 100, 700), (20, 250, 700), (300, 1500, 1003), (40, 7, 300)])
def test_nan_behind_the_rows(rows, d, vocab):
    """Gradients of views into wider buffers that hold NaN."""
    h, w = operands(rows, d, vocab, BF)
    y = labels_of(rows, vocab, 0.2)
    wide = [torch.full((t.shape[0], -(-d // 8) * 8 + 8), math.nan, dtype=BF, device="cuda") for t in (h, w)]
    views = [b[:, :d].copy_(t).requires_grad_() for b, t in zip(wide, (h, w))]
    out, same = L.linear_cross_entropy(*views, y), L.linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), y)
    assert torch.equal(out, same)
    for a, b in zip(torch.autograd.grad(out, views), torch.autograd.grad(same, (h, w))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,d,vocab", [(2, 64, 40000), (16, 100, 65536), (3, 4096, 40000), (5, 96, 65600)])
def test_few_rows_of_wide_vocabularies(rows, d, vocab):
    """Losses alone on both sides of where few rows go through tiles."""
    h, w = operands(rows, d, vocab, BF)
    hd, wd = h.to(F64), w.to(F64)
    y = labels_of(rows, vocab, 0.0)
    label = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    label[torch.arange(rows, device="cuda"), y] = 1
    z, ones = hd @ wd.t(), torch.ones(rows, device="cuda")
    want, _, _ = reference(z, label, y >= 0, ones.to(F64), 1.0, "none")
    out = L.linear_cross_entropy(h, w, y, reduction="none")
    check(out, want, (None, None), (hd, wd), z, z, label, logit_error(hd, wd), 1.0, 1.0, ones)


@pytest.mark.parametrize("rows,words", [(8193, 0), (8500, 0), (8300, 7)])
def test_rows_in_more_pieces(rows, words):
    """A second piece of the rows, of one and of some."""
    d, vocab = 64, 128256
    h, w = operands(rows, d, vocab, BF)
    h, w = h.requires_grad_(), w.requires_grad_()
    y = labels_of(rows, vocab, 0.2)
    y[-1] = 5
    one = torch.ones(rows, dtype=F64, device="cuda")
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    if words:
        ids, top = teacher_of(rows, vocab, words, False)
        out = L.linear_distillation(h, w, ids, top)
        q, some = shares(ids, top, vocab, 1.0)
    else:
        out = L.linear_cross_entropy(h, w, y)
        q, some = torch.zeros(rows, vocab, dtype=F64, device="cuda"), y != -100
        q[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    got = torch.autograd.grad(out, (h, w))
    want, dz, c = reference(hd @ wd.t(), q, some, one, 1.0, "mean")
    check(out.detach(), want, got, (hd, wd), dz, c, q, logit_error(hd, wd), 1.0, 1.0, one)


def test_no_piece_passes_the_products_offsets():
    """Sizes of the workspace go by the pieces: rows and words of any size have one."""
    from moc_amd import _native as N
    for vocab in (1, 63, 32000, 65536, 128256, 1 << 21):
        for rows in (1, 257, 16384, 1 << 17):
            need = N.query("moc_linear_loss_workspace_size", N.MOC_BF16, rows, 64, vocab, 0, 1)
            assert 0 < need < (1 << 31) + 2 * vocab * 64 * 4 + vocab * 64 * 2 + rows * 64 * 2 + (
                (1 << 31) // (vocab * 2) + 256) * (vocab // 64 + 2) * 8 + (1 << 24) + rows * 8


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_two_threads_on_one_stream(op, dtype):
    """Calls whose launches mix on a stream: products split along K, teachers, sums."""
    import threading

    rows, d, vocab, turns = (777, 512, 9000, 25) if dtype == BF else (96, 64, 3000, 25)
    sets = []
    for i in range(2):
        h, w = operands(rows, d, vocab, dtype, seed=20 * i)
        ids, top = teacher_of(rows, vocab, 5 + i, True)
        x = (3 * rand(rows, vocab, seed=i)).to(dtype)
        sets.append((h.requires_grad_(), w.requires_grad_(), x.requires_grad_(), labels_of(rows, vocab, 0.2, seed=i), ids,
                     top))

    def step(h, w, x, y, ids, top):
        if op == "kept":
            loss = L.distillation_loss(x, ids, top)
            return (loss.detach(), *torch.autograd.grad(loss, x))
        loss = L.linear_cross_entropy(h, w, y) if op == "entropy" else L.linear_distillation(h, w, ids, top)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    wrong = [None, None]

    def work(i):
        wrong[i] = [t for t in range(turns) if not all(torch.equal(a, b) for a, b in zip(step(*sets[i]), want[i]))]

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [[], []]


@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_two_streams_at_once(op):
    sets = []
    for i in range(2):
        h, w = operands(700, 256, 9000, BF, seed=20 * i)
        ids, top = teacher_of(700, 9000, 5 + i, True)
        x = (3 * rand(700, 9000, seed=i)).to(BF)
        sets.append((h.requires_grad_(), w.requires_grad_(), x.requires_grad_(), labels_of(700, 9000, 0.2, seed=i), ids, top))

    def step(h, w, x, y, ids, top):
        if op == "kept":
            loss = L.distillation_loss(x, ids, top)
            return (loss.detach(), *torch.autograd.grad(loss, x))
        loss = L.linear_cross_entropy(h, w, y) if op == "entropy" else L.linear_distillation(h, w, ids, top)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    want = [step(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(step(*s))
    torch.cuda.synchronize()
    for i, one in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(one, want[i % 2])), i


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("op", ["entropy", "teacher", "kept"])
def test_captured_rows(op, dtype):
    """reduction="none" with its backward in a graph, and losses alone."""
    h, w = operands(40, 64, 2000, dtype)
    ids, top = teacher_of(40, 2000, 8, True)
    y, g = labels_of(40, 2000, 0.2), rand(40, seed=3)
    x = (3 * rand(40, 2000, seed=1)).to(dtype)
    leaves = (x,) if op == "kept" else (h, w)
    for t in leaves:
        t.requires_grad_()

    def loss(reduction):
        return L.linear_cross_entropy(h, w, y, reduction=reduction) if op == "entropy" else (
            L.linear_distillation(h, w, ids, top, reduction=reduction) if op == "teacher" else
            L.distillation_loss(x, ids, top, reduction=reduction))

    def step():
        each = loss("none")
        with torch.no_grad():
            alone = loss("mean")
        return (each.detach(), alone, *torch.autograd.grad(each, leaves, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for t in leaves:
                t.copy_((t.float() * (0.9 + 0.1 * i)).to(dtype))
            y.copy_(labels_of(40, 2000, 0.3, seed=i))
            g.copy_(rand(40, seed=5 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


@pytest.mark.parametrize("rows,d,vocab", [(3, 1, 7), (20, 30, 1001), (129, 333, 4099), (1, 101, 50), (2, 6, 5), (64, 9, 4),
                                          (0, 5, 30)])
@pytest.mark.parametrize("only", ["both", "hidden", "weight", "losses"])
def test_f32_of_odd_sizes(rows, d, vocab, only):
    """Hidden sizes and vocabularies that are no multiple of 4, in f32, and leading
    dimensions; rows that lie apart."""
    h, w = operands(rows, d, vocab, F32) if rows else (torch.zeros(0, d, device="cuda"), operands(1, d, vocab, F32)[1])
    h = torch.cat([h, torch.full_like(h, math.nan)], 1)[:, :d].view(1, rows, d)
    y = labels_of(rows, vocab, 0.2)
    if rows:
        y[0] = vocab - 1
    h.requires_grad_(only in ("both", "hidden"))
    w.requires_grad_(only in ("both", "weight"))
    leaves = [t for t in (h, w) if t.requires_grad]
    out = L.linear_cross_entropy(h, w, y.view(1, rows), reduction="sum")
    got = iter(torch.autograd.grad(out, leaves) if leaves else ())
    got = [next(got) if t.requires_grad else None for t in (h, w)]
    assert got[0] is None or got[0].shape == h.shape
    if not rows:
        assert out == 0 and (got[1] is None or (got[1] == 0).all())
        return
    hd, wd = h.detach().view(rows, d).to(F64), w.detach().to(F64)
    q = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    q[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    one = torch.ones(rows, dtype=F64, device="cuda")
    want, dz, c = reference(hd @ wd.t(), q, y != -100, one, 1.0, "sum")
    got[0] = None if got[0] is None else got[0].view(rows, d)
    check(out.detach(), want, got, (hd, wd), dz, c, q, logit_error(hd, wd), 1.0, 1.0, one)


@pytest.mark.parametrize("rows,vocab", [(1, 2), (700, 1), (700, 2), (700, 3), (65, 6)])
def test_f32_of_a_few_words(rows, vocab):
    test_f32_of_odd_sizes(rows, 40, vocab, "both")
    test_f32_of_odd_sizes(rows, 64, vocab, "hidden")


def test_f32_weight_beyond_32_bit_offsets():
    """2.4 GB of f32 weight: dhidden from parts of the words."""
    rows, d, vocab = 9, 4096, 146001
    h, w = operands(rows, d, vocab, F32)
    h.requires_grad_()
    y = torch.tensor([5, vocab - 1, 131071, 131072, -100, 7, 9, 70000, 145999], device="cuda")
    out = L.linear_cross_entropy(h, w, y, reduction="sum")
    got = torch.autograd.grad(out, h)[0]
    hd = h.detach().to(F64)
    z = torch.cat([hd @ part.to(F64).t() for part in w.split(20000)], 1)
    q = torch.zeros(rows, vocab, dtype=F64, device="cuda")
    q[torch.arange(rows, device="cuda"), y.clamp(min=0)] = 1
    one = torch.ones(rows, dtype=F64, device="cuda")
    want, dz, c = reference(z, q, y != -100, one, 1.0, "sum")
    check(out.detach(), want, (got, None), (hd, w.to(F64)), dz, c, q, logit_error(hd, w.to(F64)), 1.0, 1.0, one)


@pytest.mark.parametrize("rows,cols,ahead", [(1, 1, 1), (3, 7, 0), (5, 8, 3), (70000, 12, 1), (9, 511, 2), (66, 513, 7),
                                             (4, 65533, 5), (1000, 1500, 4), (1, 4099, 0)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_padding_copy(rows, cols, ahead, dtype):
    """Rows at any address into aligned ones: every value, zeros behind them, nothing else."""
    from moc_amd import _native as N
    from moc_amd import kernels as K
    x = rand(rows, cols + ahead, seed=cols).to(dtype)[:, ahead:]
    pitch = K.row_pitch(cols, dtype)
    for width in (pitch, K.round_up(cols, 8) + 8):
        out = torch.full((rows + 1, K.round_up(cols, 8) + 24 + pitch), 7.0, dtype=dtype, device="cuda")
        out = out[:, :out.shape[1] // 8 * 8]
        ld = out.stride(0) // 8 * 8
        if ld != out.stride(0):
            out = torch.full((rows + 1, ld), 7.0, dtype=dtype, device="cuda")
        N.call("moc_copy_pad_2d", N.dtype_code(dtype), x.data_ptr(), rows, cols, x.stride(0) if rows > 1 else cols,
               out.data_ptr(), ld, width, N.stream_of(x))
        assert torch.equal(out[:rows, :cols], x)
        assert (out[:rows, cols:width] == 0).all() and (out[:rows, width:] == 7).all() and (out[rows:] == 7).all()


@pytest.mark.parametrize("rows", [1, 5, 16])
@pytest.mark.parametrize("d,vocab", [(64, 1000), (100, 4099), (1500, 777), (2048, 8190), (4093, 1003), (512, 65600)])
@pytest.mark.parametrize("op", ["entropy", "teacher"])
def test_gradients_of_few_rows(rows, d, vocab, op):
    h, w = operands(rows, d, vocab, BF, seed=d)
    h, w = h.requires_grad_(), w.requires_grad_()
    one = torch.ones(rows, dtype=F64, device="cuda")
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    if op == "teacher":
        ids, top = teacher_of(rows, vocab, 20, False)
        q, some = shares(ids, top, vocab, 2.0)
        out, heat = L.linear_distillation(h, w, ids, top, temperature=2.0), 2.0
    else:
        y = labels_of(rows, vocab, 0.0)
        q, some = torch.zeros(rows, vocab, dtype=F64, device="cuda"), y >= 0
        q[torch.arange(rows, device="cuda"), y] = 1
        out, heat = L.linear_cross_entropy(h, w, y), 1.0
    got = torch.autograd.grad(out, (h, w))
    want, dz, c = reference(hd @ wd.t(), q, some, one, heat, "mean")
    check(out.detach(), want, got, (hd, wd), dz, c, q, logit_error(hd, wd), heat, 1.0, one)
