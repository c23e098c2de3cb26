"""LLaMAModel.loss and .distill in f32 without autocast and in bf16 under it: the losses'
kernels, not the logits of all positions."""
import pytest
import torch

from moc_amd import model as M
from test_gpu_model_loss import batch, model_of

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


@pytest.fixture
def taken(monkeypatch):
    """The hidden rows that the linear losses were called with."""
    rows = []
    for name in ("linear_cross_entropy", "linear_distillation"):
        def spy(hidden, *args, call=getattr(M, name), **kwargs):
            rows.append(hidden)
            return call(hidden, *args, **kwargs)
        monkeypatch.setattr(M, name, spy)
    return rows


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("ffn", ["dense", "moc_gcp"])
def test_f32_step(ffn, tied, taken):
    m = model_of(ffn, F32, tied)
    ids, labels = batch()
    weight = torch.rand(3, 33, device="cuda")
    weight[0, 5] = 0
    loss = m.loss(ids, labels, weight)
    x, = taken
    assert x.dtype == F32
    got = torch.autograd.grad(loss, [x, *m.parameters()], retain_graph=True)
    w = m._head_weight().detach().to(F64).requires_grad_()
    xd = x.detach().to(F64).requires_grad_()
    z = xd @ w.t()
    on = labels[:, 1:] != -100
    each = -torch.log_softmax(z[:, :-1], -1)[on].gather(1, labels[:, 1:][on][:, None])[:, 0]
    share = weight[:, :-1][on].to(F64)
    want = (each * share).sum() / share.sum()
    s = (xd.detach().abs() @ w.detach().abs().t()).amax().item()
    # f32 sums of 256 products, exponentials and a sum over the vocabulary
    z_err = 66 * 2.0 ** -24 * s
    assert abs(loss.item() - want.item()) <= 2 * z_err + 2.0 ** -20 * 8
    dx = torch.autograd.grad(want, xd)[0]
    # p's relative error and sums of 1003 terms, of which a row's weigh 2 at most
    size = 2 * weight.max().item() / share.sum().item() * w.detach().abs().max().item()
    assert (got[0].to(F64) - dx).abs().max() <= (4 * z_err + 130 * 2.0 ** -24 + 2.0 ** -20) * size
    assert not got[0][0, 5].any()
    for (name, _), g in zip(m.named_parameters(), got[1:]):
        assert g.dtype == F32 and torch.isfinite(g).all() and g.any(), name
    assert abs(m.loss(ids, labels).item() - m(ids, labels)[1].item()) <= 2 * 2 * z_err + 2.0 ** -20 * 16


def test_f32_distill(taken):
    m = model_of("moc_gcp", F32, False)
    ids, _ = batch()
    with torch.no_grad():
        top = model_of("dense", F32, False, seed=1)(ids).topk(20)
    loss = m.distill(ids, top.indices, top.values, temperature=2.0)
    x, = taken
    xd, w = (t.detach().to(F64) for t in (x, m._head_weight()))
    z = xd @ w.t()
    log_q = torch.log_softmax(top.values.to(F64) / 2, -1)
    want = 4 * (log_q.exp() * (log_q - torch.log_softmax(z / 2, -1).gather(-1, top.indices))).sum(-1).mean()
    s = (xd.abs() @ w.abs().t()).amax().item()
    assert abs(loss.item() - want.item()) <= 2 * 2 * 66 * 2.0 ** -24 * s + 2.0 ** -20 * 4 * 8
    loss.backward()
    for name, p in m.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name


def test_bf16_under_autocast(taken):
    m = model_of("dense", BF, False)
    ids, labels = batch()
    with torch.autocast("cuda", dtype=BF):
        loss = m.loss(ids, labels)
        m.distill(ids, ids[..., None], torch.zeros(3, 33, 1, device="cuda"))
    assert [x.dtype for x in taken] == [BF, BF]
    z = taken[0].detach().to(F64) @ m._head_weight().detach().to(F64).t()
    on = labels[:, 1:] != -100
    want = -torch.log_softmax(z[:, :-1], -1)[on].gather(1, labels[:, 1:][on][:, None]).mean()
    s = (taken[0].detach().to(F64).abs() @ m._head_weight().detach().to(F64).abs().t()).amax().item()
    assert abs(loss.item() - want.item()) <= 2 * 66 * 2.0 ** -24 * s + 2.0 ** -20 * 8


def test_other_types_take_the_logits(taken):
    m = model_of("dense", torch.float16, False)
    ids, labels = batch()
    assert torch.isfinite(m.loss(ids, labels)) and not taken
    with pytest.raises(ValueError, match="plain LM head"):
        m.distill(ids, ids[..., None], torch.zeros(3, 33, 1, device="cuda"))
