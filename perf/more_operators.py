"""What the losses over a vocabulary are timed on.

Three operators of training and evaluation at the end of a model:

  entropy    losses.linear_cross_entropy: softmax cross entropy of hidden rows
             against labels through the head's weight, without kept logits;
             the loss with the gradients of hidden rows and weight, or the
             rows' losses alone (evaluation, log-probabilities of an answer);
  teacher    losses.linear_distillation: the divergence from a teacher's top
             logits, through the head's weight in the same way;
  kept       losses.distillation_loss: the same divergence of logits that the
             program holds, with their gradient.

Hidden sizes and the vocabulary of 32000 are those of the presets and the decode
model, 256 positions the presets' sequence; larger vocabularies, odd sizes and the
teacher's number of words are generic.  Sizes go by the case alone, contents by the seed.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32
TYPES = {"bf16": BF16, "f32": F32}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # The log-probability of one answered token: the launches and one read of the weight.
        dict(name="score_1", op="entropy", rows=1, hidden=2048, vocab=32000, train=False, masked=0.0, weighted=False),
        # The tokens of a batched step scored, a large vocabulary.
        dict(name="score_16", op="entropy", rows=16, hidden=1024, vocab=128256, train=False, masked=0.0, weighted=False),
        # Evaluation on text, odd sizes all through; 130m's hidden size.
        dict(name="evaluate", op="entropy", rows=4099, hidden=768, vocab=50021, train=False, masked=0.0, weighted=False),
        # A step of the 60m preset on two sequences.
        dict(name="step_60m", op="entropy", rows=512, hidden=512, vocab=32000, train=True, masked=0.0, weighted=False),
        # Answers behind prompts, at the 350m shape: the prompts' labels are masked, tokens weighted.
        dict(name="answers_350m", op="entropy", rows=8192, hidden=1024, vocab=32000, train=True, masked=0.4,
             weighted=True),
        # A step of the 1b preset on 64 sequences.
        dict(name="step_1b", op="entropy", rows=16384, hidden=2048, vocab=32000, train=True, masked=0.0, weighted=False),
        # The same work over a large vocabulary.
        dict(name="step_wide", op="entropy", rows=4096, hidden=2048, vocab=128256, train=True, masked=0.0,
             weighted=False),
        # A ragged batch of short answers against few words of a teacher.
        dict(name="teacher_60m", op="teacher", rows=777, hidden=512, vocab=32000, words=16, heat=1.0, ragged=True,
             weighted=True),
        # A distillation step at the 350m shape.
        dict(name="teacher_350m", op="teacher", rows=8192, hidden=1024, vocab=32000, words=64, heat=2.0, ragged=False,
             weighted=False),
        # Logits of one sequence.
        dict(name="kept_256", op="kept", rows=256, vocab=32000, words=20, heat=1.0, logits="bf16", ragged=False,
             weighted=False),
        # Logits of a step, bf16 as a head leaves them.
        dict(name="kept_8192", op="kept", rows=8192, vocab=32000, words=64, heat=2.0, logits="bf16", ragged=True,
             weighted=False),
        # f32 logits of a large vocabulary, an odd number of words.
        dict(name="kept_wide", op="kept", rows=2048, vocab=128256, words=101, heat=1.5, logits="f32", ragged=False,
             weighted=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))


def draw(rng):
    op = rng.choice(("entropy", "entropy", "teacher", "kept"))
    case = dict(op=op, vocab=_log(rng, 500, 128256))
    if op == "kept":
        case["rows"] = _log(rng, 1, min(16384, (1 << 28) // case["vocab"]))
        case["logits"] = rng.choice(("bf16", "f32"))
    else:
        case["hidden"] = rng.choice((64, 256, 512, 768, 1024, 2048, 4096, 100, 1500))
        case["rows"] = _log(rng, 1, min(16384, (1 << 40) // (case["vocab"] * case["hidden"])))
    if op == "entropy":
        return dict(case, train=rng.random() < 0.6, masked=rng.choice((0.0, 0.0, 0.3, 0.9)),
                    weighted=rng.random() < 0.3)
    return dict(case, words=min(case["vocab"], _log(rng, 1, 200)), heat=rng.choice((1.0, 1.0, 2.0, 0.7)),
                ragged=rng.random() < 0.5, weighted=rng.random() < 0.3)


# -------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    rows, vocab = case["rows"], case["vocab"]
    s = SimpleNamespace(op=case["op"], train=case.get("train", True), heat=case.get("heat", 1.0))
    s.row_weight = 0.5 + uniform(rows) if case["weighted"] else None
    # the word a row is likely to be followed by; common words more often than rare ones
    likely = (vocab * uniform(rows) ** 3).long().clamp(max=vocab - 1)
    sure = 6 * uniform(rows, 1)
    if s.op == "entropy":
        s.labels = torch.where(uniform(rows) < case["masked"], -100, likely)
        if case["masked"]:
            s.labels[0] = likely[0]  # a label at least
    else:
        words = case["words"]
        # distinct words, one of each stretch of the vocabulary, the likely one among them
        step = vocab // words
        ids = torch.arange(words, device="cuda") * step + (uniform(rows, words) * step).long()
        ids[:, 0] += likely - ids[:, 0]
        ids[:, 1:] = (ids[:, 1:] + likely[:, None] - likely[:, None] % max(step, 1)) % vocab
        twice = ids[:, 1:] == ids[:, :1]
        ids[:, 1:] = torch.where(twice, -1, ids[:, 1:])
        top = torch.sort(3 * normal(rows, words), -1, descending=True).values
        top[:, :1] += sure
        s.ids, s.top = ids.to(I32), top + 8
        if case["ragged"]:  # rows with fewer words, some with none
            held = torch.where(uniform(rows) < 0.2, 0, 1 + (uniform(rows) * words).long())
            held[0] = words
            s.ids = torch.where(torch.arange(words, device="cuda") < held[:, None], s.ids, -1)
    if s.op == "kept":
        x = 2.5 * normal(rows, vocab)
        x[torch.arange(rows, device="cuda"), likely] += sure[:, 0]
        s.logits = x.to(TYPES[case["logits"]]).requires_grad_()
        return s
    hidden = case["hidden"]
    # logits of standard deviation 2 around the likely word's
    weight = (normal(vocab, hidden) * (2 / math.sqrt(hidden))).to(BF16)
    x = normal(rows, hidden) + 0.5 * sure * weight[likely].float()
    s.hidden, s.weight = x.to(BF16).requires_grad_(s.train), weight.requires_grad_(s.train)
    return s


# ---------------------------------------------------------------- plain forms
def _softmax(z):
    e = torch.exp(z - z.amax(-1, keepdim=True))
    total = e.sum(-1, keepdim=True)
    return e / total, z.amax(-1) + torch.log(total[:, 0])


def _entropy_plain(s):
    h, w = s.hidden.detach().float(), s.weight.detach().float()
    z = h @ w.t()
    p, lse = _softmax(z)
    at = torch.arange(h.shape[0], device="cuda")
    scored = s.labels != -100
    label = torch.where(scored, s.labels, 0)
    loss = torch.where(scored, lse - z[at, label], 0.0)
    if not s.train:
        return loss
    share = scored.float() if s.row_weight is None else torch.where(scored, s.row_weight, 0.0)
    share = share / share.sum()
    p[at, label] -= 1
    p = p * share[:, None]
    return {"loss": (loss * share).sum(), "hidden": (p @ w).to(BF16), "weight": (p.t() @ h).to(BF16)}


def _teacher(s):
    """Words, their shares, the rows' weights (0: a row without words)."""
    there = s.ids >= 0
    some = there.any(-1)
    x = torch.where(there, s.top.float() / s.heat, -math.inf)
    x = torch.where(some[:, None], x, 0.0)
    q = torch.where(there, torch.exp(x - x.amax(-1, keepdim=True)), 0.0)
    q = q / q.sum(-1, keepdim=True).clamp(min=1e-30)
    share = some.float() if s.row_weight is None else torch.where(some, s.row_weight, 0.0)
    return torch.where(there, s.ids, 0).long(), q, share / share.sum()


def _divergence_plain(s, z):
    """The loss and its gradient by the logits z in 32 bits."""
    ids, q, share = _teacher(s)
    p, lse = _softmax(z / s.heat)
    log_p = torch.gather(z, 1, ids) / s.heat - lse[:, None]
    rows = torch.where(q > 0, q * (torch.log(q.clamp(min=1e-30)) - log_p), 0.0).sum(-1)
    p.scatter_add_(1, ids, -q)
    return s.heat ** 2 * (rows * share).sum(), p * (s.heat * share)[:, None]


def _teacher_plain(s):
    h, w = s.hidden.detach().float(), s.weight.detach().float()
    loss, dz = _divergence_plain(s, h @ w.t())
    return {"loss": loss, "hidden": (dz @ w).to(BF16), "weight": (dz.t() @ h).to(BF16)}


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        from moc_amd import losses
        if s.op == "kept":
            loss = losses.distillation_loss(s.logits, s.ids, s.top, s.row_weight, temperature=s.heat)
            return {"loss": loss.detach(), "logits": torch.autograd.grad(loss, s.logits)[0]}
        if s.op == "entropy" and not s.train:
            return losses.linear_cross_entropy(s.hidden, s.weight, s.labels, reduction="none")
        if s.op == "entropy":
            loss = losses.linear_cross_entropy(s.hidden, s.weight, s.labels, s.row_weight)
        else:
            loss = losses.linear_distillation(s.hidden, s.weight, s.ids, s.top, s.row_weight, temperature=s.heat)
        hidden, weight = torch.autograd.grad(loss, (s.hidden, s.weight))
        return {"loss": loss.detach(), "hidden": hidden, "weight": weight}
    if s.op == "entropy":
        return _entropy_plain(s)
    if s.op == "teacher":
        return _teacher_plain(s)
    loss, dz = _divergence_plain(s, s.logits.detach().float())
    return {"loss": loss, "logits": dz.to(s.logits.dtype)}


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    targets = rows * (8 * case["words"] if "words" in case else 8) + 4 * rows * case["weighted"]
    if case["op"] == "kept":
        size = 2 if case["logits"] == "bf16" else 4
        return {"bytes": 2 * size * rows * vocab + targets, "flops": 8 * rows * vocab}
    both = 2 * case["hidden"] * (rows + vocab)  # hidden rows and the weight
    product = 2 * rows * vocab * case["hidden"]
    if not case.get("train", True):
        return {"bytes": both + targets + 4 * rows, "flops": product}
    return {"bytes": 2 * both + targets, "flops": 3 * product}


# ------------------------------------------------------------- from 64 bits
def exact(case, seed):
    """Losses by log_softmax in 64 bits, gradients by differentiation."""
    s = prepare(case, seed)
    rows, vocab = case["rows"], case["vocab"]
    leaves = [s.logits] if s.op == "kept" else [s.hidden, s.weight]
    leaves = [t.detach().double().requires_grad_(s.train) for t in leaves]
    z = leaves[0] if s.op == "kept" else leaves[0] @ leaves[1].t()
    log_p = torch.log_softmax(z / s.heat, -1)
    weight = torch.ones(rows, dtype=F64, device="cuda") if s.row_weight is None else s.row_weight.double()
    if s.op == "entropy":
        picked = (s.labels != -100).nonzero()[:, 0]
        each = -log_p[picked, s.labels[picked]]
        if not s.train:
            return torch.zeros(rows, dtype=F64, device="cuda").index_put((picked,), each.detach())
    else:
        picked = (s.ids >= 0).any(1).nonzero()[:, 0]
        ids = s.ids[picked].long()
        log_q = torch.log_softmax((s.top[picked].double() / s.heat).masked_fill(ids < 0, -math.inf), -1)
        parts = log_q.exp() * (log_q - log_p[picked].gather(1, ids.clamp(min=0)))
        each = s.heat ** 2 * torch.where(ids < 0, 0.0, parts).sum(1)
    loss = (each * weight[picked]).sum() / weight[picked].sum()
    grads = torch.autograd.grad(loss, leaves)
    names = ["logits"] if s.op == "kept" else ["hidden", "weight"]
    return {"loss": loss.detach(), **dict(zip(names, grads))}
