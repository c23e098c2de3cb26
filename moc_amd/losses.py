"""Losses over a vocabulary: cross entropy against labels and the divergence from
a teacher's top logits (moc_amd/csrc/vocab_loss.hip).

    linear_cross_entropy(hidden, weight, labels)            the head's product and
    linear_distillation(hidden, weight, ids, top)           the loss as one operator
    distillation_loss(logits, ids, top)                     of logits already there

The first two never hold the logits of all rows: they exist for a piece of the rows
at a time (at most 2 GiB), and the gradients of hidden rows and weight are computed
in the forward pass, while the piece is there, so that a backward has nothing left to
do but the upstream factor.  A second backward of the same graph, and a backward
captured into a HIP graph without its forward, compute them again; reduction="none"
computes them in the backward, by the upstream gradient of each row.

Row r has a weight w_r (row_weight, 1 without), words with shares q (a label: one of
share 1) and logits z; with the temperature T, p = softmax(z / T),

    l_r = T^2 sum_i q_i (ln q_i - ln p_i)        (labels, T = 1: -ln p_label)

"mean" is sum w_r l_r / sum w_r, "sum" the sum and "none" w_r l_r for each row.  A row
of weight 0, one whose label is ignore_index and one without words count for nothing,
NaN in their hidden rows or logits included: they have loss and gradient 0 and are left
out of the mean, which is NaN where no row is left.  A label outside the vocabulary
gives NaN, as do NaN logits in rows that count.

Losses are f32.  Operands are bf16 or f32, or either under bf16 autocast, where the
products are those of bf16 casts and gradients come in the operands' own types.  An
upstream factor that is no power of two rounds bf16 gradients a second time.  A backward
with create_graph=True takes f32 tensor operations, with the logits of all rows.

Logits of bf16 products may be up to 2^22 temperatures in size.  Their gradients pass
through f16, with ranges of their own:
  gradients of logits, w_r / W (p - q) with W the largest finite row weight to a power of
    two, have all bits down to 2^-28, fewer below and none from 2^-39;
  hidden rows for dweight and the weight for dhidden are scaled by one power of two a
    tensor, so that channels far smaller than others are rounded: values below 2^-19 of
    hidden rows by up to 2^-27, below 2^-23 of a weight by up to 2^-31, or, where a
    tensor's largest is outside [2^-3, 2^13] and [2^-7, 2^9], values below 2^-32 of it by
    up to 2^-39 of it.  dweight of a channel of such values, and of a word whose p is as
    small in every row, has few bits or is 0.  (A few hundred rows: the weight stays bf16.)
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch

from . import _native as N
from . import kernels as K
from .block import graph_grads, plain

BF16, F32 = torch.bfloat16, torch.float32
REDUCTIONS = ("mean", "sum", "none")
COUNTER_BYTES = 4096  # MOC_GEMM_WS_COUNTER_BYTES
# Elements between two rows that the products' 32-bit offsets take: 256 rows, a tile and the
# fewest of a piece, within 2 GiB.
MOST_PITCH = 1 << 21


def linear_cross_entropy(hidden, weight, labels, row_weight=None, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """Cross entropy of the logits hidden @ weight.T against labels: hidden [..., d],
    weight [vocab, d], labels [...] (int64), row_weight [...] (f32)."""
    rows = _rows_of("linear_cross_entropy", hidden, labels, row_weight, reduction)
    targets = _Labels(labels.reshape(rows).contiguous(), _flat(row_weight, rows), int(ignore_index), reduction)
    return _linear("linear_cross_entropy", hidden, weight, targets)


def linear_distillation(hidden, weight, teacher_ids, teacher_logits, row_weight=None, *, temperature: float = 1.0,
                        reduction: str = "mean") -> torch.Tensor:
    """Divergence of softmax(hidden @ weight.T / temperature) from a teacher that is
    known by its top logits: teacher_ids [..., words] (int32 or int64) and
    teacher_logits [..., words] (bf16 or f32), up to 1024 words a row in any order; q =
    softmax(teacher_logits / temperature) over the words given.  An id outside the
    vocabulary (-1, say) or a logit of -infinity is no word, ids that stand twice in a
    row add up.  Teacher and row_weight get no gradient."""
    rows = _rows_of("linear_distillation", hidden, None, row_weight, reduction)
    targets = _teacher("linear_distillation", hidden, teacher_ids, teacher_logits, row_weight, rows, temperature,
                       reduction)
    return _linear("linear_distillation", hidden, weight, targets)


def distillation_loss(logits, teacher_ids, teacher_logits, row_weight=None, *, temperature: float = 1.0,
                      reduction: str = "mean") -> torch.Tensor:
    """linear_distillation of logits [..., vocab] (bf16 or f32) that are there already."""
    what = "distillation_loss"
    rows = _rows_of(what, logits, None, row_weight, reduction)
    if not 1 <= logits.shape[-1] <= 1 << 21:
        raise ValueError(f"{what}: a vocabulary of 1 to 2^21 words, got {logits.shape[-1]}")
    targets = _teacher(what, logits, teacher_ids, teacher_logits, row_weight, rows, temperature, reduction)
    _refuse_subclasses(what, logits, *targets.tensors())
    dev = N.one_device(logits, *targets.tensors())
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return _LogitsLoss.apply(targets, torch.is_grad_enabled(), logits, *targets.tensors())
    return _LogitsLoss.apply(targets, torch.is_grad_enabled(), logits, *targets.tensors())


# --------------------------------------------------------------------- targets
def _rows_of(what: str, x, labels, row_weight, reduction: str) -> int:
    if reduction not in REDUCTIONS:
        raise ValueError(f"{what}: reduction is one of {REDUCTIONS}, got {reduction!r}")
    if x.dim() < 1 or x.dtype not in (BF16, F32):
        raise ValueError(f"{what}: rows of bf16 or f32, got {x.dtype} {tuple(x.shape)}")
    lead = x.shape[:-1]
    if labels is not None and (labels.shape != lead or labels.dtype != torch.int64):
        raise ValueError(f"{what}: labels are int64 {tuple(lead)}, got {labels.dtype} {tuple(labels.shape)}")
    if row_weight is not None and (row_weight.shape != lead or row_weight.dtype != F32):
        raise ValueError(f"{what}: row_weight is f32 {tuple(lead)}, got {row_weight.dtype} {tuple(row_weight.shape)}")
    if row_weight is not None and row_weight.requires_grad:
        raise ValueError(f"{what}: row_weight has no gradient here")
    rows = math.prod(lead)
    if rows > 1 << 24:
        raise ValueError(f"{what}: up to 2^24 rows, got {rows}")
    return rows


def _refuse_subclasses(what: str, *tensors) -> None:
    if not plain(*(t for t in tensors if t is not None)):
        raise ValueError(f"{what}: plain tensors only")


def _flat(t, rows: int):
    return None if t is None else t.reshape(rows).contiguous()


class _Labels:
    words, heat = 0, 1.0

    def __init__(self, labels, row_weight, ignore: int, reduction: str):
        self.labels, self.row_weight, self.ignore, self.reduction = labels, row_weight, ignore, reduction

    def tensors(self):
        return self.labels, None, self.row_weight

    def given(self, saved):
        """moc_linear_loss's arguments from labels to temperature."""
        return saved[0].data_ptr(), self.ignore, None, N.MOC_I32, 0, None, N.MOC_F32, 0, 0, 1.0

    def counts(self, saved, vocab: int):
        """The rows with a target."""
        return saved[0] != self.ignore

    def rows_f32(self, saved, on, z):
        """Each row's loss by f32 tensor operations; finite where it is not `on`."""
        labels = torch.where(on, saved[0], 0)
        known = (labels >= 0) & (labels < z.shape[1])
        each = -torch.log_softmax(z, -1).gather(1, torch.where(known, labels, 0)[:, None])[:, 0]
        return each * torch.where(known, 1.0, math.nan)


class _Teacher:
    def __init__(self, ids, top, row_weight, heat: float, reduction: str):
        self.ids, self.top, self.row_weight, self.heat, self.reduction = ids, top, row_weight, heat, reduction
        self.words = ids.shape[1]

    def tensors(self):
        return self.ids, self.top, self.row_weight

    def given(self, saved):
        """moc_linear_loss's arguments from labels to temperature."""
        ids, top, _ = saved
        return (None, 0, ids.data_ptr(), N.idx_code(ids.dtype), ids.stride(0), top.data_ptr(), N.dtype_code(top.dtype),
                top.stride(0), self.words, self.heat)

    def counts(self, saved, vocab: int):
        return self._words(saved, vocab).any(1)

    @staticmethod
    def _words(saved, vocab: int):
        ids, top, _ = saved
        return (ids >= 0) & (ids < vocab) & (top != -math.inf)

    def rows_f32(self, saved, on, z):
        there = self._words(saved, z.shape[1]) & on[:, None]
        ids, x = torch.where(there, saved[0].long(), 0), saved[1].float()
        # from the largest, as masks of the type's lowest value over a T below 1 are beyond f32
        x = torch.where(on[:, None], torch.where(there, x, -math.inf), 0.0)
        log_q = torch.log_softmax((x - x.amax(1, keepdim=True)) / self.heat, 1)
        z = z - z.detach().amax(1, keepdim=True)
        q = torch.where(there, log_q.exp(), 0.0)
        # shares of one word added up, each entry weighing its own part of them
        whole = torch.zeros_like(z).scatter_add(1, ids, q).gather(1, ids)
        log_p = torch.log_softmax(z / self.heat, -1).gather(1, ids)
        each = torch.where(q > 0, q * (torch.log(torch.where(q > 0, whole, 1.0)) - log_p), q)
        return self.heat ** 2 * each.sum(1)


def _teacher(what: str, x, ids, top, row_weight, rows: int, temperature: float, reduction: str) -> _Teacher:
    lead = x.shape[:-1]
    if ids.dim() != x.dim() or ids.shape[:-1] != lead or top.shape != ids.shape:
        raise ValueError(f"{what}: the teacher's ids and logits are {(*lead, 'words')}, got {tuple(ids.shape)} and "
                         f"{tuple(top.shape)}")
    words = ids.shape[-1]
    if not 1 <= words <= 1024:
        raise ValueError(f"{what}: 1 to 1024 words of the teacher a row, got {words}")
    if ids.dtype not in (torch.int32, torch.int64) or top.dtype not in (BF16, F32):
        raise ValueError(f"{what}: the teacher's ids are int32 or int64 and its logits bf16 or f32, got {ids.dtype} and "
                         f"{top.dtype}")
    if top.requires_grad:
        raise ValueError(f"{what}: the teacher has no gradient here")
    temperature = float(temperature)
    if not 0 < temperature < math.inf:
        raise ValueError(f"{what}: the temperature must be above 0, got {temperature}")
    return _Teacher(_unit(ids.reshape(rows, words)), _unit(top.reshape(rows, words)), _flat(row_weight, rows),
                    temperature, reduction)


def _unit(t):
    """Rows that do not overlap, of unit stride."""
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) \
        else t.contiguous()


# -------------------------------------------------------------------- operands
def _rows16(t, most: int = 1 << 62) -> torch.Tensor:
    """t [rows, cols] with 16-byte aligned rows of unit stride, at most four times their
    length and MOST_PITCH apart and bf16 ones within `most` bytes, whose storage holds all
    of the last one's pitch (the kernels read whole chunks); a copy of any other."""
    rows, cols = t.shape
    per = 16 // t.element_size()
    pitch = _pitch(t)
    if (t.stride(1) == 1 or cols == 1) and t.data_ptr() % 16 == 0 and pitch % per == 0 and (
            cols <= pitch <= min(4 * K.round_up(cols, 64), MOST_PITCH)) and (
            t.dtype != BF16 or rows * pitch * 2 < most) and (
            (t.storage_offset() + rows * pitch) * t.element_size() <= t.untyped_storage().nbytes()):
        return t
    out = K.padded_empty(rows, cols, t.dtype, t.device)
    _copy_rows(t, out, out.stride(0))
    return out


def _copy_rows(t, out, width: int) -> None:
    """t [rows, cols] into out's rows, zeros behind it up to `width` columns."""
    rows, cols = t.shape
    t, ld = K._rows_view(t)
    if ld < cols:  # rows that overlap
        t, ld = t.contiguous(), cols
    N.call("moc_copy_pad_2d", N.dtype_code(t.dtype), t.data_ptr(), rows, cols, ld, out.data_ptr(), out.stride(0), width,
           N.stream_of(t))


def _pitch(t) -> int:
    per = 16 // t.element_size()
    return t.stride(0) if t.shape[0] > 1 else K.round_up(t.shape[1], per)


def _linear(what: str, hidden, weight, targets) -> torch.Tensor:
    if weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{what}: weight is [vocab, {hidden.shape[-1]}], got {tuple(weight.shape)}")
    _refuse_subclasses(what, hidden, weight, *targets.tensors())
    product = hidden.dtype
    if torch.is_autocast_enabled("cuda"):
        product = torch.get_autocast_dtype("cuda")
        if product != BF16:
            raise ValueError(f"{what}: autocast to bf16, got {product}")
        if weight.dtype not in (BF16, F32):
            raise ValueError(f"{what}: weight is bf16 or f32, got {weight.dtype}")
    elif weight.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden and weight of one type (or under bf16 autocast), got {hidden.dtype} and "
                         f"{weight.dtype}")
    vocab, d = weight.shape
    if vocab > 1 << 21 or d > 1 << 20:
        raise ValueError(f"{what}: a vocabulary of up to 2^21 words, a hidden size of up to 2^20")
    if product == BF16 and vocab * K.row_pitch(d, BF16) * 2 >= K.OPERAND_BYTES:
        raise ValueError(f"{what}: a bf16 weight of up to 2 GiB")
    dev = N.one_device(hidden, weight, *targets.tensors())
    if not N.is_current(dev):
        with torch.cuda.device(dev):
            return _LinearLoss.apply(targets, product, torch.is_grad_enabled(), hidden, weight, *targets.tensors())
    return _LinearLoss.apply(targets, product, torch.is_grad_enabled(), hidden, weight, *targets.tensors())


@lru_cache(maxsize=256)
def _linear_sizes(code: int, rows: int, d: int, vocab: int, words: int, grads: bool) -> tuple[int, int]:
    """(workspace, GEMM workspace) bytes of a shape."""
    return (N.query("moc_linear_loss_workspace_size", code, rows, d, vocab, words, grads),
            N.query("moc_linear_loss_gemm_workspace_size", code, rows, d, vocab, grads))


_COUNTERS: dict = {}  # (device, stream) -> zeroed bytes that every launch leaves zero


def _counters(dev: int, stream: int, where) -> torch.Tensor:
    """Arrival counters of the stream, or the graph's own under capture, since two
    graphs that were captured on one stream may run beside each other."""
    held = _COUNTERS.get((dev, stream))
    if torch.cuda.is_current_stream_capturing():
        held = torch.empty(COUNTER_BYTES, dtype=torch.uint8, device=where)
        N.call("moc_fill_zero", held.data_ptr(), COUNTER_BYTES, stream)
    elif held is None:
        held = _COUNTERS[dev, stream] = torch.zeros(COUNTER_BYTES, dtype=torch.uint8, device=where)
    return held


def _gemm_workspace(dev: int, stream: int, where, nbytes: int) -> torch.Tensor:
    """Counters alone, which are zero between two launches, or the call's own workspace:
    parts of a product wait there for another launch, between which a second thread
    may put its own on the stream.  The call clears the counters of such a one."""
    if nbytes <= COUNTER_BYTES:
        return _counters(dev, stream, where)
    return torch.empty(nbytes, dtype=torch.uint8, device=where)


def _linear_pass(targets, saved, row_weight, mean, grad, product, hidden, weight, each: bool, dh: bool, dw: bool):
    """(the loss, or with `each` the rows' losses; dhidden | None; dweight | None)."""
    dev, where = hidden.get_device(), hidden.device
    vocab, d = weight.shape
    h, w = hidden.reshape(-1, d), weight
    if h.dtype != product:
        h = h.to(product)
    if w.dtype != product:
        w = w.to(product)
    if product == F32 and d % 4:
        return _in_fours(targets, saved, row_weight, mean, grad, hidden, h, w, each, dh, dw)
    h, w = _rows16(h), _rows16(w, K.OPERAND_BYTES)
    rows, code = h.shape[0], N.dtype_code(product)
    out = torch.empty(rows if each else (), dtype=F32, device=where)
    dhidden = torch.empty(hidden.shape, dtype=hidden.dtype, device=where) if dh else None
    dweight = torch.empty((vocab, d), dtype=weight.dtype, device=where) if dw else None
    nbytes, ngemm = _linear_sizes(code, rows, d, vocab, targets.words, dh or dw)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=where)
    stream = N.stream_on(dev)
    gemm_ws = _gemm_workspace(dev, stream, where, ngemm)
    N.call("moc_linear_loss", code, h.data_ptr(), rows, d, _pitch(h), w.data_ptr(), vocab, _pitch(w),
           *targets.given(saved), N.ptr(row_weight), mean, N.ptr(grad), out.data_ptr() if each else None,
           None if each else out.data_ptr(), N.ptr(dhidden), N.dtype_code(hidden.dtype), N.ptr(dweight),
           N.dtype_code(weight.dtype), ws.data_ptr(), nbytes, gemm_ws.data_ptr(), ngemm, stream)
    return out, dhidden, dweight


def _in_fours(targets, saved, row_weight, mean, grad, hidden, h, w, each: bool, dh: bool, dw: bool):
    """_linear_pass of f32 operands with zeros up to a multiple of 4 of the hidden size,
    which the tiled f32 products take (512 rows, 250 x 32000 words: a step of 6.0 ms
    without)."""
    d, wide = h.shape[1], K.round_up(h.shape[1], 4)
    h4, w4 = (torch.empty((t.shape[0], wide), dtype=F32, device=t.device) for t in (h, w))
    _copy_rows(h, h4, wide)
    _copy_rows(w, w4, wide)
    out, *grads = _linear_pass(targets, saved, row_weight, mean, grad, F32, h4, w4, each, dh, dw)
    for i, (g, shape) in enumerate(zip(grads, (hidden.shape, w.shape))):
        if g is not None:
            grads[i] = torch.empty(shape, dtype=F32, device=g.device)
            _copy_rows(g[:, :d], grads[i].view(-1, d), d)
    return out, *grads


def _reduced_f32(targets, saved, rows, weight=None):
    """The operator by f32 tensor operations: of rows of logits, or of hidden rows with
    the head's weight.  Rows that do not count are zeros from the start, as a derivative
    of 0 times their NaN would be NaN."""
    vocab = rows.shape[1] if weight is None else weight.shape[0]
    counts, row_weight = targets.counts(saved, vocab), saved[2]
    w = counts.float() if row_weight is None else torch.where(counts, row_weight, 0.0)
    on = w != 0
    rows = torch.where(on[:, None], rows, 0.0)
    each = targets.rows_f32(saved, on, rows if weight is None else rows @ weight.t())
    each = torch.where(on, each, 0.0) * w  # whatever the upstream gradient of the others
    if targets.reduction == "none":
        return each
    return each.sum() / (w.sum() if targets.reduction == "mean" else 1.0)


def cross_entropy_f32(logits, labels, row_weight=None):
    """linear_cross_entropy's mean of logits that are there already, by f32 tensor
    operations, on any device."""
    rows = labels.numel()
    targets = _Labels(labels.reshape(rows), None if row_weight is None else row_weight.reshape(rows), -100, "mean")
    return _reduced_f32(targets, targets.tensors(), logits.float().flatten(0, -2))


def _capture(dev: int) -> int:
    """What names the HIP graph that the current stream is captured into, or 0."""
    return N.query("moc_capture_id", N.stream_on(dev)) if torch.cuda.is_current_stream_capturing() else 0


class _Kept:
    """Gradients computed ahead, handed out once: the tensors go to the caller, scaled
    in place, so that nothing of them is copied."""

    def __init__(self, grads):
        self.grads = grads
        if grads is not None:
            given = [t for t in grads if t is not None]
            a, b = given[0], given[-1]
            self.scaled = (N.dtype_code(a.dtype), a.data_ptr(), a.numel(), N.dtype_code(b.dtype), b.data_ptr(),
                           b.numel() if len(given) > 1 else 0)
            self.device = a.get_device()
            self.capture = _capture(self.device)

    def take(self, g):
        """The gradients times g, or None: there are none, or no more, or those of a
        forward outside the capture of this backward, whose replay would scale them
        again."""
        grads, self.grads = self.grads, None
        if grads is None or ((now := _capture(self.device)) and now != self.capture):
            return None
        N.call("moc_scale_inplace", *self.scaled, g.data_ptr(), N.stream_on(self.device))
        return grads


def _row_factors(saved, g):
    """reduction="none": the rows' weights times their upstream gradients."""
    g = g.reshape(-1).contiguous()
    return g if saved[2] is None else torch.where(saved[2] == 0, 0.0, g * saved[2])  # NaN g in rows without weight


class _LinearLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, targets, product, grad_mode, hidden, weight, *saved):
        needs = ctx.needs_input_grad
        dh, dw = grad_mode and needs[3], grad_mode and needs[4]
        each = targets.reduction == "none"
        out, *grads = _linear_pass(targets, saved, saved[2], targets.reduction == "mean", None, product, hidden, weight,
                                   each, dh and not each, dw and not each)
        if dh or dw:
            ctx.save_for_backward(hidden, weight, *saved)
            ctx.targets, ctx.product = targets, product
            ctx.kept = _Kept(None if each else grads)
        return out.view(hidden.shape[:-1]) if each else out

    @staticmethod
    def backward(ctx, g):
        rest = None, None, None
        if not torch.is_grad_enabled() and (kept := ctx.kept.take(g)):
            return (None, None, None, *kept, *rest)
        hidden, weight, *saved = ctx.saved_tensors
        targets = ctx.targets
        dh, dw = ctx.needs_input_grad[3:5]
        if torch.is_grad_enabled():
            def stock(h, w):
                h = h.to(ctx.product).float().reshape(-1, h.shape[-1])
                return _reduced_f32(targets, saved, h, w.to(ctx.product).float()).reshape(g.shape)
            return (None, None, None, *graph_grads(stock, (hidden, weight), (dh, dw), g), *rest)
        if targets.reduction == "none":
            got = _linear_pass(targets, saved, _row_factors(saved, g), False, None, ctx.product, hidden, weight, True, dh,
                               dw)
        else:
            got = _linear_pass(targets, saved, saved[2], targets.reduction == "mean", g, ctx.product, hidden, weight, False,
                               dh, dw)
        return (None, None, None, *got[1:], *rest)


def _logits_pass(targets, saved, row_weight, mean, grad, logits, each: bool, grads: bool):
    """(the loss, or with `each` the rows' losses; dlogits | None)."""
    dev, where = logits.get_device(), logits.device
    vocab = logits.shape[-1]
    x = logits.reshape(-1, vocab)
    if (x.stride(1) != 1 and vocab > 1) or (x.shape[0] > 1 and x.stride(0) < vocab):
        x = x.contiguous()
    rows = x.shape[0]
    out = torch.empty(rows if each else (), dtype=F32, device=where)
    dx = torch.empty(logits.shape, dtype=x.dtype, device=where) if grads else None
    nbytes = N.query("moc_logits_loss_workspace_size", rows, targets.words)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=where)
    stream = N.stream_on(dev)
    counters = _counters(dev, stream, where)
    N.call("moc_logits_loss", N.dtype_code(x.dtype), x.data_ptr(), rows, vocab, x.stride(0) if rows > 1 else vocab,
           *targets.given(saved)[2:], N.ptr(row_weight), mean, N.ptr(grad), out.data_ptr() if each else None,
           None if each else out.data_ptr(), N.ptr(dx), vocab, ws.data_ptr(), nbytes, counters.data_ptr(),
           stream)
    return out, dx


class _LogitsLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, targets, grad_mode, logits, *saved):
        need = grad_mode and ctx.needs_input_grad[2]
        each = targets.reduction == "none"
        out, dx = _logits_pass(targets, saved, saved[2], targets.reduction == "mean", None, logits, each,
                               need and not each)
        if need:
            ctx.save_for_backward(logits, *saved)
            ctx.targets = targets
            ctx.kept = _Kept(None if each else (dx,))
        return out.view(logits.shape[:-1]) if each else out

    @staticmethod
    def backward(ctx, g):
        rest = None, None, None
        if not torch.is_grad_enabled() and (kept := ctx.kept.take(g)):
            return (None, None, *kept, *rest)
        logits, *saved = ctx.saved_tensors
        targets = ctx.targets
        if torch.is_grad_enabled():
            def stock(x):
                return _reduced_f32(targets, saved, x.float().reshape(-1, x.shape[-1])).reshape(g.shape)
            return (None, None, *graph_grads(stock, (logits,), (True,), g), *rest)
        if targets.reduction == "none":
            dx = _logits_pass(targets, saved, _row_factors(saved, g), False, None, logits, True, True)[1]
        else:
            dx = _logits_pass(targets, saved, saved[2], targets.reduction == "mean", g, logits, False, True)[1]
        return (None, None, dx, *rest)
