"""What the serving operators over a paged 8-bit cache are timed on.

Three operators of a decode step over a batch of sequences:

  append     K.paged_append: queries and keys rotated by their positions, keys
             and values into pages of 8-bit codes with one scale for each page
             and head (a power of two, grown when a new token needs it);
  attention  K.paged_attention: causal attention of new tokens over such pages,
             one token a sequence or several, ragged;
  sample     K.sample_tokens: temperature, top-k, top-p and min-p from one given
             uniform number a row.

Pages lie in the pool in random order, as after some hours of serving.  Sequence
lengths are ragged and go by the case alone, contents by the seed.  Heads of 64
and 128 and the vocabularies are those of the presets, the decode model and the
loss; grouped heads, pages and contexts are generic.
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

F32, F64, BF16, I32 = torch.float32, torch.float64, torch.bfloat16, torch.int32
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


# --------------------------------------------------------------------- cases
def listed():
    return [
        # One sequence of the decode model (16 heads of 128): the launch counts.
        dict(name="append_step_1", op="append", seqs=1, new=1, context=129, q_heads=16, kv_heads=16, dim=128, page=16,
             tables="bf16"),
        # A serving batch, grouped heads: 64 pages touched, some of them grown.
        dict(name="append_step_64", op="append", seqs=64, new=1, context=8192, q_heads=32, kv_heads=8, dim=128,
             page=64, tables="f32"),
        # Prompts of the 1b shape (32 heads of 64), ragged, going into the cache.
        dict(name="append_prompts", op="append", seqs=9, new=1000, context=200, q_heads=32, kv_heads=32, dim=64,
             page=32, tables="bf16"),
        # The first step behind the decode model's prompt of 128.
        dict(name="step_1_short", op="attention", seqs=1, new=1, context=129, q_heads=16, kv_heads=16, dim=128,
             page=16, codes="e4m3", empty=0),
        # 16 sequences of the decode model, one slot of the batch not in use.
        dict(name="step_16", op="attention", seqs=16, new=1, context=4096, q_heads=16, kv_heads=16, dim=128, page=64,
             codes="e4m3", empty=1),
        # A large serving batch with grouped heads.
        dict(name="step_64_grouped", op="attention", seqs=64, new=1, context=8192, q_heads=32, kv_heads=8, dim=128,
             page=64, codes="e4m3", empty=0),
        # Two long documents, few key heads: the work has to be split over the length.
        dict(name="step_2_long", op="attention", seqs=2, new=1, context=131072, q_heads=28, kv_heads=4, dim=128,
             page=128, codes="int8", empty=0),
        # Drafted tokens being verified, heads of the 1b preset.
        dict(name="verify_5", op="attention", seqs=8, new=5, context=2000, q_heads=32, kv_heads=32, dim=64, page=32,
             codes="int8", empty=0),
        # Chunks of prompts against what is cached of them.
        dict(name="chunks", op="attention", seqs=4, new=1024, context=4096, q_heads=16, kv_heads=16, dim=128, page=64,
             codes="e4m3", empty=0),
        # One row of logits over the decode model's vocabulary, usual settings.
        dict(name="sample_1", op="sample", rows=1, vocab=32000, logits="f32", top_k=50, top_p=0.9, min_p=0.0),
        # A batch of bf16 logits (many equal values), top-p alone.
        dict(name="sample_16", op="sample", rows=16, vocab=32000, logits="bf16", top_k=0, top_p=0.95, min_p=0.0),
        # A large batch over a large vocabulary; settings differ by row.
        dict(name="sample_256", op="sample", rows=256, vocab=128256, logits="f32", top_k=-1, top_p=-1.0, min_p=-1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99))))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "sample"))
    if op == "sample":
        some = rng.random()
        return dict(op="sample", rows=_log(rng, 1, 256), vocab=_log(rng, 500, 128256), logits=rng.choice(("f32", "bf16")),
                    top_k=rng.choice((0, -1, 1, 20, 1000)) if some < 0.7 else 0,
                    top_p=rng.choice((1.0, -1.0, 0.5, 0.99)) if some > 0.3 else 1.0, min_p=rng.choice((0.0, 0.0, -1.0, 0.02)))
    kv_heads = rng.choice((1, 2, 4, 8, 16))
    case = dict(op=op, seqs=_log(rng, 1, 64), kv_heads=kv_heads, q_heads=kv_heads * rng.choice((1, 1, 2, 4, 5, 8)),
                dim=rng.choice((64, 128, 128, 256)), page=rng.choice((16, 32, 64, 128)))
    case["new"] = 1 if rng.random() < 0.6 else _log(rng, 2, max(2, 4096 // case["seqs"]))
    if op == "append":
        return dict(case, context=_log(rng, 1, 8192), tables=rng.choice(("bf16", "f32")))
    # keys and values read, and products, of the largest listed cases at most
    most = (64 << 20) * 8 // (case["seqs"] * kv_heads * case["dim"])
    if case["new"] > 1:
        most = min(most, (1 << 34) // (case["seqs"] * case["new"] * case["q_heads"] * case["dim"]))
    case["context"] = _log(rng, 1, max(64, min(65536, most)))
    return dict(case, codes=rng.choice(("e4m3", "int8")), empty=rng.choice((0, 0, 1)) if case["seqs"] > 1 else 0)


def _lengths(case):
    """(tokens in the cache before the call, new tokens) of each sequence."""
    rng = random.Random("%(seqs)d %(new)d %(context)d" % case)
    top = case["context"]
    before = [top if i == 0 else rng.randint(top // 4, top) for i in range(case["seqs"])]
    new = [case["new"] if i == 0 or case["new"] == 1 else rng.randint(1, case["new"]) for i in range(case["seqs"])]
    return before, new


# -------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    s = SimpleNamespace(op=case["op"])
    if s.op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = normal(rows, vocab) * 2.5
        x[:, : min(vocab, 40)] += 5 * normal(rows, 1).abs()  # a few likely words a row, more or less of them
        s.logits = x[:, torch.randperm(vocab, generator=gen, device="cuda")].to(BF16 if case["logits"] == "bf16" else F32)
        uniform = lambda: torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
        s.u = uniform()
        # -1: each row has its own, and some rows none
        s.temperature = 0.5 + uniform()
        if case["top_k"] < 0:
            s.temperature[::7] = 0.0
        s.top_k = torch.full((rows,), case["top_k"], dtype=I32, device="cuda") if case["top_k"] >= 0 else (
            uniform() * 100).to(I32) * (uniform() < 0.5)
        s.top_p = torch.full((rows,), case["top_p"], device="cuda") if case["top_p"] >= 0 else torch.where(
            uniform() < 0.6, 0.5 + 0.5 * uniform(), 1.0)
        s.min_p = torch.full((rows,), case["min_p"], device="cuda") if case["min_p"] >= 0 else torch.where(
            uniform() < 0.3, 0.1 * uniform(), 0.0)
        return s
    before, new = _lengths(case)
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    total = [b + n for b, n in zip(before, new)]
    if s.op == "attention" and case["empty"]:
        total[-case["empty"]:] = [0] * case["empty"]  # slots of the batch not in use
    pages = [-(-t // page) for t in total]
    pool = sum(pages) + 3
    wide = max(pages)
    order = torch.randperm(pool, generator=gen, device="cuda").to(I32)
    at = torch.arange(wide, dtype=torch.int64)[None] + (torch.tensor(pages).cumsum(0) - torch.tensor(pages))[:, None]
    s.table = order[at.clamp(max=pool - 1).cuda()].contiguous()
    s.lens = torch.tensor(total, dtype=I32, device="cuda")
    tokens, s.longest = sum(new), max(new)
    s.cu = None if case["new"] == 1 else torch.tensor([0] + new, device="cuda").cumsum(0).to(I32)
    kind, largest = CODES[case.get("codes", "e4m3")], LARGEST[case.get("codes", "e4m3")]
    shape = (pool, kv_heads, page, dim)
    # contents of unit scale: codes use the range above 2^-6 (2^-5) of it, by page
    step = 2.0 ** (-6 if kind == CODES["e4m3"] else -5)

    def cached():
        codes = torch.empty(shape, dtype=kind, device="cuda")
        finer = torch.randint(0, 2, (pool, kv_heads), generator=gen, device="cuda")
        scale = step * 2.0 ** -finer.float()
        for i in range(0, pool, 1024):
            x = normal(min(1024, pool - i), *shape[1:]) / scale[i:i + 1024, :, None, None]
            x = x.clamp(-largest, largest)
            codes[i:i + 1024] = x.round().to(kind) if kind == torch.int8 else x.to(kind)
        return codes, scale

    s.k, s.k_scale = cached()
    s.v, s.v_scale = cached()
    if s.op == "attention":
        s.q = (1.5 * normal(tokens, case["q_heads"], dim)).to(BF16)
        s.scale = 1.0 / math.sqrt(dim)
    else:
        # one projection's output, as a block has it
        width = case["q_heads"] + 2 * kv_heads
        qkv = (1.2 * normal(tokens, width, dim)).to(BF16)
        s.q, s.new_k, s.new_v = qkv.split((case["q_heads"], kv_heads, kv_heads), dim=1)
        angle = torch.arange(max(total), dtype=F64)[:, None] * 10000.0 ** (-torch.arange(0, dim, 2, dtype=F64) / dim)
        kind = BF16 if case["tables"] == "bf16" else F32
        s.cos, s.sin = angle.cos().cuda().to(kind), angle.sin().cuda().to(kind)
        s.touched = torch.cat([s.table[b, first // page: -(-t // page)] for b, (first, t) in enumerate(zip(before, total))])
    return s


# ---------------------------------------------------------------- plain forms
def _owners(s, tokens):
    """Sequence and position of each token."""
    if s.cu is None:
        return torch.arange(tokens, device="cuda"), s.lens.long() - 1
    at = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(s.cu[1:].long(), at, right=True)
    return seq, s.lens.long()[seq] - s.cu.long()[seq + 1] + at


def _rotated(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _power_above(x):
    """The least power of two, at least 2^-100, that x is no larger than."""
    m, e = torch.frexp(x.clamp(min=2.0 ** -100))
    return torch.ldexp(torch.ones_like(x), torch.where(m > 0.5, e, e - 1))


def _append_plain(s):
    seq, pos = _owners(s, s.q.shape[0])
    cos, sin = s.cos[pos].float()[:, None], s.sin[pos].float()[:, None]
    page = s.k.shape[2]
    block = s.table.long()[seq, pos // page]
    touched = s.touched.long()
    first = torch.full((s.k.shape[0],), page, device="cuda").index_reduce(0, block, pos % page, "amin")[touched]
    stale = first[:, None] == 0  # what else the page holds is another sequence's
    older = (torch.arange(page, device="cuda") < first[:, None])[:, None, :, None]

    def store(codes, scale, x):
        most = torch.zeros_like(scale).index_reduce(0, block, x.abs().amax(-1), "amax")[touched]
        old = scale[touched]
        need = torch.maximum(_power_above(torch.where(stale, 0.0, old)), _power_above(most / LARGEST["e4m3"]))
        bits = codes.view(torch.uint8)
        held = bits[touched]
        kept = (held.view(codes.dtype).float() * (old / need)[..., None, None]).to(codes.dtype)
        bits[touched] = torch.where(older, kept.view(torch.uint8), held)
        scale[touched] = need
        bits[block, :, pos % page] = (x / scale[block][..., None]).to(codes.dtype).view(torch.uint8)

    store(s.k, s.k_scale, _rotated(s.new_k.float(), cos, sin))
    store(s.v, s.v_scale, s.new_v.float())
    return _rotated(s.q.float(), cos, sin).to(BF16)


def _attention_plain(s):
    tokens, heads, dim = s.q.shape
    seqs, wide = s.table.shape
    kv_heads, page = s.k.shape[1:3]
    seq, pos = _owners(s, tokens)
    table = s.table.long()

    def cached(codes, scale):
        x = codes.view(torch.uint8)[table].view(codes.dtype).float() * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(seqs, kv_heads, wide * page, dim)

    # rows of a sequence: its tokens, padded to the longest, times the heads of a group
    slot = torch.arange(tokens, device="cuda") - (s.cu.long()[seq] if s.cu is not None else seq)
    q = torch.zeros(seqs, s.longest, heads, dim, device="cuda")
    q[seq, slot] = s.q.float()
    where = torch.full((seqs, s.longest), -1, device="cuda")
    where[seq, slot] = pos
    group = heads // kv_heads
    q = q.view(seqs, s.longest, kv_heads, group, dim).transpose(1, 2).reshape(seqs, kv_heads, s.longest * group, dim)
    x = torch.matmul(q, cached(s.k, s.k_scale).transpose(-1, -2).contiguous()) * s.scale
    seen = torch.arange(wide * page, device="cuda") <= where.repeat_interleave(group, 1)[:, None, :, None]
    x = x.masked_fill(~seen, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    y = torch.matmul(e, cached(s.v, s.v_scale)) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    y = y.view(seqs, kv_heads, s.longest, group, dim).transpose(1, 2).reshape(seqs, s.longest, heads, dim)
    return y[seq, slot].to(BF16)


def _sample_plain(s):
    """In 64 bits: the draw lies next to a border of some word's share in one row of a few hundred otherwise."""
    x, order = torch.sort(s.logits.double(), dim=-1, descending=True, stable=True)
    vocab = x.shape[1]
    heat = s.temperature.double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(heat > 0, heat, 1.0))
    k = s.top_k.long()[:, None]
    w = torch.where((k <= 0) | (torch.arange(vocab, device="cuda") < k), w, 0.0)
    total = w.cumsum(-1)
    p = s.top_p.double()[:, None]
    keep = (p >= 1) | (total - w < p * total[:, -1:])
    keep = keep & (w >= s.min_p.double()[:, None])
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    c = w.cumsum(-1)
    drawn = (c <= s.u.double()[:, None] * c[:, -1:]).sum(-1)
    return torch.where(heat[:, 0] > 0, drawn, order[:, 0])


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        from moc_amd import kernels as K
        if s.op == "sample":
            return K.sample_tokens(s.logits, s.u, s.temperature, s.top_k, s.top_p, s.min_p)
        kv = K.PagedKV(s.k, s.v, s.k_scale, s.v_scale)
        if s.op == "attention":
            return K.paged_attention(s.q, kv, s.table, s.lens, s.cu, scale=s.scale)
        q = K.paged_append(s.q, s.new_k, s.new_v, s.cos, s.sin, kv, s.table, s.lens, s.cu)
    else:
        if s.op == "sample":
            return _sample_plain(s)
        if s.op == "attention":
            return _attention_plain(s)
        q = _append_plain(s)
    return {"q": q, "k": s.k, "v": s.v, "k_scale": s.k_scale, "v_scale": s.v_scale}


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["logits"] == "bf16" else 4) + case["rows"] * 28, "flops": 6 * n}
    before, new = _lengths(case)
    heads, kv_heads, dim, page = (case[k] for k in ("q_heads", "kv_heads", "dim", "page"))
    if case["op"] == "append":
        tokens = sum(new)
        touched = sum(-(-(b + n) // page) - b // page for b, n in zip(before, new))
        return {"bytes": tokens * dim * (4 * heads + 4 * kv_heads + 2 * kv_heads + 4) + touched * (16 * kv_heads + 4),
                "flops": tokens * dim * (3 * heads + 6 * kv_heads)}
    live = list(zip(before, new))[: case["seqs"] - case["empty"]]
    pairs = sum(b * n + n * (n + 1) // 2 for b, n in live)
    cells = sum(b + n for b, n in live)
    return {"bytes": 2 * cells * kv_heads * dim + 4 * sum(new) * heads * dim + 8 * kv_heads * cells // page,
            "flops": 4 * pairs * heads * dim}


# ------------------------------------------------------------- from 64 bits
def _nearest_e4m3(y):
    """y rounded to the e4m3 grid: three bits below the leading one, steps of 2^-9 at the low end."""
    e = torch.floor(torch.log2(y.abs().clamp(min=1e-300))).clamp(min=-6)
    step = 2.0 ** (e - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "sample":
        import numpy as np
        x = s.logits.double().cpu().numpy()
        u, heat, k, p, least = (t.double().cpu().numpy() for t in (s.u, s.temperature, s.top_k, s.top_p, s.min_p))
        out = np.empty(len(x), dtype=np.int64)
        for r, row in enumerate(x):
            if heat[r] <= 0:
                out[r] = int(np.argmax(row))
                continue
            share = np.exp((row - row.max()) / heat[r])
            best = np.lexsort((np.arange(len(row)), -row))
            if k[r] > 0:
                best = best[: int(k[r])]
            if p[r] < 1:
                mass = np.cumsum(share[best])
                best = best[: max(1, int(np.searchsorted(np.concatenate(([0.0], mass[:-1])), p[r] * mass[-1], side="left")))]
            best = np.sort(best[share[best] >= least[r]])
            mass = np.cumsum(share[best])
            out[r] = best[min(len(best) - 1, int(np.searchsorted(mass, u[r] * mass[-1], side="right")))]
        return out
    before, new = _lengths(case)
    lens, table = s.lens.tolist(), s.table.tolist()
    starts = [sum(new[:i]) for i in range(len(new))]
    heads, kv_heads, dim, page = (case[n] for n in ("q_heads", "kv_heads", "dim", "page"))
    if s.op == "attention":
        out = torch.zeros(sum(new), heads, dim, dtype=F64, device="cuda")
        for b, (start, n) in enumerate(zip(starts, new)):
            length = lens[b]
            if not length:
                continue
            ids = s.table[b, : -(-length // page)].long()
            k, v = ((c.view(torch.uint8)[ids].view(c.dtype).double() * f.double()[ids][..., None, None])
                    .permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :length].contiguous()
                    for c, f in ((s.k, s.k_scale), (s.v, s.v_scale)))
            later = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
            for h in range(heads):
                x = s.q[start:start + n, h].double() @ k[h * kv_heads // heads].t().contiguous() * s.scale
                out[start:start + n, h] = torch.softmax(x.masked_fill(later, -math.inf), -1) @ v[h * kv_heads // heads]
        return out

    def turned(x, first):
        pos = slice(first, first + x.shape[0])
        z = torch.view_as_complex(x.double().reshape(*x.shape[:-1], dim // 2, 2).contiguous())
        return torch.view_as_real(z * torch.complex(s.cos[pos].double(), s.sin[pos].double())[:, None]).flatten(-2)

    q = torch.empty(sum(new), heads, dim, dtype=F64, device="cuda")
    result = {n: getattr(s, n).double() for n in ("k", "v", "k_scale", "v_scale")}
    for b, (start, n) in enumerate(zip(starts, new)):
        rows, first = slice(start, start + n), lens[b] - n
        q[rows] = turned(s.q[rows], first)
        for name, x in (("k", turned(s.new_k[rows], first)), ("v", s.new_v[rows].double())):
            for at in range(first // page, -(-(first + n) // page)):
                lo, hi = max(first, at * page), min(first + n, (at + 1) * page)
                part, id_ = x[lo - first:hi - first].transpose(0, 1), table[b][at]
                codes, scale = result[name][id_], result[name + "_scale"][id_]
                need = part.abs().amax((1, 2)) / LARGEST["e4m3"]
                old = scale if lo % page else torch.zeros_like(scale)
                grown = 2.0 ** torch.ceil(torch.log2(torch.maximum(need, old).clamp(min=2.0 ** -100)))
                codes[:, : lo % page] = _nearest_e4m3(codes[:, : lo % page] * (scale / grown)[:, None, None])
                codes[:, lo % page: lo % page + hi - lo] = _nearest_e4m3(part / grown[:, None, None])
                scale.copy_(grown)
    return {"q": q, **result}
