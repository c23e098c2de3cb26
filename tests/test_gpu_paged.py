"""K.paged_append and K.paged_attention against plain forms in 64 bits."""
import math

import pytest
import torch

from moc_amd import kernels as K
from moc_amd.inference.decode_model import rope_tables

import paged_reference as R

pytestmark = pytest.mark.gpu
BF, E4, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.int8


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _batch(new, before, page, pool_extra=2, seed=0, width=None):
    """(table, lens, cu, pages of the pool) of sequences with `before` tokens in
    the cache and `new` more; cu None where each has one."""
    total = [b + n for b, n in zip(before, new)]
    need = [-(-max(t, 0) // page) for t in total]
    pool = sum(need) + pool_extra
    order = torch.randperm(pool, generator=_gen(seed)).tolist()
    width = max(need + [1]) if width is None else width
    table = torch.full((len(new), width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    cu = None if all(n == 1 for n in new) else _ints([sum(new[:i]) for i in range(len(new) + 1)])
    return table.cuda(), _ints(total), cu, pool


def _cache(pool, kv_heads, page, dim, kind, seed=0):
    """A cache full of codes of unit scale."""
    g = _gen(seed)
    out = []
    for _ in range(2):
        x = torch.randn(pool, kv_heads, page, dim, generator=g)
        s = 2.0 ** (-torch.randint(5, 8, (pool, kv_heads), generator=g).float())
        y = (x / s[..., None, None]).clamp(-R.LARGEST[kind], R.LARGEST[kind])
        out.append(((y.round() if kind == I8 else y).to(kind).cuda(), s.cuda()))
    return K.PagedKV(out[0][0], out[1][0], out[0][1], out[1][1])


def _bits(t):
    return t.view(torch.uint8)


def _clone(kv):
    return K.PagedKV(_bits(kv.k).clone().view(kv.k.dtype), _bits(kv.v).clone().view(kv.v.dtype), kv.k_scale.clone(),
                     kv.v_scale.clone())


# ------------------------------------------------------------------ attention
def _close(o, ref, size, what=""):
    """Probabilities go to the product as bf16 (2^-8 of each at most, so of the
    sum over |v|), scores and sums in f32 (2^-10 of it covers sums of 256
    products of scores below 64), the result is rounded to bf16 (2^-8)."""
    o = o.cpu().double()
    assert torch.equal(torch.isnan(o), torch.isnan(ref)), what
    bound = (2.0 ** -8 + 2.0 ** -10) * size + 2.0 ** -8 * ref.abs() + 1e-30
    ok = ((o - ref).abs() <= bound) | torch.isnan(ref)
    assert ok.all(), (what, float(((o - ref).abs() / bound).nan_to_num().max()))


def _attend(new, before, q_heads, kv_heads, dim, page, kind, seed=1, **more):
    table, lens, cu, pool = _batch(new, before, page, seed=seed, **more)
    kv = _cache(pool, kv_heads, page, dim, kind, seed)
    q = (1.5 * torch.randn(sum(new), q_heads, dim, generator=_gen(seed + 7))).to(BF).cuda()
    o = K.paged_attention(q, kv, table, lens, cu)
    ref, size = R.attention(q, kv, table, lens, cu, dim ** -0.5)
    _close(o, ref, size)
    return q, kv, table, lens, cu, o


@pytest.mark.parametrize("kind", [E4, I8])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads,page", [(4, 4, 16), (8, 2, 32), (5, 1, 64), (14, 2, 128), (40, 2, 256)])
def test_attention_one_token(kind, dim, q_heads, kv_heads, page):
    """Lengths of one, about a tile's, a page's and a chunk's ends."""
    before = [0, 1, 14, 15, 16, 62, 63, 64, 254, 255, 256, 300]
    _attend([1] * len(before), before, q_heads, kv_heads, dim, page, kind)


@pytest.mark.parametrize("kind", [E4, I8])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [(4, 4, 64, 32), (6, 2, 128, 16), (8, 1, 256, 64), (3, 3, 128, 128)])
def test_attention_ragged(kind, q_heads, kv_heads, dim, page):
    """Several new tokens, among them whole prompts, empty sequences and one token."""
    new = [5, 1, 0, 17, 64, 33, 130]
    before = [100, 7, 50, 0, 0, 31, 200]
    _attend(new, before, q_heads, kv_heads, dim, page, kind)


@pytest.mark.parametrize("seqs,length", [(1, 5000), (2, 20000), (70, 900)])
def test_attention_split_over_the_length(seqs, length):
    """Chunks that join in a second launch; more sequences than lanes."""
    before = [length - 37 * i % length for i in range(seqs)]
    _attend([1] * seqs, before, 4, 2, 128, 64, E4)


@pytest.mark.parametrize("kind", [E4, I8])
@pytest.mark.parametrize("new,before,q_heads,kv_heads,dim,page", [
    ([700, 3, 900, 500, 1], [0, 40, 130, 7, 2000], 32, 16, 64, 32), ([1100, 0, 900], [0, 0, 513], 20, 10, 128, 64),
    ([400, 1, 1300], [65, 3, 0], 40, 8, 256, 16), ([33, 65, 300], [0, 5, 64], 3, 3, 128, 256)])
def test_attention_prompts(kind, new, before, q_heads, kv_heads, dim, page):
    """Row tiles of both sizes; the ends of each sequence and rows between."""
    table, lens, cu, pool = _batch(new, before, page, seed=2)
    kv = _cache(pool, kv_heads, page, dim, kind, 2)
    q = (1.5 * torch.randn(sum(new), q_heads, dim, generator=_gen(3))).to(BF).cuda()
    o = K.paged_attention(q, kv, table, lens, cu)
    ends = [e for s, n in zip(cu.tolist(), new) for e in (s, s + n // 3, s + n // 2 + 1, s + n - 2, s + n - 1) if n > 2]
    rows = sorted({r for r in ends + list(range(0, sum(new), 131)) if 0 <= r < sum(new)})
    ref, size = R.attention(q, kv, table, lens, cu, dim ** -0.5, set(rows))
    _close(o[rows], ref[rows], size[rows])


@pytest.mark.parametrize("kind,dim,page", [(E4, 64, 16), (I8, 128, 64), (E4, 128, 256), (E4, 256, 32)])
def test_attention_prompts_behind_a_long_cache(kind, dim, page):
    """Many rows of few sequences, split over the length: chunks that all, some or
    no rows see, a table wider than the sequences, a position without a page and a
    NaN code in one chunk, a length behind the table."""
    new, before = [300, 40, 1, 0, 130], [5000, 700, 3000, 0, 0]
    table, lens, cu, pool = _batch(new, before, page, seed=4, width=-(-5600 // page))
    kv = _cache(pool, 2, page, dim, kind, 4)
    q = (1.5 * torch.randn(sum(new), 4, dim, generator=_gen(5))).to(BF).cuda()
    ends = [0, 1, 127, 128, 200, 299, 300, 339, 340, 341, 342, 468, 470]

    def check(what):
        o = K.paged_attention(q, kv, table, lens, cu)
        ref, size = R.attention(q, kv, table, lens, cu, dim ** -0.5, set(ends))
        _close(o[ends], ref[ends], size[ends], what)
        return o

    clean = check("whole")
    hole = int(table[0, 4000 // page])
    table[0, 4000 // page] = pool
    o = check("no page")
    assert torch.isnan(o[:300]).all() and torch.equal(o[300:], clean[300:])
    table[0, 4000 // page] = hole
    if kind == E4:
        at = int(table[0, 5100 // page])
        kept = _bits(kv.v)[at].clone()
        _bits(kv.v)[at, :, 5100 % page, 3] = 0x7F
        o = K.paged_attention(q, kv, table, lens, cu)
        assert torch.equal(o[:100], clean[:100]) and torch.equal(o[300:], clean[300:])
        assert torch.isnan(o[100:300]).flatten(1).any(1).all()
        _bits(kv.v)[at] = kept
    lens[4] = 130 + table.shape[1] * page  # all its rows are behind the table
    o = check("behind the table")
    assert torch.isnan(o[341:]).all() and torch.equal(o[:341], clean[:341])


@pytest.mark.parametrize("n", [4, 12, 60, 200])
def test_attention_codes_that_later_rows_see(n):
    """NaN codes and scales, a page out of range: the rows before them are as
    without them, the rows from them on are NaN."""
    table, lens, cu, pool = _batch([n, 2], [50, 9], 16)
    kv = _cache(pool, 2, 16, 64, E4)
    q = torch.randn(n + 2, 4, 64, generator=_gen(5)).to(BF).cuda()
    clean = K.paged_attention(q, kv, table, lens, cu)
    for at in (0, 1, n // 2, n - 1):
        pos = 50 + at
        for part in ("k", "v"):
            bad = _clone(kv)
            _bits(getattr(bad, part))[table[0, pos // 16].long(), :, pos % 16, 5] = 0x7F
            o = K.paged_attention(q, bad, table, lens, cu)
            assert torch.equal(o[:at], clean[:at]) and torch.equal(o[n:], clean[n:])
            assert torch.isnan(o[at:n]).flatten(1).any(1).all()
        first = max(0, pos // 16 * 16 - 50)  # the first row that sees the page
        for part in ("k_scale", "v_scale"):
            bad = _clone(kv)
            getattr(bad, part)[table[0, pos // 16].long()] = math.nan
            o = K.paged_attention(q, bad, table, lens, cu)
            assert torch.equal(o[:first], clean[:first]) and torch.isnan(o[first:n]).all() and torch.equal(o[n:], clean[n:])
        wrong = table.clone()
        wrong[0, pos // 16] = pool + 3
        o = K.paged_attention(q, kv, wrong, lens, cu)
        assert torch.equal(o[:first], clean[:first]) and torch.isnan(o[first:n]).all() and torch.equal(o[n:], clean[n:])


def test_attention_many_ragged_sequences():
    """More sequences than a wave has lanes, some empty."""
    new = [(i * 7) % 4 for i in range(150)]
    _attend(new, [(i * 13) % 90 for i in range(150)], 4, 2, 64, 16, E4)


def test_attention_general_scales():
    """Scales from elsewhere, no powers of two; a score scale of the caller's."""
    table, lens, cu, pool = _batch([1, 1], [90, 200], 32)
    kv = _cache(pool, 2, 32, 128, E4)
    g = _gen(3)
    kv.k_scale.copy_(0.003 + 0.02 * torch.rand(kv.k_scale.shape, generator=g))
    kv.v_scale.copy_(0.003 + 0.02 * torch.rand(kv.v_scale.shape, generator=g))
    q = torch.randn(2, 4, 128, generator=g).to(BF).cuda()
    _close(K.paged_attention(q, kv, table, lens, scale=0.11), *R.attention(q, kv, table, lens, None, 0.11))


def test_attention_peaked_rows():
    """Scores of hundreds: one position holds all the weight."""
    table, lens, cu, pool = _batch([1, 3], [700, 300], 64)
    kv = _cache(pool, 2, 64, 128, E4)
    q = (60 * torch.randn(4, 4, 128, generator=_gen(5))).to(BF).cuda()
    o = K.paged_attention(q, kv, table, lens, cu).cpu().double()
    ref, size = R.attention(q, kv, table, lens, cu, 128 ** -0.5)
    # scores to 2000 with sums of 128 products: 128 2^-24 2000 = 2^-6 at worst of each probability
    assert ((o - ref).abs() <= (2.0 ** -8 + 2.0 ** -5) * size + 2.0 ** -8 * ref.abs()).all()


def test_attention_rows_that_see_nothing():
    """Slots not in use (lens 0), and new rows before position 0: zeros."""
    table, lens, cu, pool = _batch([2, 1, 3], [0, 40, 5], 16)
    kv = _cache(pool, 2, 16, 64, E4)
    q = torch.randn(6, 4, 64, generator=_gen(5)).to(BF).cuda()
    short = _ints([0, 41, 2])  # the third has three rows and two tokens
    o = K.paged_attention(q, kv, table, short, cu)
    ref, size = R.attention(q, kv, table, short, cu, 0.125)
    _close(o, ref, size)
    assert not o[:2].any() and not o[3].any() and o[4].any()
    assert not K.paged_attention(q, kv, table, _ints([0, -3, -(2 ** 31)]), cu).any()


@pytest.mark.parametrize("kind", [E4, I8])
def test_attention_reads_no_place_without_a_token(kind):
    """Places behind the last token and pages behind the last one, whatever they
    hold: NaN codes, scales of NaN and infinity, page numbers out of range."""
    new, before = [1, 1, 4, 20], [20, 63, 10, 0]
    table, lens, cu, pool = _batch(new, before, 16, seed=3)
    kv = _cache(pool, 2, 16, 128, kind)
    q = torch.randn(sum(new), 4, 128, generator=_gen(5)).to(BF).cuda()
    clean = K.paged_attention(q, kv, table, lens, cu)
    used = torch.zeros(pool, 16, dtype=torch.bool)
    for b, t in enumerate(lens.tolist()):
        for p in range(t):
            used[int(table[b, p // 16]), p % 16] = True
    for codes in (kv.k, kv.v):
        _bits(codes).permute(0, 2, 1, 3)[~used.cuda()] = 0x7F
    for scale in (kv.k_scale, kv.v_scale):
        scale[~used.any(1).cuda()] = math.nan
    wild = torch.cat((table, torch.full_like(table, 2 ** 31 - 1)), 1)
    for b, t in enumerate(lens.tolist()):
        wild[b, -(-t // 16):] = 10 ** 9
    assert torch.equal(K.paged_attention(q, kv, wild, lens, cu), clean)


def test_attention_bad_pages_and_lengths_give_nan():
    new, before = [1, 3, 1, 1], [40, 30, 20, 100]
    table, lens, cu, pool = _batch(new, before, 16)
    kv = _cache(pool, 2, 16, 64, E4)
    q = torch.randn(6, 4, 64, generator=_gen(5)).to(BF).cuda()
    good = K.paged_attention(q, kv, table, lens, cu)
    table[0, 1] = -1
    table[1, 2] = pool          # seen by the last of its three rows (positions 30, 31, 32)
    lens[3] = table.shape[1] * 16 + 1
    o = K.paged_attention(q, kv, table, lens, cu)
    assert torch.isnan(o[0]).all() and torch.isnan(o[3]).all() and torch.isnan(o[5]).all()
    assert torch.equal(o[[1, 2, 4]], good[[1, 2, 4]])
    lens[3] = 2 ** 31 - 1
    assert torch.isnan(K.paged_attention(q, kv, table, lens, cu)[5]).all()


def test_attention_strides_and_out():
    """q as a section of a projection, out as a section of a wider buffer, rows
    off the 16-byte grid, rows behind the last sequence."""
    table, lens, cu, pool = _batch([2, 3], [60, 10], 32)
    kv = _cache(pool, 2, 32, 64, E4)
    qkv = torch.randn(7, 8, 64, generator=_gen(4)).to(BF).cuda()
    want = K.paged_attention(qkv[:5, 2:6].contiguous(), kv, table, lens, cu)
    wide = torch.full((7, 10, 64), 7.0, dtype=BF, device="cuda")
    K.paged_attention(qkv[:, 2:6], kv, table, lens, cu, out=wide[:, 3:7])
    assert torch.equal(wide[:5, 3:7], want)
    wide[:5, 3:7] = 7.0
    assert (wide == 7.0).all()
    off = torch.empty(5 * 4 * 64 + 1, dtype=BF, device="cuda")[1:].view(5, 4, 64)
    off.copy_(qkv[:5, 2:6])
    assert torch.equal(K.paged_attention(off, kv, table, lens, cu), want)
    part = table.repeat(1, 3)[:, : table.shape[1]]  # rows of a wider table
    assert torch.equal(K.paged_attention(qkv[:5, 2:6], kv, part, lens, cu), want)


def test_attention_nothing_to_do():
    kv = _cache(3, 2, 16, 64, E4)
    none = _ints([])
    assert K.paged_attention(torch.empty(0, 4, 64, dtype=BF, device="cuda"), kv, none.view(0, 2), none).shape == (0, 4, 64)
    q = torch.randn(2, 4, 64, generator=_gen(1)).to(BF).cuda()
    o = K.paged_attention(q, kv, _ints([]).view(2, 0), _ints([0, 5]))
    assert not o[0].any() and torch.isnan(o[1]).all()


def test_cache_beyond_32_bit_offsets():
    """Pages behind 4 GiB of codes, read and written."""
    pages, heads, page, dim = 17000, 2, 256, 256  # 4.46e9 bytes of keys
    kv = K.PagedKV(*(torch.zeros(pages, 2 * heads, page, dim, dtype=torch.uint8, device="cuda").view(E4) for _ in range(2)),
                   *(torch.zeros(pages, 2 * heads, device="cuda") for _ in range(2)))
    small = _cache(3, 2 * heads, page, dim, E4)
    table = _ints([[0, 1, 2]])
    far = _ints([[pages - 1, 0, pages - 2]])
    for dst, src in zip(kv, small):
        for i in range(3):
            (_bits(dst) if dst.dtype == E4 else dst)[far[0, i]] = (_bits(src) if src.dtype == E4 else src)[i]
    q, k, v = (torch.randn(1, h, dim, generator=_gen(h)).to(BF).cuda() for h in (8, 4, 4))
    cos, sin = (t.cuda() for t in rope_tables(dim, 800))
    lens = _ints([701])
    turned = [K.paged_append(q, k, v, cos, sin, c, t, lens) for c, t in ((small, table), (kv, far))]
    assert torch.equal(*turned)
    assert torch.equal(K.paged_attention(turned[0], small, table, lens), K.paged_attention(turned[1], kv, far, lens))
    assert torch.equal(_bits(kv.k)[far[0].long()], _bits(small.k))


# --------------------------------------------------------------------- append
def _check_append(before_kv, kv, q, k, v, cos, sin, table, lens, cu, got):
    """The call against the definition: rotated q to a bf16 rounding, codes to
    half a step, scales, re-encoded older codes and all other bytes exactly."""
    kind, (pages, heads, page, dim) = kv.k.dtype, kv.k.shape
    spans = R.spans(q.shape[0], lens.cpu(), None if cu is None else cu.cpu())
    rows = [r for _, s, n, _ in spans for r in range(s, s + n)]
    ref = R.rotated(q, cos, sin, lens, cu)[rows]
    out = got.cpu().double()[rows]
    room = table.shape[1] * page
    keep = torch.tensor([length - n + i < room for _, _, n, length in spans for i in range(n)])
    ref[~keep] = math.nan
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    # a product and a sum in f32 (2^-22 of the pair), then bf16
    pair = q.cpu().double()[rows].abs()
    pair = (pair[..., 0::2] + pair[..., 1::2]).repeat_interleave(2, -1)
    assert (((out - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -21 * pair) | torch.isnan(ref)).all()
    turned = R.rotated(k, cos, sin, lens, cu)
    largest = R.LARGEST[kind]
    for name, x, size in (("k", turned, k.cpu().double().abs()), ("v", v.cpu().double(), None)):
        codes0, scale0 = R.values(getattr(before_kv, name)), getattr(before_kv, name + "_scale").cpu().double()
        want, want_scale = codes0.clone(), scale0.clone()
        codes, scale = R.values(getattr(kv, name)), getattr(kv, name + "_scale").cpu().double()
        for b, start, n, length in spans:
            first = length - n
            stop = min(length, room, cos.shape[0])
            for at in range(max(first, 0) // page, -(-stop // page)):
                lo, hi = max(first, at * page), min(stop, (at + 1) * page)
                page_id = int(table[b, at])
                if hi <= lo or not 0 <= page_id < pages:
                    continue
                part = x[start + lo - first:start + hi - first].transpose(0, 1)  # [heads, n, dim]
                err = torch.zeros_like(part)
                if size is not None:
                    err = size[start + lo - first:start + hi - first].transpose(0, 1)
                    err = 2.0 ** -21 * (err[..., 0::2] + err[..., 1::2]).repeat_interleave(2, -1)
                place = lo % page
                most = part.abs().amax((1, 2))
                old = scale0[page_id] if place else torch.zeros(heads, dtype=torch.float64)
                s = scale[page_id]
                assert torch.equal(torch.frexp(s)[0], torch.full_like(s, 0.5)), "powers of two"
                floor = torch.maximum(old, torch.full_like(s, 2.0 ** -100))
                slack = err.amax((1, 2))
                assert (most <= largest * s + slack).all() and (s >= floor).all()
                assert ((s / 2 < floor) | (most + slack > largest * s / 2)).all(), "the least power"
                new = codes[page_id, :, place:place + hi - lo]
                y = part / s[:, None, None]
                assert ((new - y).abs() <= R.half_step(y, kind) * (1 + 2.0 ** -18) + err / s[:, None, None]).all()
                want[page_id, :, place:place + hi - lo] = new
                want_scale[page_id] = s
                want[page_id, :, :place] = R.round_codes(codes0[page_id, :, :place] * (old / s)[:, None, None], kind)
        assert torch.equal(codes, want), name
        assert torch.equal(scale, want_scale), name


def _append(new, before, q_heads, kv_heads, dim, page, kind, table_dtype=torch.float32, seed=1, spread=1.0, angles=None):
    table, lens, cu, pool = _batch(new, before, page, seed=seed)
    kv = _cache(pool, kv_heads, page, dim, kind, seed)
    g = _gen(seed + 3)
    x = torch.randn(sum(new), q_heads + 2 * kv_heads, dim, generator=g)
    x *= torch.exp2(spread * torch.randn(sum(new), 1, 1, generator=g))  # some tokens grow their block
    q, k, v = x.to(BF).cuda().split((q_heads, kv_heads, kv_heads), 1)
    cos, sin = (t.cuda().to(table_dtype) for t in rope_tables(dim, angles or max(before) + max(new)))
    was = _clone(kv)
    got = K.paged_append(q, k, v, cos, sin, kv, table, lens, cu)
    _check_append(was, kv, q, k, v, cos, sin, table, lens, cu, got)
    return q, k, v, cos, sin, kv, table, lens, cu, got, was


@pytest.mark.parametrize("kind", [E4, I8])
@pytest.mark.parametrize("table_dtype", [BF, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads,page", [(4, 4, 16), (6, 2, 64), (5, 1, 256)])
def test_append_one_token(kind, table_dtype, dim, q_heads, kv_heads, page):
    _append([1] * 9, [0, 1, 14, 15, 16, 63, 64, 200, 257], q_heads, kv_heads, dim, page, kind, table_dtype, spread=2.0)


@pytest.mark.parametrize("kind", [E4, I8])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [(4, 4, 64, 32), (6, 2, 128, 16), (8, 1, 256, 128), (2, 2, 64, 256)])
def test_append_ragged(kind, q_heads, kv_heads, dim, page):
    _append([5, 1, 0, 17, 64, 33, 300], [100, 7, 50, 0, 0, 31, 200], q_heads, kv_heads, dim, page, kind)


def test_append_many_sequences():
    _append([(i * 7) % 5 for i in range(140)], [(i * 13) % 90 for i in range(140)], 2, 2, 64, 16, E4)
    _append([1] * 140, [(i * 13) % 90 for i in range(140)], 2, 2, 64, 16, E4)


def test_append_in_steps_equals_a_cache_of_the_same_values():
    """A prompt and single tokens, against the values: each code within the half
    steps of the roundings it went through (its own, one more for each growth of
    its block below the normal range: the last scale's half step bounds them all,
    doubled)."""
    dim, page, heads = 128, 16, 2
    g = _gen(9)
    k = torch.randn(40, heads, dim, generator=g) * torch.linspace(0.2, 6, 40)[:, None, None]
    k, v = k.to(BF).cuda(), (k * 0.5).to(BF).cuda()
    kv = K.paged_kv(4, heads, page, dim)
    table = _ints([[2, 0, 3]])
    one = torch.ones(64, dim // 2, device="cuda")
    zero = torch.zeros_like(one)
    K.paged_append(k[:21], k[:21], v[:21], one, zero, kv, table, _ints([21]), _ints([0, 21]))
    for i in range(21, 40):
        K.paged_append(k[i:i + 1], k[i:i + 1], v[i:i + 1], one, zero, kv, table, _ints([i + 1]))
    for codes, scale, x in ((kv.k, kv.k_scale, k), (kv.v, kv.v_scale, v)):
        ids = table[0].long().cpu()
        s = scale.cpu().double()[ids][..., None, None]
        y = R.values(codes)[ids]
        got = (y * s).transpose(1, 2).reshape(-1, heads, dim)[:40]
        x = x.cpu().double()
        step = (R.half_step(y.abs(), E4) * s).transpose(1, 2).reshape(-1, heads, dim)[:40]
        assert ((got - x).abs() <= 2 * step).all()
        most = x.abs().reshape(40, heads, dim)
        for i, at in enumerate(ids):
            part = most[16 * i:16 * i + 16].amax((0, 2))
            assert (part <= 448 * scale.cpu().double()[at]).all()


def test_append_zeros_and_tiny_and_huge():
    """Blocks of zeros, of values far below the least scale and near bf16's ends."""
    table, lens, cu, pool = _batch([1] * 4, [0, 3, 0, 17], 16)
    for kind in (E4, I8):
        kv = _cache(pool, 1, 16, 64, kind)
        k = torch.zeros(4, 1, 64)
        k[1, 0, :8], k[2, 0, 5], k[3, 0, 9] = 1e-38, 3e38, -3.3e38
        k = k.to(BF).cuda()
        was = _clone(kv)
        cos, sin = torch.ones(32, 32, device="cuda"), torch.zeros(32, 32, device="cuda")
        got = K.paged_append(k, k, k, cos, sin, kv, table, lens)
        _check_append(was, kv, k, k, k, cos, sin, table, lens, None, got)
        assert kv.k_scale[table[0, 0].long(), 0] == 2.0 ** -100


def test_append_values_that_are_not_finite():
    """They do not count for the scale; NaN codes (e4m3), the ends or 0 (int8)."""
    table, lens, cu, pool = _batch([1, 1], [0, 4], 16)
    x = torch.ones(2, 1, 64)
    x[0, 0, 3], x[0, 0, 4], x[1, 0, 0] = math.inf, math.nan, -math.inf
    x = x.to(BF).cuda()
    one, zero = torch.ones(16, 32, device="cuda"), torch.zeros(16, 32, device="cuda")
    for kind in (E4, I8):
        kv = _cache(pool, 1, 16, 64, kind)
        kv.v_scale.fill_(2.0 ** -7)
        K.paged_append(x, torch.ones_like(x), x, one, zero, kv, table, lens)
        at = table[:, 0].long()
        codes = R.values(kv.v)[at.cpu()]
        if kind == E4:
            assert kv.v_scale[at[0], 0] == 2.0 ** -8  # 1 <= 448 2^-8
            assert torch.isnan(codes[0, 0, 0, 3:5]).all() and torch.isnan(codes[1, 0, 4, 0])
            assert codes[0, 0, 0, 5] == 256
        else:
            assert kv.v_scale[at[0], 0] == 2.0 ** -6
            assert codes[0, 0, 0, 3] == 127 and codes[0, 0, 0, 4] == 0 and codes[1, 0, 4, 0] == -127


def test_append_tokens_without_a_place():
    """Slots not in use, positions before 0, behind the table and behind the
    angles, page numbers out of range: nothing else changes."""
    table, lens, cu, pool = _batch([1, 3, 1, 2, 1, 4], [0, 0, 40, 30, 20, 46], 16)
    kv = _cache(pool, 2, 16, 64, E4)
    lens[0], lens[1] = 0, 2                     # no token; three rows, two positions
    table[2, 2] = pool                          # position 40
    table[4, 1] = -5                            # position 20
    cos, sin = (t.cuda() for t in rope_tables(64, 49))  # the last sequence's 46 .. 49: one behind
    x = torch.randn(12, 8, 64, generator=_gen(2)).to(BF).cuda()
    q, k, v = x.split((4, 2, 2), 1)
    was = _clone(kv)
    got = K.paged_append(q, k, v, cos, sin, kv, table, lens, cu)
    _check_append(was, kv, q, k, v, cos, sin, table, lens, cu, got)
    assert not got[0].any() and not got[1].any() and torch.isnan(got[11]).all()
    now = _clone(kv)
    for far in (2 ** 31 - 1, -(2 ** 31)):
        K.paged_append(q, k, v, cos, sin, kv, table, torch.full_like(lens, far), cu)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(kv, now))


def test_append_strides_rows_left_alone_and_in_place():
    table, lens, cu, pool = _batch([2, 3], [60, 10], 32)
    cos, sin = (t.cuda() for t in rope_tables(64, 70))
    x = torch.randn(7, 8, 64, generator=_gen(4)).to(BF).cuda()
    caches = [_cache(pool, 2, 32, 64, E4) for _ in range(3)]
    parts = [t[:5].contiguous() for t in x.split((4, 2, 2), 1)]
    want = K.paged_append(*parts, cos, sin, caches[0], table, lens, cu)
    off = [torch.empty(t.numel() + 1, dtype=BF, device="cuda")[1:].view(t.shape).copy_(t) for t in parts]
    assert torch.equal(K.paged_append(*off, cos, sin, caches[1], table, lens, cu), want)
    q, k, v = x.split((4, 2, 2), 1)
    behind = q[5:].clone()
    assert K.paged_append(q, k, v, cos, sin, caches[2], table, lens, cu, out=q) is q
    assert torch.equal(q[:5], want) and torch.equal(q[5:], behind)
    for c in caches[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c, caches[0]))


# -------------------------------------------------------------- both, as used
def test_graph_replays_follow_lengths_and_tables():
    """One captured step, replayed as the sequences grow, against eager calls."""
    heads, dim, page, seqs = 4, 128, 16, 3
    g = _gen(6)
    kv, eager = (K.paged_kv(20, heads, page, dim) for _ in range(2))
    table = torch.randperm(18, generator=g).to(torch.int32).view(3, 6).cuda()
    lens = _ints([1, 1, 0])
    x = torch.empty(seqs, 3 * heads, dim, dtype=BF, device="cuda")
    cos, sin = (t.cuda() for t in rope_tables(dim, 96))

    def step(cache):
        q, k, v = x.split(heads, 1)
        return K.paged_attention(K.paged_append(q, k, v, cos, sin, cache, table, lens), cache, table, lens)

    step(eager)
    eager = K.paged_kv(20, heads, page, dim)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(kv)
    for i in range(40):
        x.copy_(torch.randn(x.shape, generator=g).to(BF))
        lens.copy_(_ints([i + 1, 2 * i + 1, 0 if i < 5 else i - 4]))
        if i % 2:
            torch.cuda.synchronize()
        want = step(eager)
        graph.replay()
        assert torch.equal(o, want), i
        assert torch.equal(_bits(kv.k), _bits(eager.k)) and torch.equal(kv.v_scale, eager.v_scale)


def test_another_stream():
    table, lens, cu, pool = _batch([1] * 3, [700, 90, 3000], 64)
    kv = _cache(pool, 2, 64, 128, E4)
    q = torch.randn(3, 4, 128, generator=_gen(5)).to(BF).cuda()
    want = K.paged_attention(q, kv, table, lens)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            got.append(K.paged_attention(q, kv, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)
