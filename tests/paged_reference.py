"""Plain forms, in 64 bits on the CPU, of the operators over a paged 8-bit cache
and of token sampling: loops over sequences, pages and words, from the
definitions."""
import math

import numpy as np
import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def values(codes: torch.Tensor) -> torch.Tensor:
    """What the codes stand for, without their scales."""
    return codes.cpu().to(torch.float64) if codes.dtype == torch.int8 else codes.cpu().float().double()


def spans(tokens, lens, cu):
    """(sequence, its rows' start, rows, tokens in the cache) of a batch."""
    lens = lens.tolist()
    cu = list(range(len(lens) + 1)) if cu is None else cu.tolist()
    return [(b, cu[b], cu[b + 1] - cu[b], lens[b]) for b in range(len(lens))]


def rotate(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def rotated(x, cos, sin, lens, cu):
    """Rows of x [tokens, heads, dim] turned by their positions; 0 before
    position 0, NaN behind the angles, None rows where no sequence has them."""
    x, cos, sin = x.cpu().double(), cos.cpu().double(), sin.cpu().double()
    y = torch.full_like(x, math.nan)
    for _, start, n, length in spans(x.shape[0], lens.cpu(), None if cu is None else cu.cpu()):
        for i in range(n):
            pos = length - n + i
            if pos < 0:
                y[start + i] = 0
            elif pos < cos.shape[0]:
                y[start + i] = rotate(x[start + i], cos[pos], sin[pos])
    return y


def round_codes(y, kind):
    """y on the codes' grid: nearest, ties to even."""
    if kind == torch.int8:
        return torch.round(y).clamp(-127, 127)
    e = torch.floor(torch.log2(y.abs().clamp(min=1e-300))).clamp(min=-6)
    step = 2.0 ** (e - 3)
    return torch.round(y / step) * step


def half_step(y, kind):
    """Half the distance of neighbouring codes at y."""
    if kind == torch.int8:
        return torch.full_like(y, 0.5)
    e = torch.floor(torch.log2(y.abs().clamp(min=1e-300))).clamp(min=-6)
    return 2.0 ** (e - 4)


def attention(q, kv, table, lens, cu, scale, rows=None):
    """(o, the same sums over |v|) in 64 bits; NaN for rows that see a position
    without a page.  rows: only these."""
    q, table = q.cpu().double(), table.cpu()
    codes_k, codes_v = values(kv.k), values(kv.v)
    ks, vs = kv.k_scale.cpu().double(), kv.v_scale.cpu().double()
    tokens, heads, dim = q.shape
    pages, kv_heads, page, _ = codes_k.shape
    room = table.shape[1] * page
    o, size = torch.zeros_like(q), torch.zeros_like(q)
    for b, start, n, length in spans(tokens, lens.cpu(), None if cu is None else cu.cpu()):
        for i in range(n):
            sees = length - n + i + 1
            if sees <= 0 or (rows is not None and start + i not in rows):
                continue
            ids = [int(table[b, p // page]) if p < room else -1 for p in range(0, sees, page)]
            if any(not 0 <= j < pages for j in ids):
                o[start + i] = size[start + i] = math.nan
                continue
            k = (codes_k[ids] * ks[ids][..., None, None]).transpose(0, 1).reshape(kv_heads, -1, dim)[:, :sees]
            v = (codes_v[ids] * vs[ids][..., None, None]).transpose(0, 1).reshape(kv_heads, -1, dim)[:, :sees]
            for h in range(heads):
                g = h // (heads // kv_heads)
                p = torch.softmax(scale * (k[g] @ q[start + i, h]), 0)
                o[start + i, h] = p @ v[g]
                size[start + i, h] = p @ v[g].abs()
    return o, size


def sample(x, u, temperature, top_k, top_p, min_p):
    """(id, how far the draw is from the nearest border, as a share of the weight)."""
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    best = x.max()
    if best == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == best, 1.0, np.exp((x - best) / temperature))
    order = np.lexsort((np.arange(len(x)), -x))
    if top_k > 0:
        order = order[:top_k]
    near = 1.0
    if top_p < 1:
        mass = np.cumsum(w[order])
        ahead = np.concatenate(([0.0], mass[:-1])) / mass[-1]
        near = np.abs(ahead[1:] - top_p).min() if len(order) > 1 else 1.0
        order = order[:max(1, int((ahead < top_p).sum()))]
    order = np.sort(order[w[order] >= min(min_p, 1.0)])
    mass = np.cumsum(w[order])
    near = min(near, np.abs(mass / mass[-1] - u).min() if u < 1 else 1.0)
    return int(order[min(len(order) - 1, int((mass <= u * mass[-1]).sum()))]), near
