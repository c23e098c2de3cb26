"""K.paged_append and K.paged_attention over rows of odd strides on axes of one
element, against contiguous ones."""
import pytest
import torch

from moc_amd import kernels as K
from moc_amd.inference.decode_model import rope_tables

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _odd(x):
    """x [1, heads, 64] as the first of rows of an odd pitch."""
    n = x.numel()
    wide = torch.zeros(3, n + 1, dtype=BF, device="cuda")
    wide[0, :n] = x.flatten()
    return wide[:, :n].unflatten(1, x.shape[1:])[:1]


def test_one_row_of_an_odd_pitch():
    g = torch.Generator().manual_seed(1)
    table, lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([[1, 0]], [20]))
    cos, sin = (t.cuda() for t in rope_tables(64, 32))
    q, k, v = (torch.randn(1, h, 64, generator=g).to(BF).cuda() for h in (4, 2, 2))
    caches = [K.paged_kv(2, 2, 16, 64) for _ in range(3)]
    want = K.paged_append(q, k, v, cos, sin, caches[0], table, lens)
    o = K.paged_attention(want, caches[0], table, lens)
    odd = [_odd(t) for t in (q, k, v)]
    assert torch.equal(K.paged_append(*odd, cos, sin, caches[1], table, lens), want)
    assert K.paged_append(*odd, cos, sin, caches[2], table, lens, out=odd[0]) is odd[0]
    assert torch.equal(odd[0], want) and torch.equal(K.paged_attention(odd[0], caches[1], table, lens), o)
    for c in caches[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c, caches[0]))
