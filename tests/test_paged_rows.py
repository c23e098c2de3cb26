"""Rows whose strides the kernels cannot take, though torch calls them contiguous:
an axis of one element may have any stride."""
import pytest
import torch

from moc_amd import kernels as K

from test_paged_refusals import BF, I32, _args, _attention, _kv, calls  # noqa: F401


def _one_row(heads):
    """The first of three rows of an odd pitch: [1, heads, 64]."""
    return torch.zeros(3, heads * 64 + 1, dtype=BF)[:, :heads * 64].unflatten(1, (heads, 64))[:1]


def _one_head(tokens):
    """[tokens, 1, 64] whose head axis has a stride of one."""
    return torch.zeros(tokens * 64, dtype=BF).as_strided((tokens, 1, 64), (64, 1, 1))


@pytest.mark.parametrize("rows", [_one_row(4), _one_head(3)], ids=["one row", "one head"])
def test_axes_of_one_element_may_have_any_stride(calls, rows):  # noqa: F811
    assert rows.is_contiguous() and (rows.stride(0) | rows.stride(1)) % 8
    n, heads = rows.shape[:2]
    ones = dict(table=torch.zeros(n, 2, dtype=I32), lens=torch.zeros(n, dtype=I32))
    kv_heads = 1 if heads == 1 else 2
    codes = lambda: torch.zeros(6, kv_heads, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    a = _args(q=rows, k=torch.zeros(n, kv_heads, 64, dtype=BF), v=torch.zeros(n, kv_heads, 64, dtype=BF),
              kv=_kv(k=codes(), v=codes(), k_scale=torch.zeros(6, kv_heads), v_scale=torch.zeros(6, kv_heads)), **ones)
    if heads == 1:
        a.update(k=rows, v=rows)
    for out in (None, rows):
        calls.clear()
        K.paged_append(**a, out=out)
        K.paged_attention(**_attention(a), out=out)
        (_, append), (_, attention) = calls
        for strides in (append[1:3], append[4:6], append[7:9], append[-3:-1], attention[1:3], attention[-5:-3]):
            assert all(s % 8 == 0 for s in strides), strides
        assert out is None or append[-4] == attention[-6] == rows.data_ptr()
