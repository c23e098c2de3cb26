"""The padding copy of bf16 rows (moc_copy_pad_2d): rows' ends at every place of a
16-byte chunk, and as many parts of rows as take two launches."""
import pytest
import torch

from moc_amd import _native as N

pytestmark = pytest.mark.gpu
BF, I16 = torch.bfloat16, torch.int16


def copy(src, dst, width):
    N.call("moc_copy_pad_2d", N.MOC_BF16, src.data_ptr(), *src.shape, src.stride(0), dst.data_ptr(), dst.stride(0), width,
           N.stream_of(src))


@pytest.mark.parametrize("cols", [*range(1, 18), *range(505, 530), 1023, 1025])
@pytest.mark.parametrize("ahead", [0, 1, 5])
def test_rows_ends(cols, ahead):
    rows, width = 7, (cols + 7) // 8 * 8 + 16
    held = torch.randint(1, 1 << 15, (rows, ahead + cols + 3), dtype=I16, device="cuda")
    src = held.view(BF)[:, ahead:ahead + cols]
    dst = torch.full((rows, width + 8), -1, dtype=I16, device="cuda")
    copy(src, dst.view(BF), width)
    assert torch.equal(dst[:, :cols], held[:, ahead:ahead + cols])
    assert not dst[:, cols:width].any() and (dst[:, width:] == -1).all()


def test_more_parts_than_a_launch_counts():
    rows = (1 << 30) + 5
    src = torch.randint(1, 1 << 15, (rows, 1), dtype=I16, device="cuda")
    dst = torch.full((rows, 8), -1, dtype=I16, device="cuda")
    copy(src.view(BF), dst.view(BF), 8)
    assert torch.equal(dst[:, :1], src)
    for part in dst.split(1 << 28):
        assert not part[:, 1:].any()
