"""What the linear losses ask for beside their operands."""
import pytest

from moc_amd import _native as N


@pytest.mark.parametrize("rows,d,vocab", [(500, 256, 128256), (1024, 768, 50257), (2048, 768, 50048), (2048, 4096, 128256),
                                          (4096, 1024, 32000), (8192, 512, 32000), (64, 512, 32000), (3, 5, 7)])
@pytest.mark.parametrize("grads", [False, True])
def test_parts_of_f32_products(rows, d, vocab, grads):
    """Parts of a K split: 64 MiB at most, not up to 16 times dweight."""
    assert N.query("moc_linear_loss_gemm_workspace_size", N.MOC_F32, rows, d, vocab, grads) <= 4096 + (64 << 20)


def test_small_f32_products_still_split():
    assert N.query("moc_linear_loss_gemm_workspace_size", N.MOC_F32, 512, 512, 32000, True) > 4096
