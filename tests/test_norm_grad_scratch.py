"""Scratch of the norms' gradients: what their launches join, and no more. Long rows are summed in 64 shares, those that a CTA holds in up to 592."""
import pytest

from metalhlo_b200 import cuda


def need(rows, hidden):
    return cuda.lib.mhlo_cuda_norm_grad_scratch_bytes(rows, hidden)


@pytest.mark.parametrize("rows,hidden", [(100, 20000), (4096, 50257), (1 << 20, 1 << 17), (1000, 1 << 24)])
def test_long_rows(rows, hidden):
    """Statistics of each row, and sums of dy y and of dy in fp32 of each share."""
    assert need(rows, hidden) == rows * 16 + min(rows, 64) * 2 * hidden * 4


@pytest.mark.parametrize("rows,hidden", [(1, 1), (100, 64), (4096, 5120), (1 << 20, 16384)])
def test_rows_of_a_cta(rows, hidden):
    assert need(rows, hidden) >= min(rows, 592) * 2 * hidden * 4
