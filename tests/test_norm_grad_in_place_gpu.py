"""Gradients of the norms written over one of their inputs: the same bits as apart from them, whichever rows are on their way meanwhile."""
import pytest
import torch

from tests.test_norm_grad_gpu import BF16, F16, F32, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,hidden,shift", [(BF16, 256, 0), (F32, 256, 0), (BF16, 2048, 0), (F16, 4096, 0), (F32, 5120, 0), (BF16, 771, 0), (F16, 1024, 1), (F32, 130, 0), (BF16, 9000, 0)])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("which", ["x", "dy", "residual"])
def test_many_rows_in_place(dtype, hidden, shift, rms, which):
    x = inputs(6007, hidden, dtype, shift=shift)
    want = run(x, rms)
    got = run(x, rms, out=x[which])
    assert got[0] is x[which] and all(torch.equal(a, b) for a, b in zip(got, want))
