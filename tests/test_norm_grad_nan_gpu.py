"""A NaN in a row of x: no kernel of the norms' gradients may turn its sum of squares into a number."""
import math

import pytest
import torch

from tests.test_norm_grad_gpu import BF16, F32, inputs, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hidden", [64, 600, 1001, 1024, 4096, 9000, 17000])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_nan_in_a_row_reaches_all_of_it(hidden, rms, dtype):
    """r of the row is NaN, and with it the whole row of dx and, through dy y, all of dgamma; other rows of dx and dbeta do not depend on it."""
    x = inputs(40, hidden, dtype)
    want = run(x, rms)
    x["x"][7, hidden // 3] = math.nan
    got = run(x, rms)
    rows = torch.arange(40, device="cuda") != 7
    assert torch.equal(got[0][rows], want[0][rows]) and got[0][7].isnan().all()
    assert got[1].isnan().all()
    if not rms:
        assert torch.equal(got[2], want[2])
