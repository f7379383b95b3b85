"""The policy loss where log probabilities lie so far apart that fp32 holds their difference to some whole units only, as with logits masked by -1e9."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FAR = [-1e9, -123456789.0, -3e7, -1e30, torch.finfo(torch.float32).min]


@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("tokens", [64, 40000])
def test_ratios_that_overflow_are_infinite_of_the_right_sign(far, tokens):
    from metalhlo_b200 import cuda

    near = -torch.linspace(0.5, 63.5, tokens, device="cuda")
    lost = torch.full_like(near, far)
    one = torch.ones_like(near)
    # exp(logprob - old) = infinity where the advantage is negative: not clipped, loss and gradient -infinity * a
    r = cuda.policy_loss(near, lost, -one)
    assert (r.grad == math.inf).all() and float(r.loss) == math.inf
    # exp(logprob - old) = 0: clipped where the advantage is negative, else a ratio of 0
    r = cuda.policy_loss(lost, near, -one)
    assert not r.grad.any() and abs(float(r.loss) - 0.8) < 1e-6
    r = cuda.policy_loss(lost, near, one)
    assert not r.grad.any() and float(r.loss) == 0
    # exp(ref - logprob) - 1 = infinity, and its negative is the gradient; the ratio is 1
    r = cuda.policy_loss(lost, lost, one, ref_logprobs=near, kl_weight=0.1)
    assert float(r.kl) == math.inf and (r.grad == -math.inf).all()
    # exp(ref - logprob) = 0: k3 = logprob - ref - 1, of the gradient kl_weight is left beside -a
    r = cuda.policy_loss(near, near, one, ref_logprobs=lost, kl_weight=0.5)
    want = (near.double() - lost.double() - 1).mean()
    assert abs(float(r.kl) / float(want) - 1) <= 2.0 ** -20
    assert ((r.grad.double() * tokens + 0.5).abs() <= 2.0 ** -20).all()
