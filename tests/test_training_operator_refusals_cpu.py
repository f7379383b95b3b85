"""What the gradients of the norms and the policy loss refuse, without a GPU: arguments are checked before any CUDA call."""
import ctypes as C

import pytest

from metalhlo_b200 import cuda

P = 1 << 20  # an aligned address that is never read
UNSUPPORTED, INVALID = 4, 10


def layer(dtype=cuda.BF16, x=P, gamma=P, dy=P, residual=None, dx=P, rows=10, hidden=64, eps=1e-5, scratch=P, size=1 << 40):
    return cuda.lib.mhlo_cuda_layer_norm_grad(dtype, x, gamma, dy, residual, dx, P, P, rows, hidden, eps, scratch, size, None)


def rms(dtype=cuda.BF16, x=P, gamma=P, dy=P, residual=None, dx=P, rows=10, hidden=64, eps=1e-5, scratch=P, size=1 << 40):
    return cuda.lib.mhlo_cuda_rms_norm_grad(dtype, x, gamma, dy, residual, dx, P, rows, hidden, eps, scratch, size, None)


@pytest.mark.parametrize("call", [layer, rms])
def test_norms(call):
    assert call(dtype=cuda.F64) == UNSUPPORTED
    for name in ("x", "dy", "dx"):
        assert call(**{name: None}) == INVALID and "null" in cuda.last_error()
    for kw in (dict(rows=-1), dict(hidden=0), dict(hidden=-8), dict(rows=1 << 31), dict(hidden=(1 << 24) + 1)):
        assert call(**kw) == INVALID and "rows of" in cuda.last_error()
    for eps in (-1e-5, float("nan")):
        assert call(eps=eps) == INVALID and "eps" in cuda.last_error()
    need = cuda.lib.mhlo_cuda_norm_grad_scratch_bytes(10, 64)
    assert need > 0 and cuda.lib.mhlo_cuda_norm_grad_scratch_bytes(-1, 64) == 0 and cuda.lib.mhlo_cuda_norm_grad_scratch_bytes(4, 0) == 0
    assert call(size=need - 1) == INVALID and "scratch" in cuda.last_error()
    assert call(scratch=None) == INVALID and call(scratch=P + 8) == INVALID


def policy(grad=P, results=P, scratch=P, size=1 << 40, **kw):
    f = dict(logprobs=P, old_logprobs=P, ref_logprobs=P, advantages=P, mask=P, starts=P, tokens=100000, seqs=7, clip_low=0.2, clip_high=0.2, kl_weight=0.1)
    f.update(kw)
    return cuda.lib.mhlo_cuda_policy_loss(C.byref(cuda.PolicyBatchArgs(**f)), grad, results, scratch, size, None)


def test_policy_loss():
    for kw in (dict(tokens=-1), dict(seqs=-1), dict(tokens=(1 << 30) + 1), dict(seqs=(1 << 24) + 1)):
        assert policy(**kw) == INVALID and "sequences" in cuda.last_error()
    for kw in (dict(clip_low=-0.1), dict(clip_low=1.0), dict(clip_low=float("nan")), dict(clip_high=-0.1), dict(clip_high=float("inf")), dict(clip_high=float("nan"))):
        assert policy(**kw) == INVALID and "clipped" in cuda.last_error()
    assert policy(kl_weight=float("nan")) == INVALID and policy(ref_logprobs=None) == INVALID and "without ref_logprobs" in cuda.last_error()
    for kw in (dict(logprobs=None), dict(old_logprobs=None), dict(advantages=None), dict(grad=None), dict(results=None)):
        assert policy(**kw) == INVALID and "null" in cuda.last_error()
    need = cuda.lib.mhlo_cuda_policy_loss_scratch_bytes(100000, 7)
    assert need > 0 and cuda.lib.mhlo_cuda_policy_loss_scratch_bytes(1000, 7) == 0 and cuda.lib.mhlo_cuda_policy_loss_scratch_bytes(-1, 7) == 0
    assert policy(size=need - 1) == INVALID and "scratch" in cuda.last_error()
    assert policy(scratch=None) == INVALID and policy(scratch=P + 4) == INVALID
    assert cuda.lib.mhlo_cuda_policy_loss(None, P, P, P, 1 << 40, None) == INVALID
