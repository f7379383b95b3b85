"""What attention over packed sequences refuses, without a GPU: arguments are checked before any CUDA call, so the addresses are never followed."""
import ctypes as C

import pytest

from metalhlo_b200 import cuda

P = 1 << 20  # an aligned address that is never read
OK, UNSUPPORTED, INVALID = 0, 4, 10
Q, K = cuda._i64s([4 * 64, 64]), cuda._i64s([2 * 64, 64])


def batch(**kw):
    f = dict(starts=P, plan=P, seqs=3, tokens=100, q_heads=4, kv_heads=2, causal=1)
    f.update(kw)
    return cuda.PackedBatchArgs(**f)


def attention(b=None, dtype=cuda.BF16, dim=64, scale=0.1, q=P, qs=Q, k=P, ks=K, v=P, vs=K, o=P, os=Q):
    return cuda.lib.mhlo_cuda_packed_attention(dtype, C.byref(b or batch()), dim, scale, q, qs, k, ks, v, vs, o, os, None, None)


def grad(b=None, dtype=cuda.BF16, dim=64, scale=0.1, q=P, qs=Q, k=P, ks=K, v=P, vs=K, o=P, os=Q, lse=P, g=P, gs=Q, dq=P, dqs=Q, dk=P, dks=K, dv=P, dvs=K, scratch=P, size=1 << 40):
    return cuda.lib.mhlo_cuda_packed_attention_grad(dtype, C.byref(b or batch()), dim, scale, q, qs, k, ks, v, vs, o, os, lse, g, gs, dq, dqs, dk, dks, dv, dvs, scratch, size, None)


@pytest.mark.parametrize("call", [attention, grad])
@pytest.mark.parametrize("want,kw,text", [
    (INVALID, dict(seqs=-1), "sequences"), (INVALID, dict(tokens=-1), "tokens"), (INVALID, dict(seqs=1 << 25), "sequences"), (INVALID, dict(tokens=1 << 31), "tokens"),
    (INVALID, dict(q_heads=3), "3 query heads on 2"), (INVALID, dict(kv_heads=0), "heads"), (INVALID, dict(q_heads=0), "heads"), (INVALID, dict(q_heads=70000, kv_heads=70000), "heads"),
    (UNSUPPORTED, dict(tokens=(1 << 28) + 1), "up to 2^30 rows"), (INVALID, dict(plan=None), "plan"), (INVALID, dict(plan=P + 8), "plan")])
def test_batch(call, want, kw, text):
    assert call(batch(**kw)) == want
    assert text in cuda.last_error()


@pytest.mark.parametrize("call", [attention, grad])
def test_call(call):
    assert call(dtype=cuda.F64) == UNSUPPORTED and call(dtype=cuda.I8) == UNSUPPORTED
    for dim in (0, -8, 129, 256):
        assert call(dim=dim) == UNSUPPORTED and "head dimension" in cuda.last_error()
    for scale in (0.0, -1.0, float("nan"), float("inf"), 2e38):
        assert call(scale=scale) == UNSUPPORTED and "scale" in cuda.last_error()
    for name in ("q", "k", "v", "o"):
        assert call(**{name: None}) == INVALID and f"null {name}" in cuda.last_error()
        assert call(**{name + "s": None}) == INVALID
        assert call(**{name + "s": cuda._i64s([-256, 64])}) == UNSUPPORTED and "negative" in cuda.last_error()
    assert call(batch(seqs=0)) == OK and call(batch(tokens=0)) == OK


def test_results_that_overlap():
    assert attention(os=cuda._i64s([255, 64])) == INVALID and "rows of o overlap" in cuda.last_error()
    assert attention(os=cuda._i64s([0, 64])) == INVALID and attention(os=cuda._i64s([256, 0])) == INVALID
    assert grad(dqs=cuda._i64s([256, 63])) == INVALID and "dq" in cuda.last_error()
    assert grad(dks=cuda._i64s([64, 64])) == INVALID and "dk" in cuda.last_error()
    assert grad(dvs=cuda._i64s([0, 64])) == INVALID and "dv" in cuda.last_error()


def test_grad():
    for name in ("g", "dq", "dk", "dv", "lse"):
        assert grad(**{name: None}) == INVALID
    need = cuda.lib.mhlo_cuda_packed_attention_grad_scratch_bytes(cuda.BF16, C.byref(batch()), 64)
    assert need >= 100 * 4 * 8
    assert grad(size=need - 1) == INVALID and "scratch" in cuda.last_error()
    assert grad(scratch=None) == INVALID and grad(scratch=P + 4) == INVALID
    assert cuda.lib.mhlo_cuda_packed_attention_grad_scratch_bytes(cuda.BF16, None, 64) == 0 and cuda.lib.mhlo_cuda_packed_attention_grad_scratch_bytes(cuda.BF16, C.byref(batch()), 0) == 0


def test_plan():
    assert cuda.lib.mhlo_cuda_packed_plan_bytes(None) == 0 and cuda.lib.mhlo_cuda_packed_plan_bytes(C.byref(batch(q_heads=3))) == 0
    # every sequence may end inside a tile of 2 x 64 tokens (two query heads to a head of keys), and inside one of 128 keys
    assert cuda.lib.mhlo_cuda_packed_plan_bytes(C.byref(batch(seqs=5, tokens=1000))) >= 16 * (1000 // 128 + 5 + 1000 // 128 + 5)
    assert cuda.lib.mhlo_cuda_packed_plan(C.byref(batch(starts=None)), None) == INVALID
    assert cuda.lib.mhlo_cuda_packed_plan(C.byref(batch(plan=P + 4)), None) == INVALID
    assert cuda.lib.mhlo_cuda_packed_plan(C.byref(batch(seqs=0, starts=None, plan=None)), None) == OK


def test_views():
    torch = pytest.importorskip("torch")
    with pytest.raises(AssertionError):
        cuda.packed_plan(torch.zeros(3, dtype=torch.int32), 10, 2, 2)  # not on a GPU
