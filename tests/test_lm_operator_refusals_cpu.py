"""What the key/value cache, the attention over it and the log probabilities refuse, without a GPU: arguments are checked before any
CUDA call, so the addresses here are never followed."""
import ctypes as C

import pytest

from metalhlo_b200 import cuda

P = 1 << 20  # an aligned address that is never read
OK, UNSUPPORTED, INVALID = 0, 4, 10


def cache(**kw):
    f = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, pages=8, heads=2, page_tokens=16, head_dim=64)
    f.update(kw)
    return cuda.KvCacheArgs(**f)


def batch(**kw):
    f = dict(page_table=P, lengths=P, token_starts=P, seqs=3, pages_per_seq=4, table_stride=4, tokens=7)
    f.update(kw)
    return cuda.KvBatchArgs(**f)


STRIDES = cuda._i64s([128, 64, 1])


def append(c=None, b=None, dtype=cuda.BF16, k=P, v=P, ks=STRIDES, vs=STRIDES, q=P, qs=STRIDES, o=P, os=STRIDES, q_heads=2, rope=P, positions=64, rotary=64):
    return cuda.lib.mhlo_cuda_kv_cache_append(dtype, C.byref(c or cache()), C.byref(b or batch()), k, ks, v, vs, q, qs, o, os, q_heads, rope, positions, rotary, 0, None)


def attention(c=None, b=None, dtype=cuda.F16, q=P, qs=STRIDES, q_heads=4, scale=0.1, o=P, os=STRIDES, scratch=P, size=1 << 40):
    return cuda.lib.mhlo_cuda_cached_attention(dtype, q, qs, C.byref(c or cache()), C.byref(b or batch()), q_heads, scale, o, os, None, scratch, size, None)


def read(c=None, b=None, dtype=cuda.F32, most=5, k=P, v=P, s=STRIDES):
    return cuda.lib.mhlo_cuda_kv_cache_read(dtype, C.byref(c or cache()), C.byref(b or batch()), most, k, v, s, None)


@pytest.mark.parametrize("call", [append, attention, read])
@pytest.mark.parametrize("want,c,b,text", [
    (UNSUPPORTED, dict(page_tokens=48), {}, "48 tokens in a page"), (UNSUPPORTED, dict(page_tokens=0), {}, "tokens in a page"),
    (UNSUPPORTED, dict(head_dim=72), {}, "head dimension 72"), (UNSUPPORTED, dict(head_dim=512), {}, "head dimension"),
    (INVALID, dict(k_codes=None), {}, "null pointer"), (INVALID, dict(v_scales=None), {}, "null pointer"), (INVALID, dict(v_codes=P + 8), {}, "aligned"),
    (INVALID, dict(pages=0), {}, "0 pages"), (INVALID, dict(heads=-1), {}, "heads"), (INVALID, {}, dict(seqs=-1), "sequences"),
    (INVALID, {}, dict(table_stride=3), "apart"), (INVALID, {}, dict(lengths=None), "null lengths"), (INVALID, {}, dict(page_table=None), "page table"),
    (INVALID, {}, dict(tokens=-1), "tokens"), (INVALID, {}, dict(pages_per_seq=1 << 40, table_stride=1 << 40), "pages a sequence")])
def test_cache_and_batch(call, want, c, b, text):
    assert call(cache(**c), batch(**b)) == want
    assert text in cuda.last_error()


@pytest.mark.parametrize("call", [append, attention])
def test_rows_need_starts_unless_there_is_one_each(call):
    assert call(b=batch(token_starts=None)) == INVALID and "token_starts" in cuda.last_error()


def test_append():
    assert append(dtype=cuda.I8) == UNSUPPORTED
    assert append(k=None) == INVALID and append(v=None) == INVALID
    assert append(ks=cuda._i64s([-128, 64])) == UNSUPPORTED and append(vs=None) == INVALID
    assert append(rope=None) == INVALID and "rotation table" in cuda.last_error()
    assert append(rotary=24) == UNSUPPORTED and append(rotary=128) == UNSUPPORTED and append(rotary=0) == UNSUPPORTED
    assert append(positions=0) == INVALID and append(rope=P + 4) == INVALID
    assert append(o=None) == INVALID and append(q_heads=0) == INVALID
    assert append(os=cuda._i64s([256, 64])) == INVALID and "in place" in cuda.last_error()
    assert append(b=batch(tokens=0)) == OK and append(b=batch(seqs=0)) == OK


def test_attention():
    assert attention(dtype=cuda.F64) == UNSUPPORTED
    assert attention(cache(head_dim=80)) == UNSUPPORTED and "head dimension 80" in cuda.last_error()
    assert attention(q_heads=3) == INVALID and attention(q_heads=0) == INVALID
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attention(scale=scale) == UNSUPPORTED
    assert attention(q=None) == INVALID and attention(o=None) == INVALID
    assert attention(os=cuda._i64s([256, 64])) == INVALID
    long = batch(pages_per_seq=400, table_stride=400)
    need = cuda.lib.mhlo_cuda_cached_attention_scratch_bytes(C.byref(cache()), C.byref(long), 4)
    assert need > 0 and cuda.lib.mhlo_cuda_cached_attention_scratch_bytes(None, None, 4) == 0
    assert attention(b=long, size=need - 1) == INVALID and attention(b=long, scratch=None) == INVALID and attention(b=long, scratch=P + 8) == INVALID
    assert attention(b=batch(tokens=0), scratch=None, size=0) == OK


def test_read():
    assert read(dtype=cuda.I32) == UNSUPPORTED and read(most=-1) == INVALID
    assert read(s=cuda._i64s([1, 2, -3])) == UNSUPPORTED
    assert read(k=None, v=None) == OK and read(most=0) == OK


def logprobs(dtype=cuda.F16, x=P, stride=100, rows=4, vocab=100, scale=1.0, t=P, tt=cuda.I64, lp=P, k=0, tl=None, ti=None):
    return cuda.lib.mhlo_cuda_token_logprobs(dtype, x, stride, rows, vocab, scale, t, tt, lp, None, None, k, tl, ti, None)


def gradient(dtype=cuda.F16, x=P, stride=100, rows=4, vocab=100, scale=1.0, t=P, tt=cuda.I64, lse=P, h=P, g=P, e=P, k=0, ids=None, gt=None, dx=P, dstride=100):
    return cuda.lib.mhlo_cuda_token_logprobs_grad(dtype, x, stride, rows, vocab, scale, t, tt, lse, h, g, e, k, ids, gt, dx, dstride, None)


@pytest.mark.parametrize("call", [logprobs, gradient])
def test_logits(call):
    assert call(dtype=cuda.F64) == UNSUPPORTED and call(rows=-1) == INVALID and call(vocab=0) == INVALID
    assert call(stride=99) == INVALID and call(x=None) == INVALID and call(tt=cuda.I16) == UNSUPPORTED
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == UNSUPPORTED
    assert call(k=33) == UNSUPPORTED and call(k=-1) == UNSUPPORTED and call(k=6, vocab=5) == UNSUPPORTED
    assert call(rows=0) == OK


def test_logprobs_and_gradient_arguments_that_go_together():
    assert logprobs(lp=None) == INVALID and logprobs(t=None) == INVALID and logprobs(k=2, ti=P) == INVALID
    assert gradient(lse=None) == INVALID and gradient(dx=None) == INVALID and gradient(t=None) == INVALID and gradient(h=None) == INVALID
    assert gradient(gt=P) == INVALID and gradient(gt=P, k=2) == INVALID
    assert gradient(dstride=99) == INVALID and gradient(dstride=200) == INVALID


def test_python_views_refuse_before_the_library():
    import torch

    codes, scales = torch.zeros(2, 1, 16, 64, dtype=torch.int8), torch.zeros(2, 1)
    with pytest.raises(AssertionError):
        cuda.KvCache(codes, codes, scales, scales)  # not on a GPU
    with pytest.raises(AssertionError):
        cuda.token_logprobs(torch.zeros(2, 5))
    table = cuda.rope_table(1 << 20, 64, device="cpu")
    assert table.shape == (1 << 20, 64) and table.dtype == torch.float32
    # far positions keep their angle: 32-bit angles are off by 0.03 there
    import math

    assert abs(float(table[1048575, 0]) - math.cos(1048575.0)) < 1e-7 and abs(float(table[1048575, 32 + 1]) - math.sin(1048575.0 * 10000.0 ** (-2 / 64))) < 1e-7


def test_what_32_bits_cannot_hold_is_refused():
    assert attention(scale=2e38) == UNSUPPORTED and logprobs(scale=2e38) == UNSUPPORTED and gradient(scale=2e38) == UNSUPPORTED
    assert attention(b=batch(tokens=1 << 29, seqs=1 << 20, token_starts=P), q_heads=4) == UNSUPPORTED


def test_rows_of_logits():
    import torch

    x = torch.zeros(4, 3, 50)
    assert cuda._logit_rows(x) == (12, 50) and cuda._logit_rows(x[0, 0]) == (1, 50) and cuda._logit_rows(x[..., :7]) == (12, 50)
    assert cuda._logit_rows(x[:, 1:2]) == (4, 150) and cuda._logit_rows(x[:, 1]) == (4, 150) and cuda._logit_rows(x[:0]) == (0, 50)
    assert cuda._logit_rows(x[..., :1]) == (12, 50) and cuda._logit_rows(x[:1, :1, :9]) == (1, 9)
    for bad in (x[0, 0].expand(4, 50), x[:, :2], x.transpose(1, 2), x.transpose(0, 1), x.as_strided((4, 50), (10, 1))):
        with pytest.raises(AssertionError):
            cuda._logit_rows(bad)
