"""Gradients of attention over packed sequences against the formula in 64 bits and against differences."""
import math

import pytest
import torch

from tests.packed_reference import check, inputs, reference

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(x, scale, causal, poison=7.0, out=None):
    from metalhlo_b200 import cuda

    plan = cuda.packed_plan(x["starts_dev"], x["rows"], x["q"].shape[1], x["k"].shape[1], causal)
    o, lse = torch.full(x["q"].shape, math.nan, dtype=x["q"].dtype, device="cuda"), torch.full(x["q"].shape[:2], math.nan, device="cuda")
    cuda.packed_attention(x["q"], x["k"], x["v"], plan, scale, out=o, lse=lse)
    grads = [torch.full(x[n].shape, poison, dtype=x[n].dtype, device="cuda") for n in ("q", "k", "v")] if out is None else out
    cuda.packed_attention_grad(x["q"], x["k"], x["v"], o, lse, x["grad"], plan, scale, *grads)
    assert cuda.device_error() == 0
    return grads


def compare(x, scale, causal):
    grads = run(x, scale, causal)
    end = x["starts"][-1]
    assert all((g[end:] == 7.0).all() for g in grads)  # rows of no sequence are left alone
    y = dict(x, **{n: x[n][:end] for n in ("q", "k", "v", "grad")})
    want, off = reference(y, scale, causal)
    check({n: g[:end] for n, g in zip(("dq", "dk", "dv"), grads)}, want, off, ("dq", "dk", "dv"))


LENGTHS = [[1], [2, 0, 3], [127, 1, 128], [129, 255], [256, 257, 1, 0], [513, 40], [1025, 300, 31]]


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 128), (BF16, 64), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("heads", [(2, 2), (4, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(dtype, dim, heads, causal, lengths):
    compare(inputs(lengths, *heads, dim, dtype, spare=5), dim ** -0.5, causal)


@pytest.mark.parametrize("q_heads,kv_heads", [(3, 1), (14, 2), (10, 2), (16, 1), (48, 1), (65, 1), (128, 1), (130, 1)])
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128), (F32, 64)])
def test_groups(q_heads, kv_heads, dtype, dim):
    compare(inputs([130, 77, 3], q_heads, kv_heads, dim, dtype, spare=1), dim ** -0.5, True)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 72, 80, 96, 104, 120, 1, 7, 33, 100, 127])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_head_dimensions(dim, dtype):
    compare(inputs([200, 65], 4, 2, dim, dtype), dim ** -0.5, True)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_tiles(dtype):
    compare(inputs([37 * i % 700 for i in range(40)], 6, 3, 64, dtype), 0.125, True)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F16, 64)])
def test_a_long_sequence(dtype, dim):
    compare(inputs([4500], 2, 1, dim, dtype), dim ** -0.5, True)


@pytest.mark.parametrize("grad_size", [2.0 ** -18, 1e-3, 3e3])
@pytest.mark.parametrize("dim", [64, 128])
def test_small_and_large_gradients_in_fp16(grad_size, dim):
    """Products of weights of a thousandth and such gradients lie below what fp16 holds, or above it."""
    compare(inputs([900, 120], 4, 2, dim, F16, grad_size=grad_size), dim ** -0.5, True)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 64)])
def test_peaked_weights(dtype, dim):
    compare(inputs([300, 140], 4, 2, dim, dtype, size=12.0), dim ** -0.5, True)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 64)])
def test_other_sequences_infinities(dtype, dim):
    x = inputs([100, 30, 129, 5], 4, 2, dim, dtype, spare=3)
    y = {n: t.clone() if torch.is_tensor(t) else t for n, t in x.items()}
    for n in ("q", "k", "v", "grad"):
        y[n][100:130] = math.inf if n in ("v", "grad") else math.nan
    z = {n: t.clone() if torch.is_tensor(t) else t for n, t in x.items()}
    for n in ("v", "grad"):
        z[n][100:130] = 0
    for a, b in zip(run(z, 0.1, True), run(y, 0.1, True)):
        for rows in (slice(0, 100), slice(130, 264)):
            assert torch.equal(a[rows], b[rows])
        assert torch.isnan(b[100:130]).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_the_same_bits_every_time(dtype):
    x = inputs([700, 90, 300], 4, 2, 64, dtype)
    first = run(x, 0.125, True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run(x, 0.125, True)))


@pytest.mark.parametrize("causal", [True, False])
def test_differences(causal):
    """fp32 gradients against central differences of the forward half in 64 bits, along random directions."""
    x = inputs([70, 1, 33], 4, 2, 16, F32)
    grads = run(x, 0.25, causal)

    def value(at):
        return float((reference(dict(x, **at), 0.25, causal)[0]["o"] * x["grad"].double()).sum())

    g = torch.Generator(device="cuda").manual_seed(5)
    for n, grad in zip(("q", "k", "v"), grads):
        way = torch.randn(x[n].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        # the reference takes its inputs to 64 bits itself; steps below fp32 need them there already
        up, down = (value({n: x[n].double() + s * h * way}) for s in (1, -1))
        got, slope = float((grad.double() * way).sum()), (up - down) / (2 * h)
        # fp32 sums of the gradient: 2^-20 of its size; differences: h^2 of the third derivative, and 2^-52 of the value over h
        assert abs(got - slope) <= 2.0 ** -20 * float((grad.double().abs() * way.abs()).sum()) + 1e-6 * max(1.0, abs(slope))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(dtype):
    x = inputs([150, 60], 4, 2, 64, dtype)
    tokens = x["rows"]
    want = run(x, 0.125, True)

    def laid(t, how):
        if how == "heads first":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        pitch = 72 if how == "wide" else 65
        odd = torch.full((tokens * t.shape[1] * pitch + 1,), math.nan, dtype=dtype, device="cuda")
        odd = (odd[1:] if how == "odd" else odd[:-1]).view(tokens, t.shape[1], pitch)[..., :64]
        odd.copy_(t)
        return odd

    for how in ("heads first", "wide", "odd"):
        y = dict(x, **{n: laid(x[n], how) for n in ("q", "k", "v", "grad")})
        out = [laid(torch.zeros_like(t), how) for t in want]
        got = run(y, 0.125, True, out=out)
        if how == "odd" and dtype != F32:  # the FMA units' kernels
            ref, off = reference(x, 0.125, True)
            check(dict(zip(("dq", "dk", "dv"), got)), ref, off, ("dq", "dk", "dv"))
        else:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one head of keys for all by a stride of zero: each head's share of the gradient
    y = dict(x, k=x["k"][:, :1].expand(-1, 2, -1), v=x["v"][:, :1].expand(-1, 2, -1))
    ref, off = reference(y, 0.125, True)
    check(dict(zip(("dq", "dk", "dv"), run(y, 0.125, True, out=[torch.empty_like(t) for t in want]))), ref, off, ("dq", "dk", "dv"))


@pytest.mark.parametrize("bits", [0x7fffffff, 0x7f800001, -1])
@pytest.mark.parametrize("where", ["q", "k", "v", "grad"])
def test_every_nan_counts(bits, where):
    """fp32 goes through the products in two parts: neither may turn a NaN into a number, whatever its bits."""
    from metalhlo_b200 import cuda

    x = inputs([90, 40], 4, 2, 64, F32)
    plan = cuda.packed_plan(x["starts_dev"], x["rows"], 4, 2, True)
    bad = {n: x[n].clone() for n in ("q", "k", "v", "grad")}
    bad[where].view(torch.int32)[20, 0, 7] = bits
    lse = torch.empty(130, 4, device="cuda")
    o = cuda.packed_attention(bad["q"], bad["k"], bad["v"], plan, 0.125, lse=lse)
    dq, dk, dv = cuda.packed_attention_grad(bad["q"], bad["k"], bad["v"], o, lse, bad["grad"], plan, 0.125)
    nan = {n: t.isnan() for n, t in dict(o=o, dq=dq, dk=dk, dv=dv).items()}
    if where == "q":
        assert nan["o"][20, 0].all() and nan["dq"][20, 0].all() and nan["dk"][:21, 0].all() and nan["dv"][:21, 0].all()
    elif where == "k":
        assert nan["o"][20:90, :2].all() and nan["dq"][20:90, :2].all() and nan["dk"][20, 0].all() and nan["dv"][20, 0].all()
    elif where == "v":
        assert nan["o"][20:90, :2, 7].all() and nan["dq"][20:90, :2].all() and nan["dk"][20, 0].all()
    else:
        assert nan["dq"][20, 0].all() and nan["dk"][:21, 0].all() and nan["dv"][:21, 0, 7].all()
    for n in nan:
        assert not nan[n][90:].any()
