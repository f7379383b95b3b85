"""Attention over packed sequences against 64 bits: lengths around the tiles' sizes, groups that do and do not divide them, head dimensions, layouts."""
import math

import pytest
import torch

from tests.packed_reference import check, inputs, reference

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def run(x, scale, causal, poison=7.0):
    from metalhlo_b200 import cuda

    plan = cuda.packed_plan(x["starts_dev"], x["rows"], x["q"].shape[1], x["k"].shape[1], causal)
    o = torch.full(x["q"].shape, poison, dtype=x["q"].dtype, device="cuda")
    lse = torch.full(x["q"].shape[:2], poison, device="cuda")
    cuda.packed_attention(x["q"], x["k"], x["v"], plan, scale, out=o, lse=lse)
    assert cuda.device_error() == 0
    return plan, o, lse


def compare(x, scale, causal):
    _, o, lse = run(x, scale, causal)
    end = x["starts"][-1]
    assert (o[end:] == 7.0).all() and (lse[end:] == 7.0).all()  # rows of no sequence are left alone
    y = dict(x, **{n: x[n][:end] for n in ("q", "k", "v", "grad")})
    want, off = reference(y, scale, causal)
    check(dict(o=o[:end], lse=lse[:end]), want, off, ("o", "lse"))


LENGTHS = [[1], [2, 0, 3], [127, 1, 128], [129, 255], [256, 257, 1, 0], [513, 40], [1025, 300, 31]]


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 64)])
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
    """More items than CTAs, of every length."""
    compare(inputs([37 * i % 700 for i in range(40)], 6, 3, 64, dtype), 0.125, True)


@pytest.mark.parametrize("dim", [64, 128])
def test_a_long_sequence(dim):
    compare(inputs([4500], 2, 1, dim, BF16), dim ** -0.5, True)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (BF16, 64), (F16, 128), (F16, 64), (F32, 64)])
def test_scores_that_grow(dtype, dim):
    """Later keys outweigh all earlier ones by far, again and again: the maximum in the exponent has to move."""
    x = inputs([700, 300], 2, 2, dim, dtype)
    for a, b in zip(x["starts"], x["starts"][1:]):
        x["q"][a:b] = x["q"][a:b].abs()
        x["k"][a:b] = (x["k"][a:b].abs().float() * torch.linspace(0.1, 6, b - a, device="cuda")[:, None, None]).to(dtype)
    compare(x, 0.25, False)
    compare(x, 0.25, True)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 64)])
def test_other_sequences_infinities(dtype, dim):
    """Infinities and NaN of one sequence do not reach the others."""
    x = inputs([100, 30, 129, 5], 4, 2, dim, dtype, spare=3)
    y = {n: t.clone() if torch.is_tensor(t) else t for n, t in x.items()}
    for n in ("q", "k", "v"):
        y[n][100:130] = math.inf if n == "v" else math.nan
    _, o, lse = run(x, 0.1, True)
    _, o2, lse2 = run(y, 0.1, True)
    for rows in (slice(0, 100), slice(130, 264)):
        assert torch.equal(o[rows], o2[rows]) and torch.equal(lse[rows], lse2[rows])
    assert torch.isnan(o2[100:130]).all() and torch.isnan(lse2[100:130]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts(dtype):
    """Heads outside, odd pitches, rows off the 16-byte grid, one head for all by a stride of zero, results into slices."""
    from metalhlo_b200 import cuda

    x = inputs([150, 60], 4, 2, 64, dtype)
    tokens = x["rows"]
    plan, want, want_lse = run(x, 0.125, True)

    def laid(t, how):
        if how == "heads first":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        if how == "wide":
            wide = torch.full((tokens, t.shape[1], 72), math.nan, dtype=dtype, device="cuda")
            wide[..., :64] = t
            return wide[..., :64]
        odd = torch.full((tokens * t.shape[1] * 65 + 1,), math.nan, dtype=dtype, device="cuda")[1:].view(tokens, t.shape[1], 65)[..., :64]
        odd.copy_(t)
        return odd

    for how in ("heads first", "wide", "odd"):
        q, k, v = (laid(x[n], how) for n in "qkv")
        out = laid(torch.zeros_like(x["q"]), how)
        lse = torch.empty_like(want_lse)
        assert cuda.packed_attention(q, k, v, plan, 0.125, out=out, lse=lse) is out
        if how == "odd" and dtype != F32:  # the FMA units' kernel: weights in fp32
            ref, off = reference(x, 0.125, True)
            check(dict(o=out, lse=lse), ref, off, ("o", "lse"))
        else:
            assert torch.equal(out, want) and torch.equal(lse, want_lse)
    one = x["k"][:, :1].expand(-1, 2, -1), x["v"][:, :1].expand(-1, 2, -1)
    y = dict(x, k=one[0], v=one[1])
    compare(y, 0.125, True)
    q = x["q"].clone()
    assert cuda.packed_attention(q, x["k"], x["v"], plan, 0.125, out=q) is q and torch.equal(q, want)  # in place


def test_nothing_to_do():
    from metalhlo_b200 import cuda

    for lengths in ([], [0, 0]):
        x = inputs(lengths, 2, 2, 64, BF16, spare=4)
        _, o, lse = run(x, 0.1, True)
        assert (o == 7.0).all() and (lse == 7.0).all()
    x = inputs([], 2, 2, 64, BF16)
    plan = cuda.packed_plan(x["starts_dev"], 0, 2, 2)
    assert cuda.packed_attention(x["q"], x["k"], x["v"], plan, 0.1).shape == (0, 2, 64)


def test_starts_and_plans_that_are_wrong():
    """Sequences out of order are passed over, plans of another batch are not followed; both are reported."""
    from metalhlo_b200 import cuda

    x = inputs([64, 64, 64], 2, 2, 64, BF16)
    good, want, _ = run(x, 0.1, True)
    starts = torch.tensor([0, 64, 500, 192], dtype=torch.int32, device="cuda")
    plan = cuda.packed_plan(starts, 192, 2, 2)
    assert cuda.device_error() == 203
    o = torch.full_like(want, 7.0)
    cuda.packed_attention(x["q"], x["k"], x["v"], plan, 0.1, out=o)
    assert torch.equal(o[:64], want[:64]) and (o[64:] == 7.0).all()
    assert cuda.device_error() == 0
    for other in (cuda.packed_plan(x["starts_dev"], 192, 2, 2, causal=False), cuda.packed_plan(x["starts_dev"], 192, 2, 1)):
        mixed = cuda.packed_plan(x["starts_dev"], 192, 2, 2)
        mixed._args.plan = other.tiles.data_ptr()
        o.fill_(7.0)
        cuda.packed_attention(x["q"], x["k"], x["v"], mixed, 0.1, out=o)
        assert cuda.device_error() == 205 and (o == 7.0).all()
    zero = cuda.packed_plan(x["starts_dev"], 192, 2, 2)
    zero.tiles.zero_()
    cuda.packed_attention(x["q"].float(), x["k"].float(), x["v"].float(), zero, 0.1, out=o.float())
    assert cuda.device_error() == 205

