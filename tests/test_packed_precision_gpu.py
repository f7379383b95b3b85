"""Attention over packed sequences where 16-bit weights have least to spare: against 64 bits, with bounds from the roundings that the header names."""
import math

import pytest
import torch

from tests.packed_reference import check, inputs, reference

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def attend(q, k, v, lengths, scale, causal):
    from metalhlo_b200 import cuda

    starts = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    plan = cuda.packed_plan(starts, q.shape[0], q.shape[1], k.shape[1], causal)
    lse = torch.empty(q.shape[:2], device="cuda")
    o = cuda.packed_attention(q, k, v, plan, scale, lse=lse)
    assert cuda.device_error() == 0
    return o, lse


def thirds(z, dtype, dim):
    """Rows of `dim` elements whose first three add up to z, as near as three numbers of the type come."""
    x = torch.zeros(*z.shape, dim, dtype=dtype, device="cuda")
    rest = z.double()
    for i in range(3):
        x[..., i] = rest.to(dtype)
        rest = rest - x[..., i].double()
    return x


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_jump_inside_a_block(dtype, dim):
    """Key 64 of a block outweighs the 64 before it by a little over 2^8, so weights that are rounded already have to follow the new largest score. Their values are 1, that
    key's is 0: whatever is lost of them together shows in the result. One rounding of each weight and one of the result are half a step each."""
    half = torch.finfo(dtype).eps / 2
    jumps, depths = torch.linspace(5.56, 7.0, 300, device="cuda"), torch.tensor([0.4983051, 0.6459321, 0.6572881, 0.68], device="cuda")
    z = torch.full((300, 4, 128), -50.0, device="cuda")
    z[..., 0] = 0.0
    z[..., 1:64] = -depths[None, :, None]
    z[..., 64] = jumps[:, None]
    n = 1200 * 128
    k = thirds(z.view(n, 1), dtype, dim)
    q = torch.zeros_like(k)
    q[..., :3] = 1.0
    v = torch.zeros_like(k)
    v.view(1200, 128, dim)[:, :64] = 1.0
    o, lse = attend(q, k, v, [128] * 1200, 1.0, False)
    z = k.double().sum(-1).view(1200, 128)
    want = torch.softmax(z, 1)[:, :64].sum(1)[:, None, None]
    bad = ~((o.view(1200, 128, dim).double() - want).abs() <= (2 * half + 2.0 ** -16) * want)
    assert not bad.any(), (int(bad.sum()), float(((o.view(1200, 128, dim).double() - want).abs() / want).max() / half))
    assert ((lse.view(1200, 128).double() - torch.logsumexp(z, 1)[:, None]).abs() <= 2.0 ** -17).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("ahead", [14.0, 15.0, 16.0])
@pytest.mark.parametrize("last", [False, True])
def test_many_small_weights_behind_a_large_one_in_fp16(dim, ahead, last):
    """One key without a value is 14 to 16 nats ahead of 16 383 equal ones: their weights, 2^-20 to 2^-23 of the largest, are all that the result has. Half a step of each weight
    and of the result, 2^-31 of the largest weight for each that is below 2^-20 of it, and 2^-16 for sums and exponentials."""
    n = 16384
    at = n - 1 if last else 0
    q, k, v = (torch.zeros(n, 1, dim, dtype=F16, device="cuda") for _ in range(3))
    q[..., 0] = 1.0
    k[at, 0, 0] = ahead
    v.fill_(1.0)
    v[at] = 0.0
    o, _ = attend(q, k, v, [n], 1.0, False)
    small = math.exp(-ahead)
    want = (n - 1) * small / (1 + (n - 1) * small)
    off = (2 * 2.0 ** -11 + 2.0 ** -16) * want + (n - 1) * 2.0 ** -31 / (1 + (n - 1) * small)
    assert float((o.double() - want).abs().max()) <= off, (float((o.double() / want - 1).abs().max()), off / want)


@pytest.mark.parametrize("dtype,size,scale", [(BF16, 2.0 ** 40, 2.0 ** 20), (BF16, 2.0 ** 16, 1.0), (F16, 64.0, 6e6), (F16, 64.0, 2e5), (F32, 2.0 ** 40, 2.0 ** 20)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_scores_far_from_zero(dtype, size, scale, dim, causal):
    """Scores of up to 2^23 and 2^67, far apart: a row is the value of its best key, however coarse an fp32 number of the score's size is. The one weight that is left need not be a
    power of two, so its rounding and that of the result count, half a step each; fp32 values go through the product in two parts, 2^-20 of them with the sum's roundings."""
    n = 255
    g = torch.Generator(device="cuda").manual_seed(0)
    rank = torch.randperm(n, generator=g, device="cuda") - 127
    q, k = (torch.zeros(n, 1, dim, dtype=dtype, device="cuda") for _ in range(2))
    q[..., 3] = 1.0
    k[:, 0, 3] = rank * size
    v = torch.randn(n, 1, dim, generator=g, device="cuda").to(dtype)
    o, lse = attend(q, k, v, [n], scale, causal)
    best = torch.cummax(rank, 0).indices if causal else torch.full((n,), int(rank.argmax()), device="cuda")
    off = 2.0 ** -20 if dtype == F32 else torch.finfo(dtype).eps + 2.0 ** -16
    assert ((o.double() - v[best].double()).abs() <= off * v[best].double().abs()).all()
    want = k[best, 0, 3].double() * scale
    assert ((lse[:, 0].double() - want).abs() <= 2.0 ** -21 * want.abs()).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_very_different_sizes_in_one_fp16_call(dim, causal):
    """Sequences whose gradients are 2^10 and 2^20 smaller than another's in the same call: each is as exact as it would be alone."""
    from metalhlo_b200 import cuda

    lengths, sizes = [500, 2000, 300], [2.0 ** 8, 2.0 ** -12, 2.0 ** -2]
    x = inputs(lengths, 4, 2, dim, F16)
    for size, a, b in zip(sizes, x["starts"], x["starts"][1:]):
        x["grad"][a:b] *= size
    plan = cuda.packed_plan(x["starts_dev"], x["rows"], 4, 2, causal)
    lse = torch.empty(x["rows"], 4, device="cuda")
    o = cuda.packed_attention(x["q"], x["k"], x["v"], plan, dim ** -0.5, lse=lse)
    grads = cuda.packed_attention_grad(x["q"], x["k"], x["v"], o, lse, x["grad"], plan, dim ** -0.5)
    assert cuda.device_error() == 0
    want, off = reference(x, dim ** -0.5, causal)
    check(dict(zip(("dq", "dk", "dv"), grads)), want, off, ("dq", "dk", "dv"))
