"""Gradients of layer norm and RMS norm against the formula in 64 bits and against differences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(rows, hidden, dtype, seed=0, mean=0.5, grad=1.0, shift=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def make(shape, size, add=0.0):
        n = math.prod(shape)
        flat = torch.empty(n + shift, dtype=dtype, device="cuda")[shift:]  # off the 16-byte grid with a shift
        return flat.copy_(torch.randn(n, generator=g, device="cuda") * size + add).view(shape)

    return dict(x=make((rows, hidden), 1.5, mean), gamma=make((hidden,), 0.3, 1.0), dy=make((rows, hidden), grad), residual=make((rows, hidden), grad))


def reference(x, gamma, dy, residual, rms, eps):
    """((dx, dgamma, dbeta), bounds). Beside the rounding of dx (half a step, eps / 2 of it), of fp32 arithmetic: an element's deviation from the mean is
    off by 2^-21 of the row's largest |x|, products and sums by 2^-20 of their terms' absolute values."""
    half = torch.finfo(x.dtype).eps / 2
    x, dy = x.double(), dy.double()
    dev = x if rms else x - x.mean(1, keepdim=True)
    r = (dev.square().mean(1, keepdim=True) + eps).rsqrt()
    y, t = dev * r, dy if gamma is None else dy * gamma.double()
    dx = t - y * (t * y).mean(1, keepdim=True)
    if not rms:
        dx = dx - t.mean(1, keepdim=True)
    dx = dx * r
    y_off = 2.0 ** -21 * (r * x.abs().amax(1, keepdim=True) + y.abs())
    ty = (t * y).abs().mean(1, keepdim=True)
    off = r * (2.0 ** -20 * (t.abs() + t.abs().mean(1, keepdim=True) + y.abs() * ty) + y_off * ty + y.abs() * (t.abs() * y_off).mean(1, keepdim=True))
    if residual is not None:
        dx = dx + residual.double()
        off = off + 2.0 ** -24 * residual.double().abs()
    off = off + half * dx.abs() + (2.0 ** -25 if half == 2.0 ** -11 else 1e-30)
    sums = (dy * y).sum(0), dy.sum(0)
    return (dx, *sums), (off, (dy.abs() * y_off + 2.0 ** -20 * (dy * y).abs()).sum(0) + 1e-30, 2.0 ** -20 * dy.abs().sum(0) + 1e-30)


def compare(got, want, off):
    for g, w, o, name in zip(got, want, off, ("dx", "dgamma", "dbeta")):
        bad = ~((g.double() - w).abs() <= o)
        assert not bad.any(), (name, int(bad.sum()), float(((g.double() - w).abs() / o).nan_to_num(1e9).max()), bad.nonzero()[:3].tolist())


def run(x, rms, eps=1e-5, residual=True, gamma=True, **kw):
    from metalhlo_b200 import cuda

    f = cuda.rms_norm_grad if rms else cuda.layer_norm_grad
    return f(x["x"], x["gamma"] if gamma else None, x["dy"], eps, residual_grad=x["residual"] if residual else None, **kw)


HIDDEN = [1, 7, 8, 64, 100, 255, 256, 257, 264, 512, 513, 520, 769, 1000, 1024, 2056, 4096, 4097, 8192, 8200, 8201, 12288, 12289, 14088, 16384, 16385, 20000]


@pytest.mark.parametrize("hidden", HIDDEN)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("rows,residual", [(1, False), (5, True), (700, True)])
def test_sizes(hidden, dtype, rms, rows, residual):
    x = inputs(rows, hidden, dtype)
    compare(run(x, rms, residual=residual), *reference(x["x"], x["gamma"], x["dy"], x["residual"] if residual else None, rms, 1e-5))


@pytest.mark.parametrize("hidden", [96, 768, 1001])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_rows(hidden, rms, dtype):
    x = inputs(20011, hidden, dtype)
    compare(run(x, rms), *reference(x["x"], x["gamma"], x["dy"], x["residual"], rms, 1e-5))


@pytest.mark.parametrize("shift", [1, 3, 4])
@pytest.mark.parametrize("hidden", [64, 200, 1024, 1003, 16400])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_off_the_grid(shift, hidden, dtype):
    x = inputs(9, hidden, dtype, shift=shift)
    compare(run(x, False), *reference(x["x"], x["gamma"], x["dy"], x["residual"], False, 1e-5))


@pytest.mark.parametrize("mean", [0.0, 300.0])
@pytest.mark.parametrize("hidden", [320, 1600, 17000])
def test_means_far_from_zero(mean, hidden):
    x = inputs(33, hidden, F32, mean=mean)
    compare(run(x, False), *reference(x["x"], x["gamma"], x["dy"], x["residual"], False, 1e-5))


@pytest.mark.parametrize("hidden", [64, 1024, 1025, 17000])
@pytest.mark.parametrize("rms", [False, True])
def test_rows_that_do_not_vary(hidden, rms):
    """A variance of zero: r is 1 / sqrt(eps)."""
    x = inputs(4, hidden, F32)
    x["x"].fill_(0.0 if rms else 2.0)
    compare(run(x, rms), *reference(x["x"], x["gamma"], x["dy"], x["residual"], rms, 1e-5))


@pytest.mark.parametrize("hidden", [128, 1024, 1001, 17000])
@pytest.mark.parametrize("which", ["x", "dy", "residual"])
def test_in_place(hidden, which):
    x = inputs(300, hidden, BF16)
    want = run(x, False)
    y = {n: t.clone() for n, t in x.items()}
    got = run(y, False, out=y[which])
    assert got[0] is y[which] and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("hidden", [128, 1024, 1001, 17000])
def test_without_gamma_and_without_sums(hidden):
    import ctypes as C

    from metalhlo_b200 import cuda

    x = inputs(50, hidden, BF16)
    got = run(x, False, gamma=False)
    compare(got, *reference(x["x"], None, x["dy"], x["residual"], False, 1e-5))
    need = cuda.lib.mhlo_cuda_norm_grad_scratch_bytes(50, hidden)
    scratch, dx, dbeta = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.empty_like(x["x"]), torch.full((hidden,), 7.0, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    P = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    for sums in ((None, None), (None, dbeta)):
        cuda.check(cuda.lib.mhlo_cuda_layer_norm_grad(cuda.BF16, P(x["x"]), None, P(x["dy"]), P(x["residual"]), P(dx), P(sums[0]), P(sums[1]), 50, hidden, 1e-5, P(scratch), need, s))
        assert torch.equal(dx, got[0])
    assert torch.equal(dbeta, got[2])
    assert C.sizeof(C.c_void_p) == 8


def test_no_rows():
    x = inputs(0, 64, BF16)
    dx, dgamma, dbeta = run(x, False)
    assert dx.shape == (0, 64) and not dgamma.any() and not dbeta.any()


def test_rows_with_infinities_stay_alone():
    x = inputs(40, 1024, BF16)
    want = run(x, False)
    x["x"][7] = math.inf
    got = run(x, False)
    rows = torch.arange(40, device="cuda") != 7
    assert torch.equal(got[0][rows], want[0][rows]) and torch.isnan(got[0][7]).all() and torch.isnan(got[1]).all() and torch.equal(got[2], want[2])


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("hidden", [48, 600])
def test_differences(rms, hidden):
    x = inputs(3, hidden, F32)
    got = run(x, rms, residual=False)

    def value(at, gamma):
        dev = at if rms else at - at.mean(1, keepdim=True)
        return float((dev * (dev.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gamma * x["dy"].double()).sum())

    g = torch.Generator(device="cuda").manual_seed(3)
    a, gamma, h = x["x"].double(), x["gamma"].double(), 1e-5
    way = torch.randn(a.shape, generator=g, device="cuda", dtype=torch.float64)
    slope = (value(a + h * way, gamma) - value(a - h * way, gamma)) / (2 * h)
    assert abs(float((got[0].double() * way).sum()) - slope) <= 2.0 ** -20 * float((got[0].double().abs() * way.abs()).sum()) + 1e-6 * max(1.0, abs(slope))
    way = torch.randn(hidden, generator=g, device="cuda", dtype=torch.float64)
    slope = (value(a, gamma + h * way) - value(a, gamma - h * way)) / (2 * h)
    assert abs(float((got[1].double() * way).sum()) - slope) <= 2.0 ** -19 * float((got[1].double().abs() * way.abs()).sum()) + 1e-6 * max(1.0, abs(slope))


def test_the_same_bits_every_time():
    x = inputs(5000, 2048, BF16)
    want = run(x, False)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(x, False), want))
