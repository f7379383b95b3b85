"""The clipped policy loss and its gradient against the definition in 64 bits and against differences."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(tokens, seed=0, width=0.2, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    rand = lambda: torch.randn(tokens, generator=g, device=device)  # noqa: E731
    new = -rand().abs() * 2
    return dict(logprobs=new, old_logprobs=new + width * rand(), advantages=rand(), ref_logprobs=new + 2 * width * rand(),
                mask=torch.rand(tokens, generator=g, device=device) < 0.8)


def reference(x, starts=None, clip_low=0.2, clip_high=0.2, kl_weight=0.0):
    """(loss, grad, kl, clipped) in 64 bits, and how far fp32 terms may be off: a term by 2^-20 of the absolute values of its parts."""
    new, old, a = (x[n].double() for n in ("logprobs", "old_logprobs", "advantages"))
    mask = torch.ones_like(new, dtype=torch.bool) if x["mask"] is None else x["mask"].bool()
    w = torch.zeros_like(new)
    if starts is None:
        w[mask] = 1.0 / max(1, int(mask.sum()))
    else:
        spans = [(s, e) for s, e in zip(starts, starts[1:]) if int(mask[s:e].sum())]
        for s, e in spans:
            w[s:e][mask[s:e]] = 1.0 / (int(mask[s:e].sum()) * len(spans))
    d = new - old
    clipped = ((a > 0) & (d > math.log1p(clip_high))) | ((a < 0) & (d < math.log1p(-clip_low)))
    ratio = torch.where(clipped, torch.where(a > 0, 1.0 + clip_high, 1.0 - clip_low), torch.exp(d))
    loss, grad = -ratio * a, torch.where(clipped, 0.0, -ratio * a)
    off = (ratio * a).abs()
    kl = kl_off = None
    if x["ref_logprobs"] is not None:
        t = x["ref_logprobs"].double() - new
        k3 = torch.expm1(t) - t
        # the parts are exp(t) - 1 and t, each rounded for itself: |exp(t) - 1| + |t|, which does not cancel for t < 0
        loss, grad, off = loss + kl_weight * k3, grad - kl_weight * torch.expm1(t), off + abs(kl_weight) * (torch.expm1(t).abs() + t.abs())
        kl, kl_off = torch.where(w > 0, w * k3, 0.0).sum(), 2.0 ** -20 * torch.where(w > 0, w * torch.expm1(t).abs(), 0.0).sum()
    pick = lambda v: torch.where(w > 0, w * v, 0.0)  # noqa: E731
    return (pick(loss).sum(), pick(grad), kl, pick(clipped.double()).sum()), (2.0 ** -20 * pick(off).sum(), 2.0 ** -20 * pick(off), kl_off, 2.0 ** -23)


def run(x, starts=None, **kw):
    from metalhlo_b200 import cuda

    s = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    r = cuda.policy_loss(x["logprobs"], x["old_logprobs"], x["advantages"], mask=x["mask"], ref_logprobs=x["ref_logprobs"], starts=s, **kw)
    return r.loss, r.grad, r.kl, r.clip_fraction


def compare(x, starts=None, **kw):
    from metalhlo_b200 import cuda

    got = run(x, starts, **kw)
    assert cuda.device_error() == 0
    want, off = reference(x, starts, **kw)
    for g, w, o, name in zip(got, want, off, ("loss", "grad", "kl", "clip_fraction")):
        if w is None:
            assert g is None
            continue
        bad = ~((g.double() - w).abs() <= o + 1e-30)
        assert not bad.any(), (name, int(bad.sum()), float((g.double() - w).abs().max()))


def cut(tokens, seqs, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [0] + sorted(torch.randint(0, tokens + 1, (seqs - 1,), generator=g).tolist()) + [tokens]


@pytest.mark.parametrize("tokens", [1, 3, 4, 127, 128, 129, 4096, 4097, 16384, 16385, 100003])
@pytest.mark.parametrize("mask,ref", [(True, True), (False, False)])
def test_one_mean(tokens, mask, ref):
    x = inputs(tokens)
    if not mask:
        x["mask"] = None
    if not ref:
        x["ref_logprobs"] = None
    compare(x, kl_weight=0.05 if ref else 0.0, clip_high=0.28)


@pytest.mark.parametrize("tokens,seqs", [(1, 1), (5, 3), (130, 40), (4000, 7), (16384, 2048), (16384, 2049), (9000, 3000), (200000, 1), (200000, 300), (50000, 20000)])
def test_means_of_sequences(tokens, seqs):
    compare(inputs(tokens), cut(tokens, seqs), kl_weight=0.1)


@pytest.mark.parametrize("tokens", [300, 30000])
def test_tokens_of_no_sequence(tokens):
    """Rows in front of the first sequence and behind the last one count for nothing."""
    from metalhlo_b200 import cuda

    x = inputs(tokens)
    starts = [10, 90, 90, tokens - 50]
    compare(x, starts, kl_weight=0.1)
    grad = run(x, starts)[1]
    assert not grad[:10].any() and not grad[tokens - 50:].any()
    r = cuda.policy_loss(x["logprobs"], x["old_logprobs"], x["advantages"], starts=torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert not r.grad.any() and float(r.loss) == 0


@pytest.mark.parametrize("tokens", [400, 40000])
@pytest.mark.parametrize("starts", [None, True])
def test_what_is_masked_does_not_matter(tokens, starts):
    """NaN and infinities where the mask is 0, and a sequence of which nothing counts."""
    starts = starts and [0, 100, 150, tokens]
    x = inputs(tokens)
    x["mask"][100:150] = False
    y = {n: t.clone() for n, t in x.items()}
    for n, bad in (("logprobs", -math.inf), ("old_logprobs", math.nan), ("advantages", math.inf), ("ref_logprobs", math.nan)):
        y[n][~x["mask"]] = bad
    compare(x, starts, kl_weight=0.3)
    for a, b in zip(run(x, starts, kl_weight=0.3), run(y, starts, kl_weight=0.3)):
        assert torch.equal(a, b)
    assert not run(y, starts)[1][~x["mask"]].any()
    x["mask"][:] = False
    for t in run(x, starts, kl_weight=0.3):
        assert not t.any()


@pytest.mark.parametrize("low,high", [(0.2, 0.2), (0.0, 0.0), (0.5, 3.0), (0.999, 1e30)])
def test_borders(low, high):
    """Ratios on both sides of a border, as near as fp32 comes, and far beyond it."""
    n = 4000
    x = inputs(n)
    f32 = torch.float32
    border = torch.where(torch.arange(n, device="cuda") % 2 == 0, math.log1p(high), math.log1p(-low))
    x["old_logprobs"] = torch.full((n,), -3.0, device="cuda")
    x["logprobs"] = ((border - 3.0).to(f32).view(torch.int32) + torch.arange(n, device="cuda", dtype=torch.int32) // 2 % 9 - 4).view(f32)
    compare(x, clip_low=low, clip_high=high, kl_weight=0.01)
    x["logprobs"] = x["old_logprobs"] + torch.linspace(-60, 60, n, device="cuda")
    x["ref_logprobs"] = x["logprobs"] + torch.linspace(30, -30, n, device="cuda")
    compare(x, clip_low=low, clip_high=high, kl_weight=0.01)


def test_kl_of_nearly_equal_policies():
    """exp(x) - x - 1 of x next to 0, where its terms cancel: the bound is that of x^2 / 2."""
    x = inputs(2000)
    x["ref_logprobs"] = x["logprobs"] + torch.logspace(-7, 0.3, 2000, device="cuda") * torch.tensor([1.0, -1.0], device="cuda").repeat(1000)
    x["mask"] = None
    kl = run(x)[2].double()
    t = x["ref_logprobs"].double() - x["logprobs"].double()
    for part in (slice(0, 500), slice(500, 1500), slice(1500, 2000)):
        y = {n: (v[part].contiguous() if v is not None else None) for n, v in x.items()}
        want = (torch.expm1(t[part]) - t[part])
        series = torch.where(t[part].abs() < 1e-3, t[part] ** 2 / 2 + t[part] ** 3 / 6 + t[part] ** 4 / 24, want).mean()
        assert abs(float(run(y)[2].double() / series) - 1) <= 2.0 ** -19
    assert torch.isfinite(kl)


def test_differences():
    x = inputs(500)
    starts = cut(500, 6)
    kw = dict(kl_weight=0.2, clip_low=0.2, clip_high=0.3)
    grad = run(x, starts, **kw)[1]
    g = torch.Generator(device="cuda").manual_seed(2)
    way = torch.randn(500, generator=g, device="cuda", dtype=torch.float64)
    d = (x["logprobs"] - x["old_logprobs"]).double()
    h = 1e-6
    far = torch.minimum((d - math.log1p(0.3)).abs(), (d - math.log1p(-0.2)).abs()) > 1e-4  # steps that pass no border
    way = torch.where(far, way, 0.0)
    up, down = (reference(dict(x, logprobs=x["logprobs"].double() + s * h * way), starts, **kw)[0][0] for s in (1, -1))
    slope = float((up - down) / (2 * h))
    assert abs(float((grad.double() * way).sum()) - slope) <= 2.0 ** -20 * float((grad.double().abs() * way.abs()).sum()) + 1e-7


@pytest.mark.parametrize("tokens", [1000, 50000])
def test_in_place_and_unaligned(tokens):
    from metalhlo_b200 import cuda

    x = inputs(tokens)
    want = run(x, kl_weight=0.1)
    for n in ("logprobs", "old_logprobs", "advantages", "ref_logprobs"):
        y = {k: v.clone() for k, v in x.items()}
        r = cuda.policy_loss(y["logprobs"], y["old_logprobs"], y["advantages"], mask=y["mask"], ref_logprobs=y["ref_logprobs"], kl_weight=0.1, grad=y[n])
        assert r.grad is y[n] and torch.equal(r.grad, want[1]) and torch.equal(r.loss, want[0])
    odd = {n: torch.cat([v[:1], v])[1:] for n, v in x.items()}
    odd["mask"] = odd["mask"].view(torch.uint8)
    for a, b in zip(run(odd, kl_weight=0.1), want):
        assert torch.equal(a, b)
    shaped = cuda.policy_loss(*(x[n].view(10, -1) for n in ("logprobs", "old_logprobs", "advantages")), mask=x["mask"].view(10, -1), ref_logprobs=x["ref_logprobs"].view(10, -1), kl_weight=0.1)
    assert shaped.grad.shape == (10, tokens // 10) and torch.equal(shaped.grad.flatten(), want[1])


@pytest.mark.parametrize("tokens", [900, 30000])
def test_starts_out_of_order_are_reported(tokens):
    from metalhlo_b200 import cuda

    x = inputs(tokens)
    for starts in ([0, 500, 100, tokens], [0, tokens + 5], [-3, tokens]):
        run(x, starts)
        assert cuda.device_error() == 203
    assert cuda.device_error() == 0


def test_nothing():
    x = inputs(0)
    for starts in (None, [0, 0, 0]):
        loss, grad, kl, clipped = run(x, starts, kl_weight=0.1)
        assert grad.shape == (0,) and float(loss) == float(kl) == float(clipped) == 0
