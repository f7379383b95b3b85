"""Log probabilities of tokens, entropies, alternatives and their gradient against fp64.

Bounds, with u = 2^-24: a logit times the scale is off by u |z|, an exponential by 2^-22 + 2 u |d| of itself (d = z - max), a sum of n
terms in 128 strands by (n / 128 + 32) u of the sum of magnitudes; a log probability also by u of itself and of the lse.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
U = 2.0 ** -24


def cuda_mod():
    from metalhlo_b200 import cuda

    return cuda


def draw(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * spread).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g)
    return x, t


def definition(x, scale):
    """fp64: z, lse, p, entropy, and the bound on the error of a sum relative to its magnitudes."""
    z = x.double() * scale
    m = z.amax(-1, keepdim=True)
    d = z - m
    lse = (m + torch.exp(d).sum(-1, keepdim=True).log())[..., 0]
    p = torch.exp(z - lse[..., None])
    pd = torch.where(p > 0, p * d, torch.zeros_like(p))
    entropy = (lse - m[..., 0]) - pd.sum(-1)
    n = x.shape[-1]
    order = (n / 128 + 32) * U
    clean = torch.where(p > 0, d, torch.zeros_like(d)).abs()
    own = (p * (2.0 ** -22 + 4 * U * clean + 2 * U * m.abs())).sum(-1)  # of the exponentials, relative to their sum
    lse_bound = order + own + 2 * U * lse.abs() + 2 * U * m[..., 0].abs()
    size = (p * clean).sum(-1)
    ent_bound = lse_bound + size * (order + own) + (p * clean * (2.0 ** -22 + 4 * U * clean)).sum(-1) + 4 * U * m[..., 0].abs()
    return z, lse, p, entropy, lse_bound, ent_bound


def top_of(x, k):
    """Ids in descending order: NaN first, the lowest id among equals."""
    return torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[..., :k]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,top,scale", [(3, 1, 1, 1.0), (5, 7, 7, 0.5), (4, 33, 20, 1.0), (2, 1000, 32, 1.7), (7, 4097, 5, 1.0), (3, 50257, 32, 1.0),
                                                  (1, 50257, 1, 2.0), (300, 513, 0, 1.0), (2, 128256, 20, 0.8), (1, 262144, 32, 1.0), (150, 8191, 20, 1.0)])
def test_forward(dtype, rows, vocab, top, scale):
    cuda = cuda_mod()
    x, t = draw(rows, vocab, dtype, rows + vocab)
    for targets in (t, t.int()):
        r = cuda.token_logprobs(x.cuda(), targets.cuda(), top_k=top, scale=scale)
        z, lse, p, entropy, lse_bound, ent_bound = definition(x, scale)
        zt = z.gather(1, t[:, None])[:, 0]
        assert bool(((r.lse.cpu() - lse).abs() <= lse_bound).all())
        assert bool(((r.logprobs.cpu() - (zt - lse)).abs() <= lse_bound + 2 * U * zt.abs() + U * (zt - lse).abs()).all())
        assert bool(((r.entropy.cpu() - entropy).abs() <= ent_bound).all())
        if top:
            ids = top_of(x, top)
            assert torch.equal(r.top_ids.cpu().long(), ids)
            zk = z.gather(1, ids)
            assert bool(((r.top_logprobs.cpu() - (zk - lse[:, None])).abs() <= lse_bound[:, None] + 2 * U * zk.abs() + U * (zk - lse[:, None]).abs()).all())
        else:
            assert r.top_ids is None


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few_values", "zeros_of_both_signs", "tail"])
@pytest.mark.parametrize("vocab", [40, 5000, 50257])
def test_alternatives_among_many_equals(dtype, kind, vocab):
    """Orders that are hard on a selection: ties resolved by the lowest id, and rows whose largest entries come last."""
    cuda = cuda_mod()
    i = torch.arange(vocab)
    x = {"equal": torch.full((vocab,), 1.5), "rising": i / 100.0, "falling": -i / 100.0, "few_values": (i * 7919 % 13).float(),
         "zeros_of_both_signs": torch.where(i % 3 == 0, -0.0, 0.0), "tail": torch.where(i >= vocab - 33, 3.0, -1.0)}[kind].to(dtype)
    x = torch.stack([x, x.roll(1), x.flip(0)])
    for top in (1, 5, 32):
        r = cuda.token_logprobs(x.cuda(), top_k=top)
        assert torch.equal(r.top_ids.cpu().long(), top_of(x, top))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [2049, 20011])
def test_alternatives_of_many_rows_of_every_order(dtype, vocab):
    """Rows in numbers that fill the machine, hard orders beside ordinary ones, most of them off the 16-byte grid; masks that leave fewer
    numbers than there are alternatives; more NaN than alternatives."""
    cuda = cuda_mod()
    i = torch.arange(vocab)
    hard = [torch.full((vocab,), 1.5), i / 50.0, -i / 50.0, (i * 7919 % 13).float(), torch.where(i >= vocab - 33, 3.0, -1.0), torch.where(i % 700 == 3, i / 50.0, -float("inf")),
            torch.full((vocab,), -float("inf")), torch.where(i % 40 == 1, float("nan"), i / 50.0), torch.where(i % 2 == 0, i / 50.0, -i / 50.0)]
    x, _ = draw(310, vocab, dtype, 41)
    for r, h in enumerate(hard * 3):
        x[11 * r] = h.roll(r).to(dtype)
    for top in (1, 20, 32):
        assert torch.equal(cuda.token_logprobs(x.cuda(), top_k=top).top_ids.cpu().long(), top_of(x, top))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [100, 50257])
def test_masked_and_broken_rows(dtype, vocab):
    """-infinity is probability 0 (log probability -infinity, no part in the entropy); a row with nothing else, an infinity or a NaN
    is NaN; the alternatives keep their order. Other rows do not notice."""
    cuda = cuda_mod()
    x, t = draw(6, vocab, dtype, 3)
    inf = float("inf")
    x[0, ::2], x[1], x[2, 7], x[3, 50], x[4, :] = -inf, -inf, inf, float("nan"), -inf
    x[4, vocab - 1] = torch.finfo(dtype).min
    t[0], t[4] = 2, vocab - 1
    r = cuda.token_logprobs(x.cuda(), t.cuda(), top_k=20)
    z, lse, p, entropy, lse_bound, ent_bound = definition(x, 1.0)
    for row in (0, 5):
        assert abs(r.lse[row].cpu() - lse[row]) <= lse_bound[row] and abs(r.entropy[row].cpu() - entropy[row]) <= ent_bound[row]
    assert r.logprobs[0] == -inf and r.logprobs[4] == 0 and r.entropy[4] == 0
    for row in (1, 2, 3):
        assert all(bool(v[row].isnan()) for v in (r.logprobs, r.entropy, r.lse)) and bool(r.top_logprobs[row].isnan().all())
    assert torch.equal(r.top_ids.cpu().long(), top_of(x, 20))
    assert bool((r.top_logprobs[4, 1:] == -inf).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("vocab", [100, 20001])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -12, 3.0])
def test_rows_far_from_zero(dtype, vocab, scale):
    """Maxima whose type has steps wider than any exponent that counts, next to the lowest number, and all equal there; every other
    entry is a step or much more below the maximum, or -infinity."""
    cuda = cuda_mod()
    big = {torch.float16: 60000.0, torch.bfloat16: 1e5, torch.float32: 1e12}[dtype]
    least = torch.finfo(dtype).min
    x = torch.full((8, vocab), -float("inf"), dtype=torch.float32)
    x[0], x[0, 3] = -big, big
    x[1], x[1, 3] = big * (1 - torch.finfo(dtype).eps), big  # next number but one below, or the one below
    x[2], x[2, 3], x[2, 4] = 0.0, -big, 1.0
    x[3] = least
    x[4, :50] = least
    x[5], x[5, 7] = least, least * (1 - torch.finfo(dtype).eps)
    x[6, 5], x[6, 9] = -big, -big
    x[7] = big
    x = x.to(dtype)
    t = torch.full((8,), 3)
    r = cuda.token_logprobs(x.cuda(), t.cuda(), scale=scale)
    z = x.double() * scale
    m = z.amax(1, keepdim=True)
    d = z - m
    log_s = torch.exp(d).sum(1).log()
    p = torch.exp(d - log_s[:, None])
    entropy = log_s - torch.where(p > 0, p * d, torch.zeros_like(p)).sum(1)
    # Relative to the maximum everything is as exact as anywhere: (x - max) scale is one rounding of the difference and one of the
    # product, and differences of equal or neighbouring numbers are exact.
    order = (vocab / 128 + 32) * U
    want = d.gather(1, t[:, None])[:, 0] - log_s
    got = r.logprobs.cpu().double()
    assert bool((torch.isinf(want) == torch.isinf(got)).all())
    off = torch.where(torch.isinf(want), torch.zeros_like(want), (got - want).abs())
    assert bool((off <= order + 2.0 ** -20 + 4 * U * torch.where(torch.isinf(want), torch.zeros_like(want), want.abs())).all())
    assert bool(((r.entropy.cpu() - entropy).abs() <= order * (1 + entropy.abs()) + 2.0 ** -18).all())


def test_targets_that_name_no_token():
    cuda = cuda_mod()
    x, t = draw(5, 77, torch.float32, 4)
    t[0], t[1], t[2] = -1, -100, 77
    for targets in (t, t.int()):
        r = cuda.token_logprobs(x.cuda(), targets.cuda())
        assert r.logprobs[0] == 0 and r.logprobs[1] == 0 and bool(r.logprobs[2].isnan()) and bool(r.logprobs[3:].isfinite().all())
        g = torch.ones(5, device="cuda")
        d = cuda.token_logprobs_grad(x.cuda(), targets.cuda(), r.lse, grad_logprobs=g)
        assert bool((d[:2] == 0).all()) and bool(d[2].isnan().all()) and bool(d[3:].isfinite().all())


def gradient(x, t, lse, entropy, g, e, ids, gt, scale):
    """fp64, and the bound on the error before the last rounding."""
    logp = x.double() * scale - lse.double()[:, None]
    p = torch.exp(logp)
    picked = torch.zeros_like(p)
    rows = torch.arange(x.shape[0])
    weight = torch.zeros(x.shape[0], dtype=torch.float64)
    if g is not None:
        ok = t >= 0
        picked[rows[ok], t[ok]] += g.double()[ok]
        weight += torch.where(ok, g.double(), torch.zeros_like(weight))
    size = weight.abs()
    if gt is not None:
        for k in range(gt.shape[1]):
            ok = ids[:, k] >= 0
            picked[rows[ok], ids[ok, k].long()] += gt[ok, k].double()
            weight += torch.where(ok, gt[:, k].double(), torch.zeros_like(weight))
            size += gt[:, k].abs()
    low = torch.where(p > 0, logp, torch.zeros_like(p))
    inner, inner_size = weight[:, None].expand_as(p), size[:, None].expand_as(p)
    if e is not None:
        inner = inner + e.double()[:, None] * (low + entropy.double()[:, None])
        inner_size = inner_size + e.double().abs()[:, None] * (low.abs() + entropy.double().abs()[:, None])
    z = torch.where(p > 0, x.double() * scale, torch.zeros_like(p)).abs()
    off = 2.0 ** -21 + 4 * U * (z + lse.double().abs()[:, None] + low.abs())  # of p, relative
    bound = p * inner_size * (off + 40 * U) + 40 * U * picked.abs()
    if e is not None:
        bound = bound + p * e.double().abs()[:, None] * 2 * U * (z + lse.double().abs()[:, None])
    return scale * (picked - p * inner), scale * bound


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,vocab,top,scale", [(3, 1, 1, 1.0), (5, 33, 20, 0.5), (4, 1000, 0, 1.0), (3, 50257, 32, 1.0), (200, 257, 5, 1.3), (2, 128256, 0, 1.0)])
@pytest.mark.parametrize("parts", ["all", "logprobs", "entropy", "top"])
def test_gradient(dtype, rows, vocab, top, scale, parts):
    cuda = cuda_mod()
    x, t = draw(rows, vocab, dtype, rows + vocab)
    t[0] = -1 if rows > 2 else t[0]
    gen = torch.Generator().manual_seed(7)
    r = cuda.token_logprobs(x.cuda(), t.cuda(), top_k=top, scale=scale)
    g = torch.randn(rows, generator=gen) if parts in ("all", "logprobs") else None
    e = torch.randn(rows, generator=gen) if parts in ("all", "entropy") else None
    gt = torch.randn(rows, top, generator=gen) if top and parts in ("all", "top") else None
    ids = r.top_ids.cpu() if top else None
    if gt is not None and top > 3:
        ids = ids.clone()
        ids[:, 2], ids[-1, 1] = ids[:, 0], -1  # an id twice, and none
    up = lambda v: None if v is None else v.cuda()
    args = (t.cuda(), r.lse)
    kw = dict(entropy=r.entropy, grad_logprobs=up(g), grad_entropy=up(e), top_ids=up(ids) if gt is not None else None, grad_top=up(gt), scale=scale)
    d = cuda.token_logprobs_grad(x.cuda(), *args, **kw)
    want, bound = gradient(x, t, r.lse.cpu(), r.entropy.cpu(), g, e, ids, gt, scale)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert bool(((d.cpu().double() - want).abs() <= HALF_STEP[dtype] * want.abs() + bound * (1 + 2.0 ** -7) + tiny).all())
    inplace = x.cuda()
    assert cuda.token_logprobs_grad(inplace, *args, out=inplace, **kw) is inplace and torch.equal(inplace, d)


def test_gradient_against_differences():
    """d / dx of a weighted sum of every result, by central differences of the fp64 definition: the step's own error is
    h^2 f''' / 6 < 1e-6 at h = 1e-3 and third derivatives below 6, the kernel's 2^-20 of values below 4."""
    cuda = cuda_mod()
    x, t = draw(2, 19, torch.float32, 8, spread=1.0)
    scale, k = 1.3, 4
    gen = torch.Generator().manual_seed(9)
    g, e, gt = torch.randn(2, generator=gen), torch.randn(2, generator=gen), torch.randn(2, k, generator=gen)
    r = cuda.token_logprobs(x.cuda(), t.cuda(), top_k=k, scale=scale)
    ids = r.top_ids.cpu().long()

    def f(y):
        logp = torch.log_softmax(y * scale, -1)
        h = -(logp.exp() * logp).sum(-1)
        return (g * logp.gather(1, t[:, None])[:, 0] + e * h + (gt * logp.gather(1, ids)).sum(1)).sum()

    d = cuda.token_logprobs_grad(x.cuda(), t.cuda(), r.lse, r.entropy, g.cuda(), e.cuda(), r.top_ids, gt.cuda(), scale=scale).cpu()
    y, h = x.double(), 1e-3
    for i in range(2):
        for j in range(19):
            up, down = y.clone(), y.clone()
            up[i, j] += h
            down[i, j] -= h
            assert abs((f(up) - f(down)) / (2 * h) - d[i, j]) <= 1e-6 + 2.0 ** -18


def test_gradient_of_masked_and_broken_rows():
    cuda = cuda_mod()
    x, t = draw(4, 300, torch.float32, 10)
    inf = float("inf")
    x[0, ::2], x[1], x[2, 9] = -inf, -inf, float("nan")
    t[0] = 1
    r = cuda.token_logprobs(x.cuda(), t.cuda())
    one = torch.ones(4, device="cuda")
    d = cuda.token_logprobs_grad(x.cuda(), t.cuda(), r.lse, r.entropy, one, one).cpu()
    assert bool((d[0, ::2] == 0).all()) and bool(d[0].isfinite().all()) and bool(d[1:3].isnan().all()) and bool(d[3].isfinite().all())
    assert abs(d[0].double().sum()) < 1e-5


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("offset,pitch", [(0, 1031), (1, 1031), (3, 1040), (0, 1030)])
def test_rows_of_any_pitch_and_alignment(dtype, offset, pitch):
    """Logits cut out of padded rows, and a gradient into such rows: the columns behind the vocabulary are left alone."""
    cuda = cuda_mod()
    rows, vocab = 9, 1029
    x, t = draw(rows, vocab, dtype, 11)
    store = torch.full((rows * pitch + 8,), float("nan"), dtype=dtype, device="cuda")
    view = store[offset:offset + rows * pitch].view(rows, pitch)[:, :vocab]
    view.copy_(x)
    a, b = cuda.token_logprobs(x.cuda(), t.cuda(), top_k=7), cuda.token_logprobs(view, t.cuda(), top_k=7)
    z, lse, p, entropy, lse_bound, ent_bound = definition(x, 1.0)
    assert torch.equal(a.top_ids, b.top_ids) and bool(((b.lse.cpu() - lse).abs() <= lse_bound).all())
    g = torch.randn(rows, generator=torch.Generator().manual_seed(12)).cuda()
    before = store.clone()
    d = cuda.token_logprobs_grad(view, t.cuda(), a.lse, a.entropy, g, g)
    cuda.token_logprobs_grad(view, t.cuda(), a.lse, a.entropy, g, g, out=view)
    assert torch.equal(view, d)
    view.copy_(x)
    assert torch.equal(store.isnan(), before.isnan())
    want, bound = gradient(x, t, a.lse.cpu(), a.entropy.cpu(), g.cpu(), g.cpu(), None, None, 1.0)
    assert bool(((d.cpu().double() - want).abs() <= HALF_STEP[dtype] * want.abs() + bound * (1 + 2.0 ** -7) + torch.finfo(dtype).smallest_normal).all())


def test_leading_dimensions_streams_graphs_and_empty_calls():
    cuda = cuda_mod()
    x, t = draw(12, 2000, torch.bfloat16, 13)
    x, t = x.cuda().view(3, 4, 2000), t.cuda().view(3, 4)
    a = cuda.token_logprobs(x, t, top_k=5)
    assert a.logprobs.shape == (3, 4) and a.top_ids.shape == (3, 4, 5)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    b = cuda.token_logprobs(x, t, top_k=5, stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros_like(x)
    with torch.cuda.graph(graph):
        c = cuda.token_logprobs(y, t, top_k=5)
        d = cuda.token_logprobs_grad(y, t, c.lse, c.entropy, c.logprobs, c.entropy)
    for scale in (1.0, 0.5):
        y.copy_(x * scale)
        graph.replay()
        e = cuda.token_logprobs(y, t, top_k=5)
        assert all(torch.equal(u, v) for u, v in zip(c, e))
        assert torch.equal(d, cuda.token_logprobs_grad(y, t, e.lse, e.entropy, e.logprobs, e.entropy))
    none = cuda.token_logprobs(torch.zeros(0, 5, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top_k=2)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 2)
    only = cuda.token_logprobs(x[0, 0], top_k=1, entropy=False)
    assert only.logprobs is None and only.entropy is None and int(only.top_ids[0]) == int(a.top_ids[0, 0, 0])
