"""Cached attention where the scales of blocks lie far apart. A row's result is a matter of the keys that it sees, and its error one of
what they contribute: whatever blocks hold that a row does not see, or sees with a weight of nothing, is not noticed.

Bounds as in test_kv_cache_gpu.py, with what a row sees of each block's value scale vs by its weights p in place of the largest scale: a
weight times its value scale is lost below 2^-31 (fp32 inputs: 2^-39) of the largest, and a sum that carries 128 with every code is off by
2^-23 of 128 sum p vs at most in each step of 16 keys."""
import math

import pytest
import torch

from test_kv_cache_gpu import HALF_STEP, HALF_SUBNORMAL, TYPES, cuda_mod, make_cache, make_table, on_gpu, starts_of

pytestmark = pytest.mark.gpu

# new tokens, lengths, query heads of a cache head: rows of the kernel of few rows (drafts, chunks) and of the one of many
CALLS = {"drafts": ([20], [263], 1), "ragged": ([5, 1, 17], [66, 33, 387], 3), "chunks": ([40, 130], [500, 290], 2), "long": ([200], [1500], 4)}


def definition(cache, q, table, lengths, starts, scale):
    """fp64 on the GPU: (o, lse, bound without the result's own rounding, keys each row sees)."""
    o, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse, seen_of = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda"), []
    heads, page, dim = cache.k.shape[1:]
    single = q.dtype == torch.float32
    for b, length in enumerate(lengths):
        first, n = int(starts[b]), int(starts[b + 1] - starts[b])
        pages = torch.from_numpy(table[b, :-(-length // page)]).long().cuda()
        (k, ks), (v, vs) = ((c[pages].double(), s[pages].double()[:, :, None].expand(-1, -1, page)) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        k, v = ((c * s[..., None]).transpose(0, 1).flatten(1, 2)[:, :length] for c, s in ((k, ks), (v, vs)))  # [heads, keys, dim]
        ks, vs = (s.transpose(0, 1).flatten(1, 2)[:, None, None, :length] for s in (ks, vs))
        x = q[first:first + n].double().unflatten(1, (heads, -1)).permute(1, 2, 0, 3)  # [heads, group, new, dim]
        position = torch.arange(length - n, length, device="cuda")
        seen = torch.arange(length, device="cuda")[None] <= position[:, None]
        z = (x @ k[:, None].transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(z, -1)
        products = (x.abs() @ k.abs()[:, None].transpose(2, 3)) + (0 if single else 128) * ks * x.abs().sum(-1, keepdim=True)
        products = torch.where(p > 2.0 ** -60, products, 0).amax(-1, keepdim=True)
        weight = 2 * (dim / 16) * 2.0 ** -22 * scale * products + 2.0 ** -20 + (0 if single else 2.0 ** -11)
        v = torch.nan_to_num(v)[:, None]
        vs = torch.nan_to_num(vs)
        lost = (2.0 ** -39 if single else 2.0 ** -31) * 127 * (position + 1)[:, None] * (p * vs).amax(-1, keepdim=True)
        if not single:
            lost = lost + 2.0 ** -27 * 128 * (position + 1)[:, None] * (p * vs).sum(-1, keepdim=True)

        def rows(t):
            return t.permute(2, 0, 1, 3).flatten(1, 2)

        o[first:first + n], bound[first:first + n] = rows(p @ v), rows(weight * (p @ v.abs()) + lost)
        lse[first:first + n] = rows(z.logsumexp(-1, keepdim=True))[..., 0]
        seen_of += (position + 1).tolist()
    return o, lse, bound, seen_of


def run(cache, q, table, lengths, starts, scale):
    lse = torch.zeros(q.shape[:2], device="cuda")
    o = cuda_mod().cached_attention(q, cache, on_gpu(table), on_gpu(lengths), scale, token_starts=on_gpu(starts), lse=lse)
    assert cuda_mod().device_error() == 0
    return o, lse


def check(o, want, bound, rows):
    """The rows ``rows``; elements beyond their type may be anything."""
    error = torch.nan_to_num((o.double() - want).abs(), nan=math.inf, posinf=math.inf) - HALF_STEP[o.dtype] * want.abs() - bound - HALF_SUBNORMAL[o.dtype]
    error = torch.where(want.abs() > 0.99 * torch.finfo(o.dtype).max, -1.0, error)[rows]
    assert bool((error <= 0).all()), f"{float(error.max())} above the bound"


def setup(call, page, dim, dtype, seed):
    new, lengths, group = CALLS[call]
    pages = sum(-(-n // page) for n in lengths) + 1
    cache, _ = make_cache(pages, 2, page, dim, seed)
    starts = starts_of(new)
    q = torch.randn(int(starts[-1]), 2 * group, dim, generator=torch.Generator().manual_seed(seed + 1)).to(dtype).cuda()
    return cache, q, make_table(lengths, page, pages, seed + 2), lengths, starts


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("page,dim", [(16, 64), (32, 128), (64, 128), (128, 64), (16, 96), (32, 256)])
@pytest.mark.parametrize("call", CALLS)
def test_values_of_pages_that_a_row_does_not_see(dtype, page, dim, call):
    """The newest page of each sequence stands for far larger values than all others: finite ones, and then NaN."""
    cache, q, table, lengths, starts = setup(call, page, dim, dtype, 41)
    last = torch.tensor([int(table[b, (n - 1) // page]) for b, n in enumerate(lengths)]).cuda()
    ordinary = cache.v_scale[last].clone()
    scale = 1.5 / math.sqrt(dim)
    for factor in (2.0 ** 20, 1e19, 1e30):
        cache.v_scale[last] = ordinary * factor
        o, lse = run(cache, q, table, lengths, starts, scale)
        want, want_lse, bound, seen_of = definition(cache, q, table, lengths, starts, scale)
        check(o, want, bound, slice(None))
        assert bool(((lse - want_lse).abs() <= 2.0 ** -14).all())
    cache.v_scale[last] = float("nan")
    o, lse = run(cache, q, table, lengths, starts, scale)
    want, want_lse, bound, seen_of = definition(cache, q, table, lengths, starts, scale)
    end_of = [lengths[b] for b in range(len(lengths)) for _ in range(int(starts[b + 1] - starts[b]))]
    before = torch.tensor([seen <= (end - 1) // page * page for seen, end in zip(seen_of, end_of)]).cuda()
    assert bool(before.any()) and bool((~before).any())
    check(o, want, bound, before)
    assert bool(o[~before].isnan().all())
    assert bool(((lse - want_lse).abs() <= 2.0 ** -14).all())  # the sum of exponentials is one of keys alone


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (32, 256)])
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("power", [-40, 40, 90])
def test_values_far_from_the_others_that_nobody_attends_to(dtype, page, dim, call, power):
    """The first page of each sequence holds values 2^power times the others' behind scores far below all others."""
    cache, q, table, lengths, starts = setup(call, page, dim, dtype, 44)
    first = torch.tensor([int(table[b, 0]) for b in range(len(lengths))]).cuda()
    cache.k[first] = -120  # q is positive: these scores are negative, the others' of both signs
    cache.k_scale[first] = 0.25
    cache.v_scale[first] *= 2.0 ** power
    q = (q.abs() + 0.4).to(dtype)
    o, lse = run(cache, q, table, lengths, starts, 1 / math.sqrt(dim))
    want, want_lse, bound, seen_of = definition(cache, q, table, lengths, starts, 1 / math.sqrt(dim))
    rows = torch.tensor(seen_of).cuda() > page + 16  # they see others
    assert bool(rows.any())
    check(o, want, bound, rows)
    assert bool(((lse - want_lse).abs() <= 2.0 ** -13)[rows].all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("scales", [(1e-36, 1e-36), (1e30, 1e30), (1e-30, 1e30), (0.0, 1.0), (0.0, 0.0), (1e-38, 1.0)], ids=str)
def test_value_scales_at_the_ends_of_their_range(dtype, call, scales):
    """Blocks whose value scales take turns between two numbers; values beyond fp16 are not looked at."""
    cache, q, table, lengths, starts = setup(call, 32, 128, dtype, 47)
    turn = torch.arange(cache.v_scale.shape[0], device="cuda")[:, None] % 2 == 0
    cache.v_scale.copy_(torch.where(turn, scales[0], scales[1]).expand_as(cache.v_scale))
    o, lse = run(cache, q, table, lengths, starts, 0.1)
    want, want_lse, bound, _ = definition(cache, q, table, lengths, starts, 0.1)
    check(o, want, bound, slice(None))
    assert bool(((lse - want_lse).abs() <= 2.0 ** -14).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (32, 256)])
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("order", ["first", "last"])
def test_pages_without_values_that_have_all_the_weight(dtype, page, dim, call, order):
    """The first page, or the last that all rows see whole, has value scale 0 and scores some 2^95 above all others; those grow by 2^40 on
    their way. What is left of a row is 2^-95 of its other pages' average, as exact as if it were all."""
    cache, q, table, lengths, starts = setup(call, page, dim, dtype, 56)
    q = (q.abs() * 0.05 + 1.0).to(dtype)
    for b, length in enumerate(lengths):
        known = (length - int(starts[b + 1] - starts[b])) // page  # pages that all of its rows see whole
        pages = torch.from_numpy(table[b, :-(-length // page)].copy()).long().cuda()
        for i, at in enumerate(pages.tolist()):  # scores of 2^-20 .. 2^20 around 0
            cache.k[at] = 0
            cache.k[at, :, :, 0] = -100 + 200 * i // max(1, len(pages) - 1)
            cache.k_scale[at] = 0.2
        if known > 1:
            at = pages[0 if order == "first" else known - 1]
            cache.k[at], cache.k_scale[at], cache.v_scale[at] = 100, 86 / 100 / dim, 0.0
    o, lse = run(cache, q, table, lengths, starts, 1.0)
    want, want_lse, bound, _ = definition(cache, q, table, lengths, starts, 1.0)
    check(o, want, bound, slice(None))
    assert bool(((lse - want_lse).abs() <= 2.0 ** -13).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("values", [0.02, 1e-9, 3e5])
@pytest.mark.parametrize("scale", [30.0, 3e4, 1e6])
def test_scores_far_from_zero(dtype, call, values, scale):
    """Scores of thousands to 10^8: one key has all of a row's weight but e^-30 unless the next one is within the scores' own rounding (rows
    for which it is are not looked at). Then the result is its value: the weight's rounding, the result's, and e^-30 of the others,
    whatever log2 of the value scale is beside the score."""
    cache, q, table, lengths, starts = setup(call, 32, 128, dtype, 50)
    cache.v_scale.fill_(values)
    o, lse = run(cache, q, table, lengths, starts, scale)
    heads, page, dim = cache.k.shape[1:]
    looked_at = 0
    for b, length in enumerate(lengths):
        n = int(starts[b + 1] - starts[b])
        pages = torch.from_numpy(table[b, :-(-length // page)]).long().cuda()
        k, v = ((c[pages].double() * s[pages].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :length] for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        for i in range(n):
            row = int(starts[b]) + i
            x = q[row].double().unflatten(0, (heads, -1))
            seen = length - n + i + 1
            z = torch.einsum("hgd,hkd->hgk", x, k[:, :seen]) * scale
            error = (dim / 16) * 2.0 ** -22 * scale * (x.abs().sum(-1) * 255 * 0.025)
            two, at = z.topk(2, dim=-1)
            clear = (two[..., 0] - two[..., 1] > 2 * error + 30).flatten()
            want = torch.stack([v[h, at[h, :, 0]] for h in range(heads)]).flatten(0, 1)
            off = (o[row].double() - want).abs() - (HALF_STEP[dtype] + (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -11 + 2.0 ** -20)) * want.abs() - HALF_SUBNORMAL[dtype]
            others = seen * math.exp(-30) * 127 * values
            lost = 0 if dtype == torch.float32 else 2.0 ** -27 * 128 * seen * values  # of sums with 128 beside every code
            off = torch.where(want.abs() > 0.99 * torch.finfo(dtype).max, -1.0, off - lost - others)
            assert bool((off[clear] <= 0).all()), float(off[clear].max())
            assert bool(((lse[row].double() - two[..., 0].flatten()).abs() <= error.flatten() + 2.0 ** -22 * two[..., 0].abs().flatten() + 2.0 ** -19)[clear].all())
            looked_at += int(clear.sum())
    assert looked_at > 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("scale,keys,queries", [(1e33, 1e-33, 1), (1e38, 1e-36, 1e-2), (1e-30, 1e30, 1), (1e-33, 1, 1e33), (1e-1, 1e-36, 1e37), (1e30, 1, 1e-30)])
def test_scales_of_scores_keys_and_queries_that_make_up_for_one_another(dtype, call, scale, keys, queries):
    """Ordinary scores from numbers that are not; a row of zeros has scores of zero whatever the scale."""
    if dtype == torch.float16 and queries not in (1, 1e-2):
        pytest.skip("queries beyond fp16")
    cache, q, table, lengths, starts = setup(call, 32, 128, dtype, 53)
    cache.k_scale.mul_(keys)
    q = (q.double() * queries).to(dtype)
    q[0] = 0
    o, lse = run(cache, q, table, lengths, starts, scale * 0.1)
    want, want_lse, bound, _ = definition(cache, q, table, lengths, starts, float(torch.tensor(scale * 0.1, dtype=torch.float32)))
    check(o, want, bound, slice(None))
    assert bool(((lse - want_lse).abs() <= 2.0 ** -14).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 12), (96, 4), (256, 2)])
@pytest.mark.parametrize("length", [8192, 131072])
def test_averages_over_many_keys(dtype, dim, group, length):
    """q = 0: every key has the same probability, and value scales of 11 bits are exact as fp16 weights, so nothing is rounded but sums and the
    result. What it costs to carry 128 with every code may not grow with the number of keys: between two corrections there are 8 steps of
    16 keys, each off by 2^-22 of at most 255 times the weights since the last, together 2^-11 of the sum of the weights, which is below 2.
    The codes' own sum: a step is off by 2^-22 of it; after k of a warp's n keys it is below six deviations, 6 * 73.6 * 1.5 sqrt(k), so over
    n / 16 steps and divided by n it is 2^-22 * 6 * 110 * (2 / 3) sqrt(n) / 16, for a warp's 37900 keys at most (head dimension 256: three
    warps) 2^-9.6."""
    heads, seqs, page = 4, 64, 128
    cuda = cuda_mod()
    pages = length // page
    cache = cuda.KvCache.empty(pages, heads, dim, page)
    g = torch.Generator(device="cuda").manual_seed(47)
    for codes in (cache.k, cache.v):
        codes.copy_(torch.randint(-127, 128, codes.shape, generator=g, device="cuda", dtype=torch.int8))
    cache.k_scale.fill_(1.0)
    cache.v_scale.copy_(1 + torch.randint(0, 1024, cache.v_scale.shape, generator=g, device="cuda") / 1024)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(seqs, pages).contiguous()  # all sequences read the same pages
    lengths = torch.full((seqs,), length, dtype=torch.int32, device="cuda")
    q = torch.zeros(seqs, heads * group, dim, dtype=dtype, device="cuda")
    o = cuda.cached_attention(q, cache, table, lengths, 1.0).double()
    want = (cache.v.double() * cache.v_scale.double()[:, :, None, None]).mean(dim=(0, 2)).repeat_interleave(group, 0)
    worst = ((o - want).abs() - HALF_STEP[dtype] * want.abs()).max()
    assert float(worst) <= 2.0 ** -10 + 2.0 ** -9.6, float(worst)
