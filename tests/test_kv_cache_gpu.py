"""The paged 8-bit key/value cache and the attention over it against numpy (tests/kv_reference.py).

Appending is defined operation by operation in fp32, so codes and scales are compared bit for bit. Rotated queries: two products
and a sum in fp32, each off by 2^-24 of its own size at most, then one rounding to the type. Below the smallest normal number the steps of a type no longer
shrink: there a rounding is off by up to half of (smallest normal * eps), for fp16 2^-14 * 2^-10 / 2 = 2^-25 whatever the value.

Attention: with u = half a step of the result's type, an output is off by u |o| and by sum p |v| times the relative error of a
weight. That error is twice a score's absolute error (numerator and denominator) plus the weight's own rounding: 2^-11 where weights
are held in fp16 (16-bit types), 2^-20 for exponential, sums and the two-part weights of fp32. A score is a sum of head_dim products in
steps of 16, each step off by 2^-22 of the sum of magnitudes at most (the tensor cores cut their sums off). Weights far below the
largest one vanish: in fp16 times 2^14 (fp32 inputs) or 2^6 (others) the last step is 2^-24, so each key may lose 2^-39 or 2^-31 of the
largest weight times the largest value.

With 16-bit inputs the sums carry 128 with every code (code + 128 is what is multiplied) and lose it at the end. So a score's sum of
magnitudes is that of |q| (|k| + 128 scale); and in an output each step of 16 keys is off by 2^-23 of a sum of up to 128 times the
weights (which add up to 1) times the largest scale: n / 16 steps make n * 128 * 2^-27 scale, that is 2^-27 of (n * 127 * scale), whatever |v|.
"""
import math

import numpy as np
import pytest
import torch

import kv_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
HALF_SUBNORMAL = {t: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for t in HALF_STEP}


def cuda_mod():
    from metalhlo_b200 import cuda

    return cuda


def make_cache(pages, heads, page, dim, seed):
    """A pool whose pages hold something already."""
    g = torch.Generator().manual_seed(seed)
    codes = [torch.randint(-127, 128, (pages, heads, page, dim), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [0.005 + 0.02 * torch.rand(pages, heads, generator=g) for _ in range(2)]
    return cuda_mod().KvCache(*(t.cuda() for t in codes + scales)), ref.Cache(*(t.numpy() for t in codes + scales))


def make_table(lengths, page, pages, seed, extra=0):
    """Pages of the pool in any order; entries that no sequence reaches are no pages at all."""
    counts = [-(-max(0, n) // page) for n in lengths]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = np.full((len(lengths), max(counts + [1]) + extra), -7, np.int32)
    for b, n in enumerate(counts):
        table[b, :n] = order[:n]
        del order[:n]
    return table


def on_gpu(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def assert_same_cache(cache, want):
    for got, exp in ((cache.k_scale, want.scales[0]), (cache.v_scale, want.scales[1])):
        np.testing.assert_array_equal(got.cpu().numpy(), exp)
    for got, exp in ((cache.k, want.codes[0]), (cache.v, want.codes[1])):
        np.testing.assert_array_equal(got.cpu().numpy(), exp)


def assert_rotated(got, x, want_rows, rope, positions, interleaved, dtype):
    """|error| <= 2^-23 (|a c| + |b s|) + half a step."""
    got, x = got.double().cpu().numpy(), x.double().cpu().numpy()
    for row, pos in zip(want_rows, positions):
        t = rope[pos].astype(np.float64)
        want = ref.rotate(x[row], t, interleaved)
        size = ref.rotate(np.abs(x[row]), np.concatenate([np.abs(t[:t.size // 2]), -np.abs(t[t.size // 2:])]), interleaved)
        # second elements: b c + a s with the sine's sign turned round
        size = np.maximum(size, ref.rotate(np.abs(x[row]), np.abs(t), interleaved))
        bound = 2.0 ** -23 * size + HALF_STEP[dtype] * np.abs(want) * (1 + 2.0 ** -8) + HALF_SUBNORMAL[dtype]
        assert bool(np.all(np.abs(got[row] - want) <= bound)), f"row {row}: {np.max(np.abs(got[row] - want) - bound)} above the bound"


SETS = [  # new tokens, lengths with them
    ([1, 1, 1, 1, 1], [1, 16, 17, 64, 129]),
    ([5, 0, 33, 1, 130], [5, 40, 33, 128, 200]),
    ([257], [300]),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,lengths", SETS, ids=["one_each", "ragged", "long"])
@pytest.mark.parametrize("page,heads,dim,rotary,interleaved", [(16, 3, 64, 64, False), (64, 2, 128, 128, True), (32, 1, 96, 32, False), (128, 2, 256, 256, False),
                                                               (16, 5, 16, 16, True), (64, 2, 80, 48, False)])
def test_append(dtype, new, lengths, page, heads, dim, rotary, interleaved):
    cuda = cuda_mod()
    g = torch.Generator().manual_seed(dim + page)
    starts = starts_of(new)
    tokens, behind = int(starts[-1]), 3  # rows of no sequence
    if new == [1] * len(new):
        behind = 0
    pages = sum(-(-n // page) for n in lengths) + 2
    cache, want = make_cache(pages, heads, page, dim, 1)
    table = make_table(lengths, page, pages, 2, extra=1)
    q_heads = 2 * heads
    qkv = torch.randn(tokens + behind, q_heads + 2 * heads, dim, generator=g).to(dtype)
    rope = ref.rope_rows(max(lengths), rotary)
    d = qkv.cuda()
    q, k, v = d[:, :q_heads], d[:, q_heads:q_heads + heads], d[:, q_heads + heads:]
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    plain = new == [1] * len(new)
    r = cuda.kv_cache_append(cache, k, v, on_gpu(table), on_gpu(lengths), token_starts=None if plain else on_gpu(starts),
                             rope=torch.from_numpy(rope).cuda(), interleaved=interleaved, q=q, q_out=out)
    assert r is out and cuda.device_error() == 0
    x = qkv.float().numpy()
    want.append(x[:, q_heads:q_heads + heads], x[:, q_heads + heads:], table, lengths, starts, rope, interleaved)
    assert_same_cache(cache, want)
    rows = [(int(starts[b]) + i, lengths[b] - new[b] + i) for b in range(len(new)) for i in range(new[b])]
    assert_rotated(out, q, [r for r, _ in rows], rope, [p for _, p in rows], interleaved, dtype)
    assert bool((out[tokens:] == 7).all())


@pytest.mark.parametrize("offset", [0, 1])
def test_append_of_tensors_off_the_16_byte_grid(offset):
    cuda = cuda_mod()
    cache, want = make_cache(5, 2, 16, 32, 3)
    table, lengths, new = make_table([40], 16, 5, 4), [40], [29]
    flat = torch.randn(29 * 131 + 8, generator=torch.Generator().manual_seed(5)).half()
    x = flat.cuda()[offset:offset + 29 * 131].view(29, 131)
    k, v, q = (x[:, i:i + 64].unflatten(1, (2, 32)) for i in (0, 66, 30))
    rope = ref.rope_rows(40, 32)
    out = cuda.kv_cache_append(cache, k, v, on_gpu(table), on_gpu(lengths), token_starts=on_gpu(starts_of(new)), rope=torch.from_numpy(rope).cuda(), q=q)
    want.append(k.float().cpu().numpy(), v.float().cpu().numpy(), table, lengths, starts_of(new), rope)
    assert_same_cache(cache, want)
    assert_rotated(out, q, range(29), rope, range(11, 40), False, torch.float16)


def test_append_token_by_token_rewrites_growing_blocks():
    """Values that double every few tokens: every scale grows several times while its block fills. The stored values stay within
    half a step per growth of what was put in."""
    cuda = cuda_mod()
    heads, dim, page, n = 2, 64, 16, 40
    cache, want = make_cache(4, heads, page, dim, 6)
    table = make_table([n], page, 4, 7)
    g = torch.Generator().manual_seed(8)
    k = torch.randn(n, heads, dim, generator=g) * (2.0 ** (torch.arange(n) / 3.0))[:, None, None]
    v = torch.randn(n, heads, dim, generator=g)
    steps = []
    for t in range(n):
        cuda.kv_cache_append(cache, k[t:t + 1].cuda(), v[t:t + 1].cuda(), on_gpu(table), on_gpu([t + 1]))
        want.append(k[t:t + 1].numpy(), v[t:t + 1].numpy(), table, [t + 1], [0, 1])
        steps.append(cache.k_scale[int(table[0, t // page])].cpu().double().numpy())
    assert_same_cache(cache, want)
    got, _ = cuda.kv_cache_read(cache, on_gpu(table), on_gpu([n]), n)
    for t in range(n):
        last = min(n, (t // page + 1) * page)
        bound = sum(0.5 * steps[j] * (1 + 2.0 ** -15) for j in range(t, last) if j == t or np.any(steps[j] > steps[j - 1]))
        assert np.all(np.abs(got[0, t].cpu().double().numpy() - k[t].double().numpy()) <= bound[:, None])


def test_append_of_values_that_are_not_finite_zero_or_tiny():
    cuda = cuda_mod()
    heads, dim, page = 4, 32, 16
    cache, want = make_cache(3, heads, page, dim, 9)
    table, lengths, starts = np.array([[2, 0]], np.int32), [20], [0, 20]
    k = torch.randn(20, heads, dim, generator=torch.Generator().manual_seed(10))
    v = k.clone()
    k[3, 0, 5], k[2, 1, 0], v[19, 2, 1] = float("nan"), float("-inf"), float("inf")
    v[:16, 3] = 0
    k[16:, 3] = 1e-37
    cuda.kv_cache_append(cache, k.cuda(), v.cuda(), on_gpu(table), on_gpu(lengths), token_starts=on_gpu(starts))
    want.append(k.numpy(), v.numpy(), table, lengths, starts)
    assert_same_cache(cache, want)
    assert np.isnan(want.scales[0][2, :2]).all() and want.scales[1][2, 3] == 0 and want.scales[0][0, 3] == 0
    # a later token into the poisoned block leaves it so; a fresh start clears it
    one = torch.ones(1, heads, dim)
    for lengths in ([21], [17]):
        cuda.kv_cache_append(cache, one.cuda(), one.cuda(), on_gpu(table), on_gpu(lengths))
        want.append(one.numpy(), one.numpy(), table, lengths, [0, 1])
    assert_same_cache(cache, want)
    assert np.isnan(want.scales[0][2, 0]) and np.isfinite(want.scales[1][0]).all()
    k, v = cuda.kv_cache_read(cache, on_gpu(table), on_gpu([17]), 17)
    assert bool(k[0, :16, :2].isnan().all()) and bool((k[0, 16] - 1).abs().max() < 2.0 ** -22) and bool((v[0, :16, 3] == 0).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128), (32, 80)])
def test_read(dtype, page, dim):
    cuda = cuda_mod()
    lengths = [0, 1, page, 2 * page + 3]
    cache, want = make_cache(9, 3, page, dim, 11)
    table = make_table(lengths, page, 9, 12)
    most = 2 * page + 1  # one sequence is longer, the others are filled up with zeros
    k, v = cuda.kv_cache_read(cache, on_gpu(table), on_gpu(lengths), most, dtype=dtype)
    assert cuda.device_error() == 0 and k.shape == (4, most, 3, dim)
    for b, n in enumerate(lengths):
        n = min(n, most)
        for which, got in ((0, k), (1, v)):
            x = torch.from_numpy(want.values(which, table[b], n)[0].astype(np.float32)) if n else torch.zeros(0, 3, dim)
            codes = torch.from_numpy(np.zeros((0, 3, dim), np.float32)) if not n else torch.from_numpy(
                (want.codes[which][table[b, :-(-n // page)]].astype(np.float32) * want.scales[which][table[b, :-(-n // page)]][:, :, None, None])
                .transpose(0, 2, 1, 3).reshape(-1, 3, dim)[:n])
            assert torch.equal(got[b, :n].cpu(), codes.to(dtype)) and x.shape == codes.shape
            assert bool((got[b, n:] == 0).all())
    # into a head-major tensor
    kt = torch.empty(4, 3, most, dim, dtype=dtype, device="cuda").transpose(1, 2)
    k2, v2 = cuda.kv_cache_read(cache, on_gpu(table), on_gpu(lengths), most, k_out=kt)
    assert k2 is kt and torch.equal(k2, k) and torch.equal(v2, v)


def check_attention(cache, want, q, table, lengths, starts, scale, got, lse, before):
    dtype = q.dtype
    o, want_lse, magnitude, products, reach = ref.attention(want, q.double().cpu().numpy(), table, lengths, starts, scale, before,
                                                              bias=0 if dtype == torch.float32 else 128)
    dim = q.shape[2]
    score = (dim / 16) * 2.0 ** -22 * scale * products
    weight = 2 * score + (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -11 + 2.0 ** -20)
    lost = 2.0 ** -39 if dtype == torch.float32 else 2.0 ** -31 + 2.0 ** -27 * (128 / 127)
    bound = HALF_STEP[dtype] * np.abs(o) + weight[:, :, None] * magnitude + lost * reach[:, :, None] + HALF_SUBNORMAL[dtype]
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    worst = np.max((np.abs(got - o) - bound) / (magnitude + 1e-30))
    assert worst <= 0, f"{worst} of sum p |v| above the bound"
    if lse is not None:
        lse = lse.double().cpu().numpy()
        inside = ~np.isnan(want_lse)
        assert np.array_equal(np.isinf(lse[inside]), np.isinf(want_lse[inside]))
        fin = inside & np.isfinite(want_lse)
        assert np.all(np.abs(lse[fin] - want_lse[fin]) <= score[fin] + 2.0 ** -19 + 2.0 ** -22 * np.abs(want_lse[fin]))


ATTENTION_SETS = [
    ([1, 1, 1, 1, 1, 1], [1, 15, 16, 17, 300, 1025]),
    ([3, 1, 0, 5, 2], [3, 64, 10, 129, 700]),
    ([70, 1, 33], [70, 65, 200]),
    ([1], [5000]),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("new,lengths", ATTENTION_SETS, ids=["one_each", "few", "chunks", "long"])
@pytest.mark.parametrize("page,heads,group,dim", [(16, 2, 1, 64), (64, 2, 4, 128), (32, 1, 7, 96), (128, 1, 16, 128), (64, 1, 3, 256), (16, 1, 33, 64)])
def test_attention(dtype, new, lengths, page, heads, group, dim):
    cuda = cuda_mod()
    starts = starts_of(new)
    pages = sum(-(-n // page) for n in lengths) + 1
    cache, want = make_cache(pages, heads, page, dim, 13)
    table = make_table(lengths, page, pages, 14)
    plain = new == [1] * len(new)
    behind = 0 if plain else 2
    q = torch.randn(int(starts[-1]) + behind, heads * group, dim, generator=torch.Generator().manual_seed(15)).to(dtype).cuda()
    out, lse = torch.full_like(q, 3.0), torch.zeros(q.shape[:2], device="cuda")
    scale = 1 / math.sqrt(dim)
    r = cuda.cached_attention(q, cache, on_gpu(table), on_gpu(lengths), scale, token_starts=None if plain else on_gpu(starts), out=out, lse=lse)
    assert r is out and cuda.device_error() == 0
    check_attention(cache, want, q, table, lengths, starts, scale, out, lse, np.full(q.shape, 3.0))
    again = cuda.cached_attention(q, cache, on_gpu(table), on_gpu(lengths), scale, token_starts=None if plain else on_gpu(starts))
    assert torch.equal(again[:int(starts[-1])], out[:int(starts[-1])])  # no order of arrival in the result


@pytest.mark.parametrize("new", [[0, 1, 1, 1], [4, 4, 4, 4], [40, 3, 2, 50]], ids=str)
def test_attention_of_unused_entries_and_far_scores(new):
    """Length 0 marks an unused entry: zeros. Large scores put all weight on one key, and blocks far below the maximum vanish."""
    cuda = cuda_mod()
    starts, page, heads, group, dim = starts_of(new), 32, 2, 4, 128
    lengths = [0, 100, 0, 230]
    cache, want = make_cache(12, heads, page, dim, 16)
    table = make_table(lengths, page, 12, 17)
    for w, s in ((want.scales[0], cache.k_scale), (want.scales[1], cache.v_scale)):  # blocks of very unequal size
        w *= np.float32(8.0) ** (np.arange(12) % 4 - 2).astype(np.float32)[:, None]
        s.copy_(torch.from_numpy(w))
    for dtype in TYPES:
        q = (4 * torch.randn(int(starts[-1]), heads * group, dim, generator=torch.Generator().manual_seed(18))).to(dtype).cuda()
        lse = torch.zeros(q.shape[:2], device="cuda")
        got = cuda.cached_attention(q, cache, on_gpu(table), on_gpu(lengths), 0.3, token_starts=on_gpu(starts), lse=lse)
        assert cuda.device_error() == 0
        check_attention(cache, want, q, table, lengths, starts, 0.3, got, lse, np.zeros(q.shape))


def test_attention_reads_and_writes_strided_rows_and_in_place():
    cuda = cuda_mod()
    page, heads, group, dim, lengths, new = 16, 2, 3, 64, [50, 31], [2, 9]
    starts = starts_of(new)
    cache, want = make_cache(7, heads, page, dim, 19)
    table = make_table(lengths, page, 7, 20)
    wide = torch.randn(11, 10, dim, generator=torch.Generator().manual_seed(21)).bfloat16().cuda()
    q = wide[:, 3:9]
    out = torch.zeros(6, 11, dim, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    cuda.cached_attention(q, cache, on_gpu(table), on_gpu(lengths), 0.125, token_starts=on_gpu(starts), out=out)
    check_attention(cache, want, q, table, lengths, starts, 0.125, out, None, np.zeros(q.shape))
    odd = torch.randn(11 * 391, generator=torch.Generator().manual_seed(22)).half().cuda().view(11, 391)[:, 1:385].unflatten(1, (6, dim))  # off the 16-byte grid
    got = cuda.cached_attention(odd, cache, on_gpu(table), on_gpu(lengths), 0.125, token_starts=on_gpu(starts))
    check_attention(cache, want, odd, table, lengths, starts, 0.125, got, None, np.zeros(q.shape))
    rest = wide.clone()
    cuda.cached_attention(q, cache, on_gpu(table), on_gpu(lengths), 0.125, token_starts=on_gpu(starts), out=q)
    assert torch.equal(q, out) and torch.equal(wide[:, :3], rest[:, :3]) and torch.equal(wide[:, 9:], rest[:, 9:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (128, 128)])
def test_chunks_off_the_grid_in_place_and_with_rows_behind(dtype, dim, page):
    """Many rows: tensors whose rows are off the 16-byte grid, results in place of the queries, one sequence of few rows in a call that
    could have held many, and rows behind the last sequence."""
    cuda = cuda_mod()
    heads, group = 2, 4
    for new, lengths, behind in (([150, 1, 40], [150, 77, 700], 3), ([5], [333], 60), ([129], [1000], 0)):
        starts = starts_of(new)
        pages = sum(-(-n // page) for n in lengths) + 1
        cache, want = make_cache(pages, heads, page, dim, 31)
        table = make_table(lengths, page, pages, 32)
        rows, width = int(starts[-1]) + behind, heads * group * dim + 6
        flat = torch.randn(rows, width, generator=torch.Generator().manual_seed(33)).to(dtype).cuda()
        q = flat[:, 3:3 + heads * group * dim].unflatten(1, (heads * group, dim))
        args = (cache, on_gpu(table), on_gpu(lengths), 0.11)
        lse = torch.full(q.shape[:2], 5.0, device="cuda")
        out = torch.full(q.shape, 2.0, dtype=dtype, device="cuda")
        cuda.cached_attention(q, *args, token_starts=on_gpu(starts), out=out, lse=lse)
        assert cuda.device_error() == 0
        check_attention(cache, want, q, table, lengths, starts, 0.11, out, lse, np.full(q.shape, 2.0))
        assert bool((lse[int(starts[-1]):] == 5).all())
        before = flat.clone()
        cuda.cached_attention(q, *args, token_starts=on_gpu(starts), out=q)
        assert torch.equal(q[:int(starts[-1])], out[:int(starts[-1])])
        assert torch.equal(flat[int(starts[-1]):], before[int(starts[-1]):]) and torch.equal(flat[:, :3], before[:, :3]) and torch.equal(flat[:, -3:], before[:, -3:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_chunks_of_unequal_blocks_and_growing_scores(dtype):
    """Value scales that differ by 2^12 and blocks without values (scale 0), key norms that grow along the sequence: the maximum moves
    many times, and what was summed up before is scaled anew."""
    cuda = cuda_mod()
    page, heads, group, dim, lengths, new = 32, 2, 8, 128, [900, 333], [40, 333]
    starts = starts_of(new)
    cache, want = make_cache(42, heads, page, dim, 34)
    table = make_table(lengths, page, 42, 35)
    for b, n in enumerate(lengths):
        for i in range(-(-n // page)):
            want.scales[0][table[b, i]] *= np.float32(0.05 * (i + 1))
            want.scales[1][table[b, i]] *= np.float32(0.0 if i % 5 == 3 else 4.0 ** (i % 7 - 3))
    cache.k_scale.copy_(torch.from_numpy(want.scales[0]))
    cache.v_scale.copy_(torch.from_numpy(want.scales[1]))
    q = (2 * torch.randn(int(starts[-1]), heads * group, dim, generator=torch.Generator().manual_seed(36))).to(dtype).cuda()
    lse = torch.zeros(q.shape[:2], device="cuda")
    got = cuda.cached_attention(q, cache, on_gpu(table), on_gpu(lengths), 0.2, token_starts=on_gpu(starts), lse=lse)
    assert cuda.device_error() == 0
    check_attention(cache, want, q, table, lengths, starts, 0.2, got, lse, np.zeros(q.shape))


def test_a_poisoned_block_reaches_only_rows_that_see_it():
    cuda = cuda_mod()
    page, dim = 16, 64
    cache, _ = make_cache(6, 1, page, dim, 23)
    table, lengths, new = make_table([40, 40], page, 6, 24), [40, 40], [20, 20]
    cache.v_scale[int(table[0, 2])] = float("nan")  # positions 32 ..: seen by the last 8 rows of sequence 0
    cache.k_scale[int(table[1, 2])] = float("nan")
    for dtype in TYPES:
        q = torch.randn(40, 2, dim, generator=torch.Generator().manual_seed(25)).to(dtype).cuda()
        o = cuda.cached_attention(q, cache, on_gpu(table), on_gpu(lengths), 0.125, token_starts=on_gpu(starts_of(new))).cpu()
        for b in range(2):
            assert bool(o[20 * b:20 * b + 12].isfinite().all()) and bool(o[20 * b + 12:20 * b + 20].isnan().all())


def test_pages_lengths_and_starts_that_cannot_be_are_reported_and_not_followed():
    cuda = cuda_mod()
    page, heads, dim = 16, 2, 64
    lengths, new = [40, 20], [10, 20]
    starts = starts_of(new)
    g = torch.Generator().manual_seed(26)
    k, v = (torch.randn(30, heads, dim, generator=g) for _ in range(2))
    q = torch.randn(30, heads, dim, generator=g)
    rope = ref.rope_rows(40, dim)

    def run(table, lengths, starts, code, known=True, rope=rope):
        cache, want = make_cache(6, heads, page, dim, 27)
        cuda.kv_cache_append(cache, k.cuda(), v.cuda(), on_gpu(table), on_gpu(lengths), token_starts=on_gpu(starts), rope=torch.from_numpy(rope).cuda(), q=q.cuda())
        assert cuda.device_error() == code
        if known:
            want.append(k.numpy(), v.numpy(), np.asarray(table), lengths, starts, rope)
            assert_same_cache(cache, want)
        if code == 204:
            return
        o = cuda.cached_attention(q.cuda(), cache, on_gpu(table), on_gpu(lengths), 0.125, token_starts=on_gpu(starts))
        assert cuda.device_error() == code
        if known:
            check_attention(cache, want, q.cuda(), np.asarray(table), lengths, starts, 0.125, o, None, np.zeros(q.shape))
        cuda.kv_cache_read(cache, on_gpu(table), on_gpu(lengths), 40)
        cuda.device_error()

    good = make_table(lengths, page, 6, 28)
    run(good, lengths, starts, 0)
    for entry in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        bad = good.copy()
        bad[0, 2] = entry
        run(bad, lengths, starts, 201)
    for bad in ([40, 49], [40, 19], [-3, 20], [2 ** 31 - 1, 20]):
        run(good, bad, starts, 202)
    for bad in ([0, 40, 30], [0, 10, 2 ** 31 - 1], [-5, 10, 30], [0, 10, 5]):
        run(good, lengths, bad, 203, known=False)
    run(good, lengths, starts, 204, rope=rope[:35])


def test_the_three_together_on_other_streams_and_in_a_replayed_graph():
    """A decoding loop as a program runs it: rotate and append a token, attend; eager on a side stream, then captured once and
    replayed with new inputs in the same buffers. Both give the bits of the eager loop on the default stream."""
    cuda = cuda_mod()
    page, heads, group, dim, seqs, steps = 32, 2, 4, 128, 3, 40
    g = torch.Generator().manual_seed(29)
    qkv = torch.randn(steps, seqs, heads * (group + 2), dim, generator=g).bfloat16().cuda()
    table = on_gpu(np.arange(6).reshape(3, 2)[:, ::-1].copy())
    rope = cuda.rope_table(64, dim)

    def step(cache, x, lengths, out, stream=None):
        q = cuda.kv_cache_append(cache, x[:, heads * group:heads * (group + 1)], x[:, heads * (group + 1):], table, lengths, rope=rope, q=x[:, :heads * group], stream=stream)
        return cuda.cached_attention(q, cache, table, lengths, 0.09, out=out, stream=stream)

    def loop(run):
        cache = cuda.KvCache.empty(6, heads, dim, page)
        x, lengths = qkv[0].clone(), torch.zeros(seqs, dtype=torch.int32, device="cuda")
        out = torch.zeros(seqs, heads * group, dim, dtype=torch.bfloat16, device="cuda")
        results = []
        call = run(cache, x, lengths, out)
        for t in range(steps):
            x.copy_(qkv[t])
            lengths.add_(1)
            torch.cuda.synchronize()
            call()
            torch.cuda.synchronize()
            results.append(out.clone())
        return torch.stack(results), cache

    eager, c0 = loop(lambda *a: lambda: step(*a))
    side = torch.cuda.Stream()
    other, c1 = loop(lambda *a: lambda: step(*a, stream=side.cuda_stream))

    def captured(cache, x, lengths, out):
        graph = torch.cuda.CUDAGraph()
        lengths.add_(1)
        step(cache, x, lengths, out)  # before the capture, as programs warm up; the cache starts afresh with the first token
        lengths.sub_(1)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            step(cache, x, lengths, out)
        return graph.replay

    replayed, c2 = loop(captured)
    assert cuda.device_error() == 0
    assert torch.equal(eager, other) and torch.equal(eager, replayed)
    for c in (c1, c2):
        assert torch.equal(c.k, c0.k) and torch.equal(c.v_scale, c0.v_scale)
    # against dense attention over what the cache stands for
    k, v = (t.double() for t in cuda.kv_cache_read(c0, table, torch.full((seqs,), steps, dtype=torch.int32, device="cuda"), steps))
    q = cuda.kv_cache_append(cuda.KvCache.empty(6, heads, dim, page), *(qkv[-1][:, i * heads:(i + 1) * heads] for i in (group, group + 1)), table,
                             torch.full((seqs,), steps, dtype=torch.int32, device="cuda"), rope=rope, q=qkv[-1][:, :heads * group]).double()
    z = torch.einsum("bhgd,bkhd->bhgk", q.unflatten(1, (heads, group)), k) * 0.09
    want = torch.einsum("bhgk,bkhd->bhgd", z.softmax(-1), v).flatten(1, 2)
    size = torch.einsum("bhgk,bkhd->bhgd", z.softmax(-1), v.abs()).flatten(1, 2)
    assert bool(((eager[-1].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -15) * size).all())


def test_empty_calls():
    cuda = cuda_mod()
    cache, want = make_cache(2, 1, 16, 64, 30)
    none = torch.zeros(0, 1, 64, device="cuda")
    table, lengths = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    cuda.kv_cache_append(cache, none, none, table, lengths)
    assert cuda.cached_attention(none, cache, table, lengths, 1.0).shape == (0, 1, 64)
    k, _ = cuda.kv_cache_read(cache, table, lengths, 5)
    assert k.shape == (0, 5, 1, 64)
    assert_same_cache(cache, want)
