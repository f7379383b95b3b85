"""Sequences of many rows (and of few beside them) whose pages, lengths, starts or scales are not what they should be, in calls that cut
them between CTAs: what the kernels meet is reported and not followed, and nobody else notices. Bounds as in test_kv_cache_gpu.py."""
import numpy as np
import pytest
import torch

import kv_reference as ref
from test_kv_cache_gpu import check_attention, cuda_mod, make_cache, make_table, on_gpu, starts_of

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
HEADS, GROUP = 1, 2
NEW, LENGTHS = [130, 3, 70], [700, 520, 410]  # 260, 6 and 140 rows


def setup(dtype, dim, page, seed):
    starts, behind = starts_of(NEW), 2
    pages = sum(-(-n // page) for n in LENGTHS) + 1
    cache, want = make_cache(pages, HEADS, page, dim, seed)
    q = torch.randn(int(starts[-1]) + behind, HEADS * GROUP, dim, generator=torch.Generator().manual_seed(seed + 1)).to(dtype).cuda()
    return cache, want, q, make_table(LENGTHS, page, pages, seed + 2), starts, pages


def run(cache, q, table, lengths, starts, scale=0.09):
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 4.0, device="cuda")
    cuda_mod().cached_attention(q, cache, on_gpu(table), on_gpu(lengths), scale, token_starts=on_gpu(starts), out=out, lse=lse)
    assert bool((out[int(starts_of(NEW)[-1]):] == 3).all()) and bool((lse[int(starts_of(NEW)[-1]):] == 4).all())  # rows behind the last sequence
    return out, lse


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (128, 128)])
@pytest.mark.parametrize("entry", [-1, "pages", 2 ** 31 - 1, -2 ** 31])
def test_pages_that_are_none(dtype, dim, page, entry):
    """In the middle of one sequence, at the end of another, and all of a third: their keys count as masked."""
    cache, want, q, table, starts, pages = setup(dtype, dim, page, 60)
    bad = pages if entry == "pages" else entry
    for b, which in ((0, [200 // page, 201 // page]), (2, [(LENGTHS[2] - 1) // page]), (1, range(-(-LENGTHS[1] // page)))):
        table[b, list(which)] = bad
    o, lse = run(cache, q, table, LENGTHS, starts)
    assert cuda_mod().device_error() == 201 and cuda_mod().device_error() == 0  # both kernels may have met one: reported once
    check_attention(cache, want, q, table, LENGTHS, starts, 0.09, o, lse, np.full(q.shape, 3.0))
    first = int(starts[1])
    assert bool((o[first:first + NEW[1]] == 0).all()) and bool((lse[first:first + NEW[1]] == -float("inf")).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("lengths", [[129, 520, 410], [-1, 520, 410], [2 ** 31 - 1, 520, 410], [700, 520, 69], [0, 520, 410], [700, 0, 0]], ids=str)
def test_lengths_that_cannot_be_and_unused_entries(dtype, dim, page, lengths):
    """A sequence with such a length is passed over: its rows get zeros and log-sum-exp -infinity."""
    cache, want, q, table, starts, _ = setup(dtype, dim, page, 63)
    o, lse = run(cache, q, table, lengths, starts)
    wrong = any(n < 0 or (n != 0 and n < k) or n > table.shape[1] * page for n, k in zip(lengths, NEW))
    assert cuda_mod().device_error() == (202 if wrong else 0) and cuda_mod().device_error() == 0
    check_attention(cache, want, q, table, lengths, starts, 0.09, o, lse, np.full(q.shape, 3.0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("starts", [[0, 130, 100, 203], [0, 130, 133, 2 ** 31 - 1], [-5, 130, 133, 203], [0, 130, 133, 20], [203, 0, 0, 203]], ids=str)
def test_starts_out_of_order(dtype, starts):
    """Rows may be left alone; nothing outside the call's rows is touched, and the next call is right."""
    dim, page = 128, 64
    cache, want, q, table, good, _ = setup(dtype, dim, page, 66)
    run(cache, q, table, LENGTHS, starts)
    assert cuda_mod().device_error() in (202, 203)  # a sequence that is too long for its length is reported as such
    assert cuda_mod().device_error() == 0
    o, lse = run(cache, q, table, LENGTHS, good)
    assert cuda_mod().device_error() == 0
    check_attention(cache, want, q, table, LENGTHS, good, 0.09, o, lse, np.full(q.shape, 3.0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32)])
def test_blocks_that_are_no_numbers(dtype, dim, page):
    """A NaN scale of keys or of values reaches the rows that see its block, and no other."""
    cache, want, q, table, starts, _ = setup(dtype, dim, page, 69)
    reached = np.zeros(int(starts[-1]), bool)
    for b, scales in ((0, cache.v_scale), (2, cache.k_scale)):
        page_of = (LENGTHS[b] - 20) // page
        scales[int(table[b, page_of])] = float("nan")
        reached[int(starts[b]):int(starts[b + 1])] = np.arange(LENGTHS[b] - NEW[b], LENGTHS[b]) >= page_of * page
    o, lse = run(cache, q, table, LENGTHS, starts)
    assert cuda_mod().device_error() == 0 and reached.any() and not reached.all()
    rows = torch.from_numpy(np.concatenate([reached, [False, False]])).cuda()
    assert bool(o[rows].isnan().all())
    expect = ref.attention(want, q.double().cpu().numpy(), table, LENGTHS, starts, 0.09, np.full(q.shape, 3.0))
    o[rows] = torch.from_numpy(expect[0]).cuda()[rows].to(dtype)
    lse[rows] = torch.from_numpy(expect[1]).cuda()[rows].float()
    check_attention(cache, want, q, table, LENGTHS, starts, 0.09, o, lse, np.full(q.shape, 3.0))
