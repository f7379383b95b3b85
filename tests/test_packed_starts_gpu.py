"""Starts of packed sequences that go back: what is reported, and that a plan never holds more tiles than it has room for."""
import pytest
import torch

from tests.packed_reference import inputs

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
ROW_TILES, KEY_TILES = 5, 6  # words of a plan


def plan_of(starts, tokens, q_heads=2, kv_heads=2):
    from metalhlo_b200 import cuda

    return cuda.packed_plan(torch.tensor(starts, dtype=torch.int32, device="cuda"), tokens, q_heads, kv_heads)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("starts", [[0, 192, 0, 192], [0, 192, 100, 192], [0, 150, 0, 150, 0, 150], [0, 64, 1, 64, 1, 64, 1, 64, 1, 192]], ids=str)
def test_more_tokens_than_there_are(dtype, starts):
    """Nothing is computed, forward or backward."""
    from metalhlo_b200 import cuda

    x = inputs([192], 2, 2, 64, dtype)
    plan = plan_of(starts, 192)
    assert cuda.device_error() == 203 and cuda.device_error() == 0
    assert plan.tiles[ROW_TILES] == 0 and plan.tiles[KEY_TILES] == 0
    lse = torch.full((192, 2), 7.0, device="cuda")
    outs = [torch.full(x[n].shape, 7.0, dtype=dtype, device="cuda") for n in ("q", "q", "k", "v")]
    cuda.packed_attention(x["q"], x["k"], x["v"], plan, 0.1, out=outs[0], lse=lse)
    cuda.packed_attention_grad(x["q"], x["k"], x["v"], outs[0], lse, x["grad"], plan, 0.1, *outs[1:])
    assert cuda.device_error() == 0 and all((t == 7.0).all() for t in (*outs, lse))


def test_sequences_over_one_another_that_fit():
    """Rows that only one sequence has are what they are without the other."""
    from metalhlo_b200 import cuda

    x = inputs([192], 2, 2, 64, BF16)
    want, out = (torch.full((192, 2, 64), 7.0, dtype=BF16, device="cuda") for _ in range(2))
    cuda.packed_attention(x["q"], x["k"], x["v"], plan_of([0, 64], 192), 0.1, out=want)
    assert cuda.device_error() == 0
    cuda.packed_attention(x["q"], x["k"], x["v"], plan_of([0, 64, 32, 64], 192), 0.1, out=out)
    assert cuda.device_error() == 203
    assert torch.equal(out[:32], want[:32]) and (out[64:] == 7.0).all()


@pytest.mark.parametrize("pairs", [300, 2000])
def test_starts_whose_tiles_no_32_bits_count(pairs):
    """Sequences of 2^30 tokens again and again have 2^31 tiles and more between them."""
    from metalhlo_b200 import cuda

    tokens = 1 << 30
    plan = plan_of([0, tokens] * pairs, tokens, 1, 1)
    assert cuda.device_error() == 203 and cuda.device_error() == 0
    assert plan.tiles[ROW_TILES] == 0 and plan.tiles[KEY_TILES] == 0
    del plan
    # one of them fills the lists
    plan = plan_of([0, tokens], tokens, 1, 1)
    assert cuda.device_error() == 0
    assert plan.tiles[ROW_TILES] == tokens // 256 and plan.tiles[KEY_TILES] == tokens // 128


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("starts", [[100, 150, 50, 60], [60, 90, 30, 50, 50, 10, 20], [120, 192, 0, 120]], ids=str)
def test_sequences_in_front_of_earlier_ones(dtype, starts):
    """A start that goes back without another sequence's rows being met: those around it have the results and gradients that they have alone."""
    from metalhlo_b200 import cuda

    x = inputs([192], 2, 2, 64, dtype)

    def run(starts):
        plan = plan_of(starts, 192)
        lse = torch.zeros(192, 2, device="cuda")
        o = cuda.packed_attention(x["q"], x["k"], x["v"], plan, 0.1, lse=lse)
        scratch = torch.full((1 << 18,), float("nan"), device="cuda")  # what lay in memory before is no result
        del scratch
        return (o, lse, *cuda.packed_attention_grad(x["q"], x["k"], x["v"], o, lse, x["grad"], plan, 0.1))

    got = run(starts)
    assert cuda.device_error() == 203
    for a, b in zip(starts, starts[1:]):
        if b <= a:
            continue
        alone = run([a, b])
        assert cuda.device_error() == 0
        for g, w in zip(got, alone):
            assert torch.isfinite(w[a:b]).all()
            # few tiles of keys are cut into shares by the number of sequences, and added in another order
            assert (g[a:b].double() - w[a:b].double()).abs().max() <= 4 * torch.finfo(dtype).eps * w[a:b].double().abs().max()
