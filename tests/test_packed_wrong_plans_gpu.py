"""A plan that is not of the call's batch is reported and nothing is written, in either half and by every kernel."""
import pytest
import torch

from tests.packed_reference import inputs

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def other_plan(x, which):
    from metalhlo_b200 import cuda

    starts = {"fewer": [0, 192], "more": [0, 1, 2, 3, 64, 64, 100, 128, 192]}.get(which)
    starts = x["starts_dev"] if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    tokens = 193 if which == "tokens" else 192
    heads = {"kv_heads": (4, 4), "q_heads": (8, 2)}.get(which, (4, 2))
    return cuda.packed_plan(starts, tokens, *heads, causal=which != "causal")


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("which", ["fewer", "more", "tokens", "q_heads", "kv_heads", "causal"])
def test_both_halves(dtype, dim, which):
    from metalhlo_b200 import cuda

    x = inputs([64, 64, 64], 4, 2, dim, dtype)
    good, other = cuda.packed_plan(x["starts_dev"], 192, 4, 2), other_plan(x, which)
    mixed = cuda.packed_plan(x["starts_dev"], 192, 4, 2)
    mixed._args.plan = other.tiles.data_ptr()
    lse = torch.empty(192, 4, device="cuda")
    o = cuda.packed_attention(x["q"], x["k"], x["v"], good, 0.1, lse=lse)
    assert cuda.device_error() == 0
    out, out_lse = torch.full_like(o, 7.0), torch.full_like(lse, 7.0)
    cuda.packed_attention(x["q"], x["k"], x["v"], mixed, 0.1, out=out, lse=out_lse)
    assert cuda.device_error() == 205 and (out == 7.0).all() and (out_lse == 7.0).all()
    grads = [torch.full(x[n].shape, 7.0, dtype=dtype, device="cuda") for n in ("q", "k", "v")]
    cuda.packed_attention_grad(x["q"], x["k"], x["v"], o, lse, x["grad"], mixed, 0.1, *grads)
    assert cuda.device_error() == 205 and all((g == 7.0).all() for g in grads)
