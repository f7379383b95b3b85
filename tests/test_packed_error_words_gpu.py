"""Error words of the packed operators: one call of mhlo_cuda_device_error reports one, what other calls recorded is left for the next."""
import pytest
import torch

from tests.packed_reference import inputs

pytestmark = pytest.mark.gpu


def test_words_of_several_calls_are_reported_one_after_the_other():
    from metalhlo_b200 import cuda

    assert cuda.device_error() == 0
    x = inputs([64, 64], 2, 2, 64, torch.bfloat16)
    other = cuda.packed_plan(x["starts_dev"], 128, 2, 2, causal=False)
    wrong = cuda.packed_plan(x["starts_dev"], 128, 2, 2)
    wrong._args.plan = other.tiles.data_ptr()
    lse = torch.zeros(128, 2, device="cuda")
    o = torch.zeros_like(x["q"])

    def start():
        cuda.packed_plan(torch.tensor([0, 100, 50, 128], dtype=torch.int32, device="cuda"), 128, 2, 2)

    def forward():
        cuda.packed_attention(x["q"], x["k"], x["v"], wrong, 0.1, out=o, lse=lse)

    def backward():
        cuda.packed_attention_grad(x["q"], x["k"], x["v"], o, lse, x["grad"], wrong, 0.1)

    for calls, codes in (((start, forward), [203, 205]), ((forward, backward), [205, 205]), ((start, forward, backward), [203, 205, 205]), ((backward,), [205]), ((start, backward), [203, 205])):
        for call in calls:
            call()
        assert [cuda.device_error() for _ in range(len(codes) + 1)] == codes + [0]


def test_the_word_of_the_norms_gradients():
    """A copy that does not come is reported (the word is written from the host here), behind what others met."""
    from metalhlo_b200 import cuda

    assert cuda.device_error() == 0
    assert cuda.lib.mhlo_cuda_debug_store_device_error(2, 40) == 0
    cuda.packed_plan(torch.tensor([0, 100, 50, 128], dtype=torch.int32, device="cuda"), 128, 2, 2)
    assert [cuda.device_error() for _ in range(2)] == [203, 240] and "bounded wait (code 240)" in cuda.last_error()
    assert cuda.device_error() == 0
    x = torch.randn(4, 1024, device="cuda")
    cuda.layer_norm_grad(x, None, x)
    assert cuda.device_error() == 0


def test_texts_name_no_other_operator():
    from metalhlo_b200 import cuda

    cuda.packed_plan(torch.tensor([0, 100, 50, 128], dtype=torch.int32, device="cuda"), 128, 2, 2)
    assert cuda.device_error() == 203 and "cached or packed sequences met starts out of order (code 203)" in cuda.last_error()
    assert cuda.lib.mhlo_cuda_debug_store_device_error(2, 40) == 0
    assert cuda.device_error() == 240 and "tensor-core" not in cuda.last_error()
