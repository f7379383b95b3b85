"""Where mhlo_cuda_kv_cache_read puts its results: both, one or none of the tensors given, of any strides."""
import pytest
import torch

from test_kv_cache_gpu import cuda_mod, make_cache, make_table, on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("layout", ["slice", "head_major", "plain"])
def test_one_result_given(dtype, layout):
    cuda = cuda_mod()
    heads, dim, page, lengths, most = 3, 48, 16, [5, 40, 0], 33
    cache, _ = make_cache(5, heads, page, dim, 70)
    args = (cache, on_gpu(make_table(lengths, page, 5, 71)), on_gpu(lengths), most)
    want_k, want_v = cuda.kv_cache_read(*args, dtype=dtype)

    def given():
        if layout == "slice":  # columns of a wider tensor, off the 16-byte grid
            return torch.full((3, most, heads, dim + 5), 2.0, dtype=dtype, device="cuda")[..., 1:dim + 1]
        if layout == "head_major":
            return torch.full((3, heads, most, dim), 2.0, dtype=dtype, device="cuda").transpose(1, 2)
        return torch.full((3, most, heads, dim), 2.0, dtype=dtype, device="cuda")

    for which in ("k_out", "v_out"):
        out = given()
        k, v = cuda.kv_cache_read(*args, **{which: out})
        assert (k if which == "k_out" else v) is out and k.dtype == v.dtype == dtype
        assert torch.equal(k, want_k) and torch.equal(v, want_v)
    a, b = given(), given()
    k, v = cuda.kv_cache_read(*args, k_out=a, v_out=b)
    assert k is a and v is b and torch.equal(k, want_k) and torch.equal(v, want_v)
    assert cuda.device_error() == 0
