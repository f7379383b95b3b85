"""mhlo_cuda_device_error with several words set: each call reports and clears one, and what reads some of them leaves the others."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def bad_page(cuda, attend):
    """A call whose page table names no page of the cache: append (or attention) records code 1."""
    cache = cuda.KvCache.empty(2, 1, 64, 16)
    table, lengths = torch.full((1, 1), 7, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 1, 64, device="cuda")
    if attend:
        cuda.cached_attention(x, cache, table, lengths, 1.0)
    else:
        cuda.kv_cache_append(cache, x, x, table, lengths)


def take(cuda):
    code = C.c_int32(0)
    return cuda.lib.mhlo_cuda_device_error(C.byref(code)), code.value


def test_words_are_reported_one_after_the_other():
    from metalhlo_b200 import cuda

    assert cuda.device_error() == 0
    assert cuda.lib.mhlo_cuda_debug_store_device_error(0, 3) == 0 and cuda.lib.mhlo_cuda_debug_store_device_error(1, 8) == 0
    bad_page(cuda, attend=False)
    bad_page(cuda, attend=True)
    failed = 8  # MHLO_CUDA_EXECUTION_FAILED
    assert [take(cuda) for _ in range(5)] == [(failed, 3), (failed, 108), (failed, 201), (failed, 201), (0, 0)]
    bad_page(cuda, attend=False)
    assert take(cuda) == (failed, 201) and "a page outside the cache" in cuda.last_error()
    assert take(cuda) == (0, 0)


def test_a_tuner_neither_takes_nor_minds_the_words_of_the_cache(tmp_path):
    """In a process of its own: what a tuner measures goes into the process's database, and compiled programs take it from there."""
    program = """
import sys
sys.path.insert(0, "tests")
from test_device_error_words_gpu import bad_page
from metalhlo_b200 import capi, cuda
bad_page(cuda, attend=False)
capi.tuning.open(sys.argv[1])
client = capi.Client()
assert capi.tuning.tune_gemm(client, capi.F16, 1, 256, 256, 256, max_trials=2)["configsTried"] == 2
assert capi.tuning.tune_attention(client, capi.BF16, 1, 2, 256, 256, 64)["configsTried"] >= 1
assert cuda.device_error() == 201 and cuda.device_error() == 0
print("left alone")
"""
    r = subprocess.run([sys.executable, "-c", program, str(tmp_path / "gemm.json")], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "left alone" in r.stdout, r.stderr[-2000:]
