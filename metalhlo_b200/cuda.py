"""ctypes binding of ``libmhlo_cuda.so`` (declared in ``include/mhlo_cuda.h``).

This is the thin Python view of the device runtime used by the tests and the benchmark. It adds nothing to
the C ABI: every function takes raw device pointers (for example ``torch.Tensor.data_ptr()``), sizes and a
CUDA stream handle, and a non-zero status raises :class:`MhloCudaError` with the library's message.
There is no fallback: if the shared library has not been built, importing this module raises.
"""
from __future__ import annotations

import collections
import ctypes as C
import functools
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libmhlo_cuda.so")

F16, F32, F64, BF16, I1, I8, I16, I32, I64, UI8, UI16, UI32, UI64 = range(13)


class MhloCudaError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"mhlo_cuda status {status}: {message}")
        self.status = status


class RowTuning(C.Structure):
    _fields_ = [("threads", C.c_int32), ("vecs_per_thread", C.c_int32), ("ctas_per_sm", C.c_int32)]


class RowHead(C.Structure):
    _fields_ = [("gamma", C.c_void_p), ("beta", C.c_void_p), ("y", C.c_void_p), ("value", C.c_float), ("op", C.c_int32)]


class RowHeads(C.Structure):
    _fields_ = [("head", RowHead * 3), ("count", C.c_int32)]


class View(C.Structure):
    _fields_ = [("base", C.c_void_p), ("dtype", C.c_int32), ("rank", C.c_int32), ("shape", C.c_int64 * 8),
                ("stride", C.c_int64 * 8)]


class EwInst(C.Structure):
    _fields_ = [("op", C.c_int32), ("a", C.c_int32), ("b", C.c_int32), ("c", C.c_int32), ("imm", C.c_double)]


class ConvertJob(C.Structure):
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("count", C.c_int64), ("src_dtype", C.c_int32), ("dst_dtype", C.c_int32)]


class GatherDims(C.Structure):
    _fields_ = [("n_offset_dims", C.c_int32), ("n_collapsed", C.c_int32), ("n_operand_batching", C.c_int32),
                ("n_start_index_map", C.c_int32), ("offset_dims", C.c_int32 * 8), ("collapsed_slice_dims", C.c_int32 * 8),
                ("operand_batching_dims", C.c_int32 * 8), ("start_indices_batching_dims", C.c_int32 * 8),
                ("start_index_map", C.c_int32 * 8), ("index_vector_dim", C.c_int32), ("slice_sizes", C.c_int64 * 8)]


class Window(C.Structure):
    _fields_ = [("rank", C.c_int32), ("size", C.c_int64 * 8), ("stride", C.c_int64 * 8), ("base_dilation", C.c_int64 * 8),
                ("window_dilation", C.c_int64 * 8), ("pad_low", C.c_int64 * 8)]


class Conv(C.Structure):
    _fields_ = [("n_spatial", C.c_int32), ("reverse", C.c_int32 * 6), ("batch", C.c_int64), ("in_features", C.c_int64),
                ("out_features", C.c_int64), ("feature_group_count", C.c_int64), ("batch_group_count", C.c_int64),
                ("in_size", C.c_int64 * 6), ("kernel_size", C.c_int64 * 6), ("out_size", C.c_int64 * 6), ("stride", C.c_int64 * 6),
                ("pad_low", C.c_int64 * 6), ("lhs_dilation", C.c_int64 * 6), ("rhs_dilation", C.c_int64 * 6),
                ("in_batch_stride", C.c_int64), ("in_feature_stride", C.c_int64), ("in_spatial_stride", C.c_int64 * 6),
                ("kernel_in_stride", C.c_int64), ("kernel_out_stride", C.c_int64), ("kernel_spatial_stride", C.c_int64 * 6),
                ("out_batch_stride", C.c_int64), ("out_feature_stride", C.c_int64), ("out_spatial_stride", C.c_int64 * 6)]


class ScatterDims(C.Structure):
    _fields_ = [("n_update_window_dims", C.c_int32), ("n_inserted_window_dims", C.c_int32), ("n_input_batching", C.c_int32),
                ("n_scatter_dims_to_operand", C.c_int32), ("update_window_dims", C.c_int32 * 8),
                ("inserted_window_dims", C.c_int32 * 8), ("input_batching_dims", C.c_int32 * 8),
                ("scatter_indices_batching_dims", C.c_int32 * 8), ("scatter_dims_to_operand_dims", C.c_int32 * 8),
                ("index_vector_dim", C.c_int32)]


class KvCacheArgs(C.Structure):
    _fields_ = [("k_codes", C.c_void_p), ("v_codes", C.c_void_p), ("k_scales", C.c_void_p), ("v_scales", C.c_void_p), ("pages", C.c_int64),
                ("heads", C.c_int64), ("page_tokens", C.c_int64), ("head_dim", C.c_int64)]


class KvBatchArgs(C.Structure):
    _fields_ = [("page_table", C.c_void_p), ("lengths", C.c_void_p), ("token_starts", C.c_void_p), ("seqs", C.c_int64),
                ("pages_per_seq", C.c_int64), ("table_stride", C.c_int64), ("tokens", C.c_int64)]


if not os.path.exists(LIB_PATH):
    raise ImportError(
        f"{LIB_PATH} is missing: build it with `make -C metalhlo_b200/csrc` "
        "(or `python -c 'import __graft_entry__ as g; g.build()'`). There is no CPU fallback."
    )

lib = C.CDLL(LIB_PATH)

_vp, _i64, _i32, _f32, _sz = C.c_void_p, C.c_int64, C.c_int32, C.c_float, C.c_size_t
_PROTOTYPES = {
    "mhlo_cuda_version": (C.c_char_p, []),
    "mhlo_cuda_last_error": (C.c_char_p, []),
    "mhlo_cuda_dtype_size": (_sz, [C.c_int]),
    "mhlo_cuda_device_count": (C.c_int, [C.POINTER(C.c_int)]),
    "mhlo_cuda_device_set": (C.c_int, [C.c_int]),
    "mhlo_cuda_device_current": (C.c_int, [C.POINTER(C.c_int)]),
    "mhlo_cuda_device_name": (C.c_int, [C.c_int, C.c_char_p, _sz]),
    "mhlo_cuda_stream_create": (C.c_int, [C.POINTER(_vp)]),
    "mhlo_cuda_stream_destroy": (C.c_int, [_vp]),
    "mhlo_cuda_stream_sync": (C.c_int, [_vp]),
    "mhlo_cuda_alloc": (C.c_int, [_sz, C.POINTER(_vp)]),
    "mhlo_cuda_free": (C.c_int, [_vp]),
    "mhlo_cuda_host_alloc": (C.c_int, [_sz, C.POINTER(_vp)]),
    "mhlo_cuda_host_free": (C.c_int, [_vp]),
    "mhlo_cuda_upload": (C.c_int, [_vp, _vp, _sz, _vp]),
    "mhlo_cuda_download": (C.c_int, [_vp, _vp, _sz, _vp]),
    "mhlo_cuda_copy": (C.c_int, [_vp, _vp, _sz, _vp]),
    "mhlo_cuda_memset": (C.c_int, [_vp, C.c_int, _sz, _vp]),
    "mhlo_cuda_event_create": (C.c_int, [C.POINTER(_vp)]),
    "mhlo_cuda_event_destroy": (C.c_int, [_vp]),
    "mhlo_cuda_event_record": (C.c_int, [_vp, _vp]),
    "mhlo_cuda_event_elapsed_ms": (C.c_int, [_vp, _vp, C.POINTER(_f32)]),
    "mhlo_cuda_layer_norm": (C.c_int, [C.c_int, _vp, _vp, _vp, _vp, _i64, _i64, _f32, C.POINTER(RowTuning), _vp]),
    "mhlo_cuda_rms_norm": (C.c_int, [C.c_int, _vp, _vp, _vp, _i64, _i64, _f32, C.POINTER(RowTuning), _vp]),
    "mhlo_cuda_softmax": (C.c_int, [C.c_int, _vp, _vp, _i64, _i64, _i64, C.POINTER(RowTuning), _vp]),
    "mhlo_cuda_row_group": (C.c_int, [C.c_int, _vp, C.POINTER(RowHeads), _i64, _i64, _vp]),
    "mhlo_cuda_batch_norm": (C.c_int, [C.c_int, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, C.c_float, _vp]),
    "mhlo_cuda_elementwise": (C.c_int, [C.POINTER(View), _i32, C.POINTER(EwInst), _i32, _vp, _i32, C.POINTER(_i64), _i32, _vp]),
    "mhlo_cuda_elementwise_to_view": (C.c_int, [C.POINTER(View), _i32, C.POINTER(EwInst), _i32, C.POINTER(View), _vp]),
    "mhlo_cuda_reduce": (C.c_int, [C.POINTER(View), _i32, _i32, _vp, _vp, _vp, _i32, _vp]),
    "mhlo_cuda_add_layer_norm": (C.c_int, [C.c_int, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, C.c_float, C.POINTER(RowTuning), _vp]),
    "mhlo_cuda_add_rms_norm": (C.c_int, [C.c_int, _vp, _vp, _vp, _vp, _vp, _i64, _i64, C.c_float, C.POINTER(RowTuning), _vp]),
    "mhlo_cuda_fft_axis": (C.c_int, [C.c_int, C.c_int, _vp, _vp, _i64, _i64, _i64, _vp]),
    "mhlo_cuda_fft_axis_scratch_bytes": (_i64, [C.c_int, _i64, _i64, _i64]),
    "mhlo_cuda_fft_axis_long": (C.c_int, [C.c_int, C.c_int, _vp, _vp, _vp, _i64, _i64, _i64, _vp]),
    "mhlo_cuda_add_layer_norm_rows": (C.c_int, [C.c_int, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _i64, _i64, C.c_float, C.POINTER(RowTuning), _vp]),
    "mhlo_cuda_add_rms_norm_rows": (C.c_int, [C.c_int, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _i64, C.c_float, C.POINTER(RowTuning), _vp]),
    "mhlo_cuda_graph_capture_begin": (C.c_int, [_vp]),
    "mhlo_cuda_graph_capture_end": (C.c_int, [_vp, C.POINTER(_vp)]),
    "mhlo_cuda_graph_launch": (C.c_int, [_vp, _vp]),
    "mhlo_cuda_graph_destroy": (C.c_int, [_vp]),
    "mhlo_cuda_ipc_export": (C.c_int, [_vp, C.c_char_p]),
    "mhlo_cuda_ipc_open": (C.c_int, [C.c_char_p, C.POINTER(_vp)]),
    "mhlo_cuda_ipc_close": (C.c_int, [_vp]),
    "mhlo_cuda_gemm_all_gather": (C.c_int, [_i32, _i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), C.POINTER(_vp), _i32, _i32, _i64, _i64, _i64,
                                            _vp, _i32, _vp]),
    "mhlo_cuda_gemm_all_gather_tuned": (C.c_int, [_i32, _i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), C.POINTER(_vp), _i32, _i32, _i64, _i64,
                                                  _i64, _vp, _i32, _vp, _i32, _vp]),
    "mhlo_cuda_gemm_residual": (C.c_int, [_i32, _i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, _i64, _i64, _i64, _i64, _i64, _vp, _vp,
                                          _vp, _vp]),
    "mhlo_cuda_event_sync": (C.c_int, [_vp]),
    "mhlo_cuda_stream_wait_event": (C.c_int, [_vp, _vp]),
    "mhlo_cuda_stream_host_callback": (C.c_int, [_vp, _vp, _vp]),
    "mhlo_cuda_conv2d_nhwc": (C.c_int, [_i32, _i32, _vp, _vp, _vp] + [_i64] * 13 + [_vp, _i32, _vp]),
    "mhlo_cuda_conv2d_nhwc_strided": (C.c_int, [_i32, _i32, _vp, _vp, _vp] + [_i64] * 15 + [_vp, _i32, _vp]),
    "mhlo_cuda_rng": (C.c_int, [_i32, _i32, _vp, _vp, _vp, _vp, _i64, _vp]),
    "mhlo_cuda_rng_bit_generator": (C.c_int, [_vp, _vp, _vp, _i64, _i32, _vp]),
    "mhlo_cuda_peer_barrier": (C.c_int, [C.POINTER(_vp), _i32, _i32, C.c_uint64, C.c_uint64, _vp]),
    "mhlo_cuda_convert_many": (C.c_int, [C.POINTER(ConvertJob), _i32, _vp]),
    "mhlo_cuda_reduce_static_scratch": (C.c_int, [C.POINTER(View), _i32, _i32, _vp, _vp, _vp, _i32, _i32, _vp]),
    "mhlo_cuda_gather": (C.c_int, [_vp, _i32, C.POINTER(_i64), _i32, _vp, _i32, C.POINTER(_i64), _i32, C.POINTER(GatherDims),
                                   _vp, C.POINTER(_i64), _i32, _vp]),
    "mhlo_cuda_convolution": (C.c_int, [_i32, _vp, _vp, _vp, C.POINTER(Conv), _vp]),
    "mhlo_cuda_im2col": (C.c_int, [_i32, _vp, _vp, _i64, C.POINTER(Conv), _vp]),
    "mhlo_cuda_reduce_window": (C.c_int, [C.POINTER(View), C.POINTER(Window), _i32, _vp, _vp, C.POINTER(_i64), _vp]),
    "mhlo_cuda_select_and_scatter": (C.c_int, [C.POINTER(View), _vp, C.POINTER(_i64), _vp, C.POINTER(Window), _i32, _i32, _vp, _vp]),
    "mhlo_cuda_scatter": (C.c_int, [_vp, _i32, C.POINTER(_i64), _i32, _vp, _i32, C.POINTER(_i64), _i32, _vp, C.POINTER(_i64), _i32,
                                    C.POINTER(ScatterDims), _i32, _vp]),
    "mhlo_cuda_sort_scratch_bytes": (_i64, [C.POINTER(_i64), _i32, _i32]),
    "mhlo_cuda_sort": (C.c_int, [C.POINTER(_vp), C.POINTER(_vp), C.POINTER(_i32), _i32, C.POINTER(_i64), _i32, _i32, _i32, _vp, _i64, _vp]),
    "mhlo_cuda_dynamic_slice": (C.c_int, [_vp, _i32, C.POINTER(_i64), _i32, C.POINTER(_vp), _i32, C.POINTER(_i64), _vp, _vp]),
    "mhlo_cuda_dynamic_update_slice": (C.c_int, [_vp, _i32, C.POINTER(_i64), _i32, _vp, C.POINTER(_i64), C.POINTER(_vp), _i32, _vp]),
    "mhlo_cuda_dot_strided": (C.c_int, [_i32, _i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, _i64, _i64, _i64, _i64, _i64, _vp]),
    "mhlo_cuda_gemm": (C.c_int, [_i32, _i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, _i64, _i64, _i64, _i64, _i64, _vp,
                                 _i32, _vp]),
    "mhlo_cuda_cholesky": (C.c_int, [_i32, _vp, _vp, _i64, _i64, _i32, _vp]),
    "mhlo_cuda_triangular_solve": (C.c_int, [_i32, _vp, _vp, _vp, _i64, _i64, _i64, _i32, _i32, _i32, _i32, _vp]),
    "mhlo_cuda_kernel_lookup": (C.c_int, [C.c_char_p, _i32, C.POINTER(_i32)]),
    "mhlo_cuda_plan_create": (C.c_int, [_vp, _i32, _i32, _i32, _i64, C.c_char_p, _i64, C.POINTER(_vp)]),
    "mhlo_cuda_plan_execute": (C.c_int, [_vp, C.POINTER(_vp), _i32, C.POINTER(_vp), _i32, _vp]),
    "mhlo_cuda_plan_destroy": (C.c_int, [_vp]),
    "mhlo_cuda_tuner_measure": (C.c_int, [_vp, C.POINTER(_vp), _i32, C.POINTER(_vp), _i32, _i32, _i32, C.POINTER(_f32)]),
    "mhlo_cuda_comm_init": (C.c_int, [_i32, C.POINTER(_vp)]),
    "mhlo_cuda_comm_size": (C.c_int, [_vp]),
    "mhlo_cuda_all_gather": (C.c_int, [_vp, C.POINTER(_vp), _i64]),
    "mhlo_cuda_comm_destroy": (C.c_int, [_vp]),
    "mhlo_cuda_gemm_tuned": (C.c_int, [_i32, _i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, _i64, _i64, _i64, _i64, _i64, _vp,
                                       _i32, _vp, _vp]),
    "mhlo_cuda_device_error": (C.c_int, [C.POINTER(_i32)]),
    "mhlo_cuda_device_error_fetch": (C.c_int, [_vp]),
    "mhlo_cuda_device_error_take": (C.c_int, [C.POINTER(_i32)]),
    "mhlo_cuda_debug_store_device_error": (C.c_int, [_i32, _i32]),
    "mhlo_cuda_debug_refuse_allocs": (C.c_int, [_i32]),
    "mhlo_cuda_debug_wait_expiry_probe": (C.c_int, [C.c_uint64, _vp]),
    "mhlo_cuda_attention": (C.c_int, [_i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, _vp,
                                      C.POINTER(_i64), _i64, _i64, _i64, _i64, _i64, _f32, _i32, _vp]),
    "mhlo_cuda_attention_tuned": (C.c_int, [_i32, _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp, _vp,
                                            C.POINTER(_i64), _i64, _i64, _i64, _i64, _i64, _f32, _i32, _vp, _vp]),
    "mhlo_cuda_kv_cache_append": (C.c_int, [_i32, C.POINTER(KvCacheArgs), C.POINTER(KvBatchArgs), _vp, C.POINTER(_i64), _vp, C.POINTER(_i64), _vp,
                                            C.POINTER(_i64), _vp, C.POINTER(_i64), _i64, _vp, _i64, _i64, _i32, _vp]),
    "mhlo_cuda_kv_cache_read": (C.c_int, [_i32, C.POINTER(KvCacheArgs), C.POINTER(KvBatchArgs), _i64, _vp, _vp, C.POINTER(_i64), _vp]),
    "mhlo_cuda_cached_attention_scratch_bytes": (_i64, [C.POINTER(KvCacheArgs), C.POINTER(KvBatchArgs), _i64]),
    "mhlo_cuda_cached_attention": (C.c_int, [_i32, _vp, C.POINTER(_i64), C.POINTER(KvCacheArgs), C.POINTER(KvBatchArgs), _i64, _f32, _vp,
                                             C.POINTER(_i64), _vp, _vp, _i64, _vp]),
    "mhlo_cuda_token_logprobs": (C.c_int, [_i32, _vp, _i64, _i64, _i64, _f32, _vp, _i32, _vp, _vp, _vp, _i32, _vp, _vp, _vp]),
    "mhlo_cuda_token_logprobs_grad": (C.c_int, [_i32, _vp, _i64, _i64, _i64, _f32, _vp, _i32, _vp, _vp, _vp, _vp, _i32, _vp, _vp, _vp, _i64, _vp]),
}
for _name, (_res, _args) in _PROTOTYPES.items():
    _fn = getattr(lib, _name)  # AttributeError here = the library does not export a declared symbol
    _fn.restype = _res
    _fn.argtypes = _args


def declared_symbols() -> list[str]:
    """Names bound above; the CPU test suite checks them against ``include/mhlo_cuda.h``."""
    return sorted(_PROTOTYPES)


def last_error() -> str:
    return lib.mhlo_cuda_last_error().decode()


def check(status: int) -> None:
    if status != 0:
        raise MhloCudaError(status, last_error())


@functools.lru_cache(maxsize=None)
def torch_dtype_code(dtype) -> int:
    import torch

    return {torch.float16: F16, torch.float32: F32, torch.float64: F64, torch.bfloat16: BF16, torch.bool: I1,
            torch.int8: I8, torch.int16: I16, torch.int32: I32, torch.int64: I64, torch.uint8: UI8}[dtype]


def _stream(stream=None) -> int:
    if stream is not None:
        return int(stream)
    import torch

    return torch.cuda.current_stream().cuda_stream


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


def _tuning(t):
    if t is None:
        return None
    if isinstance(t, RowTuning):
        return C.byref(t)
    return C.byref(RowTuning(*t))


def layer_norm(x, gamma, beta, eps: float = 1e-5, out=None, tuning=None, stream=None):
    """LayerNorm over the last axis of a contiguous CUDA tensor (see ``mhlo_cuda_layer_norm``)."""
    import torch

    assert x.is_cuda and x.is_contiguous()
    out = torch.empty_like(x) if out is None else out
    hidden = x.shape[-1]
    rows = x.numel() // hidden if hidden else 0
    check(lib.mhlo_cuda_layer_norm(torch_dtype_code(x.dtype), _ptr(x), _ptr(gamma), _ptr(beta), _ptr(out), rows,
                                   hidden, eps, _tuning(tuning), _stream(stream)))
    return out


def rms_norm(x, gamma, eps: float = 1e-5, out=None, tuning=None, stream=None):
    import torch

    assert x.is_cuda and x.is_contiguous()
    out = torch.empty_like(x) if out is None else out
    hidden = x.shape[-1]
    rows = x.numel() // hidden if hidden else 0
    check(lib.mhlo_cuda_rms_norm(torch_dtype_code(x.dtype), _ptr(x), _ptr(gamma), _ptr(out), rows, hidden, eps,
                                 _tuning(tuning), _stream(stream)))
    return out


def add_layer_norm(x, residual, gamma, beta, eps: float = 1e-5, tuning=None, stream=None):
    """(x + residual, LayerNorm(x + residual)) in one pass (see ``mhlo_cuda_add_layer_norm``)."""
    import torch

    assert x.is_cuda and x.is_contiguous() and residual.is_contiguous()
    total, out = torch.empty_like(x), torch.empty_like(x)
    hidden = x.shape[-1]
    rows = x.numel() // hidden if hidden else 0
    if residual.shape != x.shape:  # a block of rows repeated down x (``mhlo_cuda_add_layer_norm_rows``)
        check(lib.mhlo_cuda_add_layer_norm_rows(torch_dtype_code(x.dtype), _ptr(x), _ptr(residual), residual.numel() // hidden, _ptr(gamma),
                                                _ptr(beta), _ptr(total), _ptr(out), rows, hidden, eps, _tuning(tuning), _stream(stream)))
        return total, out
    check(lib.mhlo_cuda_add_layer_norm(torch_dtype_code(x.dtype), _ptr(x), _ptr(residual), _ptr(gamma), _ptr(beta), _ptr(total), _ptr(out),
                                       rows, hidden, eps, _tuning(tuning), _stream(stream)))
    return total, out


def add_rms_norm(x, residual, gamma, eps: float = 1e-5, tuning=None, stream=None):
    import torch

    assert x.is_cuda and x.is_contiguous() and residual.is_contiguous()
    total, out = torch.empty_like(x), torch.empty_like(x)
    hidden = x.shape[-1]
    rows = x.numel() // hidden if hidden else 0
    if residual.shape != x.shape:
        check(lib.mhlo_cuda_add_rms_norm_rows(torch_dtype_code(x.dtype), _ptr(x), _ptr(residual), residual.numel() // hidden, _ptr(gamma),
                                              _ptr(total), _ptr(out), rows, hidden, eps, _tuning(tuning), _stream(stream)))
        return total, out
    check(lib.mhlo_cuda_add_rms_norm(torch_dtype_code(x.dtype), _ptr(x), _ptr(residual), _ptr(gamma), _ptr(total), _ptr(out), rows, hidden,
                                     eps, _tuning(tuning), _stream(stream)))
    return total, out


def device_error() -> int:
    """Synchronises, and returns and clears the first error word that a kernel left (0: none did): a bounded wait of a tensor-core kernel
    expired, or (201 and above) a key/value cache kernel met a page, length, start or position that cannot be."""
    code = C.c_int32(0)
    lib.mhlo_cuda_device_error(C.byref(code))
    return code.value


EPILOGUES = {"none": 0, "relu": 1, "gelu_tanh": 2, "gelu_erf": 3, "silu": 4, "tanh": 5, "sigmoid": 6}


def _i64s(vals):
    return (C.c_int64 * len(vals))(*[int(v) for v in vals])


class Binding(C.Structure):
    _fields_ = [("source", C.c_int32), ("index", C.c_int32), ("offset", C.c_int64)]


class PlanOp(C.Structure):
    _fields_ = [("kernel", C.c_int32), ("dtype", C.c_int32), ("out_dtype", C.c_int32), ("args", Binding * 6), ("dims", C.c_int64 * 6),
                ("strides", C.c_int64 * 16), ("scalars", C.c_float * 2), ("flags", C.c_int32 * 2), ("tuning", C.c_int32 * 4)]


SRC_NONE, SRC_INPUT, SRC_OUTPUT, SRC_UNIFIED, SRC_CONSTANT = range(5)


def plan_op(kernel_name, dtype, args, dims, strides=(), scalars=(), flags=(), tuning=(), out_dtype=None) -> PlanOp:
    """One op of a dispatch plan. args: (source, index, offset) triples in the kernel's argument order."""
    k = C.c_int32()
    check(lib.mhlo_cuda_kernel_lookup(kernel_name.encode(), dtype, C.byref(k)))
    op = PlanOp()
    op.kernel, op.dtype, op.out_dtype = k.value, dtype, dtype if out_dtype is None else out_dtype
    for i, a in enumerate(args):
        op.args[i] = Binding(*a)
    for name, vals in (("dims", dims), ("strides", strides), ("scalars", scalars), ("flags", flags), ("tuning", tuning)):
        arr = getattr(op, name)
        for i, v in enumerate(vals):
            arr[i] = v
    return op


class Plan:
    """mhlo_cuda_plan_*: a list of kernel dispatches with their buffer bindings, an arena and a constant pool."""

    def __init__(self, ops, n_inputs, n_outputs, arena_bytes=0, constants: bytes = b""):
        arr = (PlanOp * max(len(ops), 1))(*ops)
        h = C.c_void_p()
        check(lib.mhlo_cuda_plan_create(arr, len(ops), n_inputs, n_outputs, arena_bytes, constants if constants else None, len(constants), C.byref(h)))
        self._h = h.value

    def __del__(self):
        if getattr(self, "_h", None) and lib is not None:
            lib.mhlo_cuda_plan_destroy(self._h)
            self._h = None

    def _lists(self, inputs, outputs):
        return (C.c_void_p * max(len(inputs), 1))(*[_ptr(t) for t in inputs]), (C.c_void_p * max(len(outputs), 1))(*[_ptr(t) for t in outputs])

    def execute(self, inputs, outputs, stream=None):
        ins, outs = self._lists(inputs, outputs)
        check(lib.mhlo_cuda_plan_execute(self._h, ins, len(inputs), outs, len(outputs), _stream(stream)))

    def measure(self, inputs, outputs, warmup=5, iterations=20) -> float:
        ins, outs = self._lists(inputs, outputs)
        ms = C.c_float()
        check(lib.mhlo_cuda_tuner_measure(self._h, ins, len(inputs), outs, len(outputs), warmup, iterations, C.byref(ms)))
        return ms.value


class GemmTuning(C.Structure):
    _fields_ = [("tile_n", C.c_int32), ("stages", C.c_int32), ("cta_group", C.c_int32), ("split_k", C.c_int32)]


def gemm(a, b, bias=None, epilogue: str = "none", out_dtype=None, trans_a: bool = False, trans_b: bool = False,
         out=None, stream=None, tuning=None, residual=None):
    """C[..., M, N] = act(A . B + bias) through ``mhlo_cuda_gemm`` (+ residual, without activation: ``mhlo_cuda_gemm_residual``).

    a: [batch..., M, K] (or [batch..., K, M] with trans_a), b: [batch..., K, N] (or [batch..., N, K] with trans_b);
    up to two leading batch dimensions, both operands dense CUDA tensors of the same dtype.
    """
    import torch

    assert a.is_cuda and b.is_cuda and a.is_contiguous() and b.is_contiguous() and a.dtype == b.dtype
    batch = list(a.shape[:-2])
    assert len(batch) <= 2 and list(b.shape[:-2]) == batch
    b0, b1 = ([1, 1] + batch)[-2:]
    m, k = (a.shape[-1], a.shape[-2]) if trans_a else (a.shape[-2], a.shape[-1])
    n = b.shape[-2] if trans_b else b.shape[-1]
    a_mat, b_mat = a.shape[-2] * a.shape[-1], b.shape[-2] * b.shape[-1]
    a_str = [b1 * a_mat, a_mat] + ([1, m] if trans_a else [k, 1])
    b_str = [b1 * b_mat, b_mat] + ([1, k] if trans_b else [n, 1])
    out_dtype = a.dtype if out_dtype is None else out_dtype
    if out is None:
        out = torch.empty(batch + [m, n], dtype=out_dtype, device=a.device)
    if residual is not None:  # C = A . B + bias + residual, one rounding: mhlo_cuda_gemm_residual
        assert epilogue == "none" and residual.is_contiguous() and tuple(residual.shape) == tuple(out.shape) and residual.dtype == out.dtype
        t = GemmTuning(*tuning, 0) if tuning is not None else None
        check(lib.mhlo_cuda_gemm_residual(torch_dtype_code(a.dtype), torch_dtype_code(out_dtype), _ptr(a), _i64s(a_str), _ptr(b), _i64s(b_str),
                                          _ptr(out), b0, b1, m, n, k, _ptr(bias), _ptr(residual), None if t is None else C.addressof(t),
                                          _stream(stream)))
        return out
    if tuning is not None:  # (tile_n, stages, cta_group): mhlo_cuda_gemm_tuned
        t = GemmTuning(*tuning, 0)
        check(lib.mhlo_cuda_gemm_tuned(torch_dtype_code(a.dtype), torch_dtype_code(out_dtype), _ptr(a), _i64s(a_str), _ptr(b), _i64s(b_str),
                                       _ptr(out), b0, b1, m, n, k, _ptr(bias), EPILOGUES[epilogue], C.addressof(t), _stream(stream)))
        return out
    check(lib.mhlo_cuda_gemm(torch_dtype_code(a.dtype), torch_dtype_code(out_dtype), _ptr(a), _i64s(a_str), _ptr(b),
                             _i64s(b_str), _ptr(out), b0, b1, m, n, k, _ptr(bias), EPILOGUES[epilogue], _stream(stream)))
    return out


class AttentionTuning(C.Structure):
    _fields_ = [("tile_order", C.c_int32), ("reserved", C.c_int32 * 3)]


def attention(q, k, v, scale: float, causal: bool = False, mask=None, layout: str = "BHSD", out=None, stream=None, tile_order=None):
    """Fused attention through ``mhlo_cuda_attention``. q/k/v are dense [B,H,S,D] (layout "BHSD") or [B,S,H,D] ("BSHD")."""
    import torch

    assert q.is_cuda and q.is_contiguous() and k.is_contiguous() and v.is_contiguous()
    if layout == "BHSD":
        B, H, Sq, D = q.shape
        Sk = k.shape[2]
        strides = lambda S: [H * S * D, S * D, D]
    else:
        B, Sq, H, D = q.shape
        Sk = k.shape[1]
        strides = lambda S: [S * H * D, D, H * D]
    out = torch.empty_like(q) if out is None else out
    if tile_order is not None:  # mhlo_cuda_attention_tuned
        t = AttentionTuning(tile_order)
        check(lib.mhlo_cuda_attention_tuned(torch_dtype_code(q.dtype), _ptr(q), _i64s(strides(Sq)), _ptr(k), _i64s(strides(Sk)), _ptr(v),
                                            _i64s(strides(Sk)), _ptr(mask), _ptr(out), _i64s(strides(Sq)), B, H, Sq, Sk, D, scale,
                                            1 if causal else 0, C.addressof(t), _stream(stream)))
        return out
    check(lib.mhlo_cuda_attention(torch_dtype_code(q.dtype), _ptr(q), _i64s(strides(Sq)), _ptr(k), _i64s(strides(Sk)), _ptr(v),
                                  _i64s(strides(Sk)), _ptr(mask), _ptr(out), _i64s(strides(Sq)), B, H, Sq, Sk, D, scale,
                                  1 if causal else 0, _stream(stream)))
    return out


def softmax(x, axis: int = -1, out=None, tuning=None, stream=None):
    import math

    import torch

    assert x.is_cuda and x.is_contiguous()
    out = torch.empty_like(x) if out is None else out
    axis = axis % x.dim()
    outer = math.prod(x.shape[:axis])
    inner = math.prod(x.shape[axis + 1:])
    check(lib.mhlo_cuda_softmax(torch_dtype_code(x.dtype), _ptr(x), _ptr(out), outer, x.shape[axis], inner,
                                _tuning(tuning), _stream(stream)))
    return out


# ---- a paged cache of keys and values in 8 bits, and the attention over it ------------------------------------------------


def _run_on(device, stream, call):
    """call(stream handle) with ``device`` current and ``stream`` (a raw handle, or None: the current one of that device) as the stream
    that owns what is allocated inside. A decoding step makes several of these calls a layer: the ordinary case, everything on the
    current device and stream, enters no context."""
    import torch

    index = device.index
    if torch.cuda.current_device() == index:
        current = torch._C._cuda_getCurrentRawStream(index)
        if stream is None or stream == current:
            return call(current)
        with torch.cuda.stream(torch.cuda.ExternalStream(int(stream), device=device)):
            return call(int(stream))
    with torch.cuda.device(device):
        return _run_on(device, stream, call)


def _dense_like(t):
    import torch

    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _same_device(first, *others):
    device = first.device
    assert device.type == "cuda"
    for t in others:
        assert t is None or t.device == device, f"{t.device} and {device} in one call"


class KvCache:
    """The tensors of a ``mhlo_cuda_kv_cache``: int8 codes ``k``, ``v`` [pages, heads, page_tokens, head_dim] and float32 scales
    ``k_scale``, ``v_scale`` [pages, heads]. Its owner hands pages to sequences (``page_table``) as they grow."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch

        _same_device(k, v, k_scale, v_scale)
        assert k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype == torch.int8 and k.is_contiguous() and v.is_contiguous()
        assert k_scale.shape == v_scale.shape == k.shape[:2] and k_scale.dtype == v_scale.dtype == torch.float32
        assert k_scale.is_contiguous() and v_scale.is_contiguous()
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._args = KvCacheArgs(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.shape)
        self.pointer = C.byref(self._args)
        self.head_shape = (k.shape[1], k.shape[3])

    @classmethod
    def empty(cls, pages: int, heads: int, head_dim: int, page_tokens: int = 64, device="cuda") -> "KvCache":
        import torch

        codes = [torch.zeros(pages, heads, page_tokens, head_dim, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.zeros(pages, heads, dtype=torch.float32, device=device) for _ in range(2)]
        return cls(*codes, *scales)


def _kv_batch(page_table, lengths, token_starts, tokens) -> KvBatchArgs:
    import torch

    (seqs, pages), (pitch, step) = page_table.shape, page_table.stride()
    assert lengths.shape == (seqs,) and page_table.dtype == lengths.dtype == torch.int32 and lengths.is_contiguous()
    assert (seqs <= 1 or pages == 0 or pitch >= pages) and (pages <= 1 or step == 1)
    if token_starts is not None:
        assert token_starts.dtype == torch.int32 and token_starts.is_contiguous() and token_starts.shape == (seqs + 1,)
    return KvBatchArgs(page_table.data_ptr(), lengths.data_ptr(), _ptr(token_starts), seqs, pages, max(pitch, pages), tokens)


@functools.lru_cache(maxsize=1024)
def _strides(*values):
    return _i64s(values)


def _rows(x):
    """[tokens, heads, head_dim] with a contiguous last dimension: its {token, head} strides."""
    token, head, step = x.stride()
    assert step == 1 or x.shape[2] <= 1, (tuple(x.shape), x.stride())
    return _strides(token, head)


def rope_table(positions: int, rotary_dim: int, base: float = 10000.0, device="cuda"):
    """Rotation table of :func:`kv_cache_append`: float32 [positions, rotary_dim], cosines then sines of position * base^(-2i / rotary_dim),
    computed in 64 bits (at far positions a 32-bit angle has no correct digit behind the point)."""
    import torch

    angle = torch.arange(positions, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device)


def kv_cache_append(cache: KvCache, k, v, page_table, lengths, token_starts=None, rope=None, interleaved: bool = False, q=None, q_out=None, stream=None):
    """Puts the newest tokens' k, v [tokens, heads, head_dim] into the cache, keys rotated by ``rope`` (see :func:`rope_table`), and
    returns q [tokens, q_heads, head_dim] rotated beside them (None without q; rows of no sequence are not written). ``lengths``
    counts the new tokens already. See ``mhlo_cuda_kv_cache_append``."""
    import torch

    _same_device(cache.k, k, v, page_table, lengths, token_starts, rope, q, q_out)
    shape, dtype = k.shape, k.dtype
    tokens, heads, dim = shape
    assert (heads, dim) == cache.head_shape and v.dtype == dtype and v.shape == shape
    positions, rotary = 0, 0
    if rope is not None:
        positions, rotary = rope.shape
        assert rope.dtype == torch.float32 and rope.is_contiguous()
    batch = _kv_batch(page_table, lengths, token_starts, tokens)
    q_heads, q_strides = 0, None
    if q is not None:
        q_tokens, q_heads, q_dim = q.shape
        assert q.dtype == dtype and q_tokens == tokens and q_dim == dim
        q_strides = _rows(q)
    assert q_out is None or (q is not None and q_out.shape == q.shape and q_out.dtype == dtype)

    def call(s):
        out = _dense_like(q) if q is not None and q_out is None else q_out
        check(lib.mhlo_cuda_kv_cache_append(torch_dtype_code(dtype), cache.pointer, C.byref(batch), k.data_ptr(), _rows(k), v.data_ptr(), _rows(v),
                                            _ptr(q), q_strides, _ptr(out), None if q is None else _rows(out), q_heads, _ptr(rope), positions, rotary,
                                            1 if interleaved else 0, s))
        return out

    return _run_on(k.device, stream, call)


def kv_cache_read(cache: KvCache, page_table, lengths, max_tokens: int, dtype=None, k_out=None, v_out=None, stream=None):
    """(k, v), each [seqs, max_tokens, heads, head_dim] of ``dtype`` (float32): the values in the cache, zero behind a sequence's
    length. ``k_out`` and ``v_out`` have one set of strides; one that is not given gets the other's. See ``mhlo_cuda_kv_cache_read``."""
    import torch

    _same_device(cache.k, page_table, lengths, k_out, v_out)
    seqs = lengths.shape[0]
    batch = _kv_batch(page_table, lengths, None, seqs)
    shape = (seqs, max_tokens, *cache.head_shape)
    given = k_out if k_out is not None else v_out
    dtype = given.dtype if given is not None else dtype or torch.float32

    def fresh():
        return torch.empty(shape, dtype=dtype, device=lengths.device) if given is None else torch.empty_strided(shape, given.stride(), dtype=dtype, device=lengths.device)

    def call(s):
        k = fresh() if k_out is None else k_out
        v = fresh() if v_out is None else v_out
        seq, token, head, step = k.stride()
        assert k.shape == v.shape == shape and v.dtype == dtype and v.stride() == k.stride() and step == 1
        check(lib.mhlo_cuda_kv_cache_read(torch_dtype_code(dtype), cache.pointer, C.byref(batch), max_tokens, k.data_ptr(), v.data_ptr(),
                                          _strides(seq, token, head), s))
        return k, v

    return _run_on(lengths.device, stream, call)


def cached_attention(q, cache: KvCache, page_table, lengths, scale: float, token_starts=None, out=None, lse=None, stream=None):
    """Attention of the newest tokens' q [tokens, q_heads, head_dim] over the cache, which holds them (and ``lengths`` counts them).
    ``lse`` (float32 [tokens, q_heads]) receives the logarithms of the sums of exponentials. See ``mhlo_cuda_cached_attention``."""
    import torch

    _same_device(q, cache.k, page_table, lengths, token_starts, out, lse)
    shape, dtype = q.shape, q.dtype
    tokens, q_heads, dim = shape
    assert dim == cache.head_shape[1]
    assert out is None or (out.shape == shape and out.dtype == dtype)
    assert lse is None or (lse.shape == shape[:2] and lse.dtype == torch.float32 and lse.is_contiguous())
    batch = _kv_batch(page_table, lengths, token_starts, tokens)

    def call(s):
        o = _dense_like(q) if out is None else out
        need = lib.mhlo_cuda_cached_attention_scratch_bytes(cache.pointer, C.byref(batch), q_heads)
        scratch = lengths.new_empty(need >> 2) if need > 0 else None
        check(lib.mhlo_cuda_cached_attention(torch_dtype_code(dtype), q.data_ptr(), _rows(q), cache.pointer, C.byref(batch), q_heads, scale, o.data_ptr(),
                                             _rows(o), _ptr(lse), _ptr(scratch), need, s))
        return o

    return _run_on(q.device, stream, call)


# ---- log probabilities ------------------------------------------------------------------------------------------------

TokenLogprobs = collections.namedtuple("TokenLogprobs", "logprobs entropy lse top_logprobs top_ids")


def _logit_rows(x):
    """[..., vocab] as rows of one stride: (rows, stride)."""
    vocab = x.shape[-1]
    assert x.stride(-1) == 1 or vocab == 1
    lead = [(n, step) for n, step in zip(x.shape[:-1], x.stride()[:-1]) if n != 1]
    for (_, outer), (n, inner) in zip(lead, lead[1:]):
        assert outer == n * inner, "the rows of the logits need one stride"
    if not lead or not x.numel():
        return x.numel() // vocab if vocab else 0, vocab
    assert lead[-1][1] >= vocab, "the rows of the logits overlap"
    return x.numel() // vocab, lead[-1][1]


def token_logprobs(logits, targets=None, top_k: int = 0, scale: float = 1.0, entropy: bool = True, stream=None) -> TokenLogprobs:
    """Log probabilities of ``targets`` [...] (int32 or int64; negative: none) under softmax(scale * logits [..., vocab]), the entropy,
    the logarithm of the sum of exponentials and the ``top_k`` likeliest ids with their log probabilities. See ``mhlo_cuda_token_logprobs``."""
    import torch

    _same_device(logits, targets)
    rows, pitch = _logit_rows(logits)
    lead = logits.shape[:-1]
    assert targets is None or (targets.shape == lead and targets.is_contiguous())
    assert top_k >= 0

    def call(s):
        # one allocation for the numbers of a row, one for its alternatives
        logprobs, ent, lse = torch.empty((3, *lead), dtype=torch.float32, device=logits.device).unbind(0)
        top = ids = None
        if top_k:
            top = torch.empty((*lead, top_k), dtype=torch.float32, device=logits.device)
            ids = torch.empty((*lead, top_k), dtype=torch.int32, device=logits.device)
        r = TokenLogprobs(None if targets is None else logprobs, ent if entropy else None, lse, top, ids)
        check(lib.mhlo_cuda_token_logprobs(torch_dtype_code(logits.dtype), logits.data_ptr(), pitch, rows, logits.shape[-1], scale, _ptr(targets),
                                           I64 if targets is None else torch_dtype_code(targets.dtype), _ptr(r.logprobs), _ptr(r.entropy), lse.data_ptr(),
                                           top_k, _ptr(top), _ptr(ids), s))
        return r

    return _run_on(logits.device, stream, call)


def token_logprobs_grad(logits, targets, lse, entropy=None, grad_logprobs=None, grad_entropy=None, top_ids=None, grad_top=None, scale: float = 1.0,
                        out=None, stream=None):
    """Gradient of :func:`token_logprobs` with respect to the logits, from the gradients of its results; ``out`` may be ``logits``. See
    ``mhlo_cuda_token_logprobs_grad``."""
    import torch

    _same_device(logits, targets, lse, entropy, grad_logprobs, grad_entropy, top_ids, grad_top, out)
    rows, pitch = _logit_rows(logits)
    lead = logits.shape[:-1]
    assert targets is None or (targets.shape == lead and targets.is_contiguous())
    for t in (lse, entropy, grad_logprobs, grad_entropy):
        assert t is None or (t.shape == lead and t.dtype == torch.float32 and t.is_contiguous())
    assert grad_top is None or (top_ids is not None and grad_top.shape == top_ids.shape and top_ids.shape[:-1] == lead and grad_top.dtype == torch.float32
                                and top_ids.dtype == torch.int32 and grad_top.is_contiguous() and top_ids.is_contiguous())
    assert out is None or (out.shape == logits.shape and out.dtype == logits.dtype)

    def call(s):
        dx = _dense_like(logits) if out is None else out
        check(lib.mhlo_cuda_token_logprobs_grad(torch_dtype_code(logits.dtype), logits.data_ptr(), pitch, rows, logits.shape[-1], scale, _ptr(targets),
                                                I64 if targets is None else torch_dtype_code(targets.dtype), lse.data_ptr(), _ptr(entropy), _ptr(grad_logprobs),
                                                _ptr(grad_entropy), 0 if grad_top is None else grad_top.shape[-1], _ptr(top_ids), _ptr(grad_top),
                                                dx.data_ptr(), _logit_rows(dx)[1], s))
        return dx

    return _run_on(logits.device, stream, call)
