// What the kernels over the paged 8-bit key/value cache share: the sequences of a call and their checks.
#pragma once

#include "contraction.cuh"

namespace mhlo {

// mhlo_cuda_kv_cache and mhlo_cuda_kv_batch as the kernels take them.
struct KvArgs {
    int8_t* k_codes;
    int8_t* v_codes;
    float* k_scales;
    float* v_scales;
    const int32_t* page_table;
    const int32_t* lengths;
    const int32_t* starts;  // null: one row per sequence
    int64_t table_stride;
    int32_t pages, heads, head_dim;
    int32_t page_shift;  // log2(page_tokens)
    int32_t seqs, pages_per_seq, tokens;
};

// Checks what the host can see and fills *out. what: the entry point's name for messages.
int kv_args(const char* what, const mhlo_cuda_kv_cache* cache, const mhlo_cuda_kv_batch* batch, KvArgs* out);
// Element strides {token, head} of a [tokens, heads, head_dim] tensor: none negative.
int kv_row_strides(const char* what, const char* name, const int64_t* strides);

namespace {

// The error word of the including file's kernels: MHLO_CUDA_KV_ERROR_*, 0 when none.
__device__ int g_kv_error = 0;
__device__ __forceinline__ void kv_report(int code) { g_kv_error = code; }

// Reads and clears the word (-1: CUDA error).
inline int take_kv_error() {
    int v = 0, zero = 0;
    if (cudaDeviceSynchronize() != cudaSuccess) return -1;
    if (cudaMemcpyFromSymbol(&v, g_kv_error, sizeof v) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(g_kv_error, &zero, sizeof zero);
    return v;
}

// Rows first .. first + count - 1 of the call are the newest tokens of a sequence of `length` tokens.
struct KvSequence {
    int32_t first, count, length;
    __device__ __forceinline__ int32_t position(int32_t row) const { return length - count + row - first; }
};

// Sequence b of the call. count = 0: its starts are out of order; length = 0: unused, or a length that cannot be.
__device__ __forceinline__ KvSequence kv_sequence(const KvArgs& a, int32_t b) {
    KvSequence s{b, 1, a.lengths[b]};
    if (a.starts != nullptr) {
        const int32_t end = a.starts[b + 1];
        s.first = a.starts[b];
        s.count = end - s.first;
        if (s.first < 0 || end > a.tokens || end < s.first) {
            kv_report(MHLO_CUDA_KV_ERROR_STARTS);
            s.first = s.count = s.length = 0;
            return s;
        }
    }
    if (s.length < 0 || (s.length != 0 && s.length < s.count) || s.length > static_cast<int64_t>(a.pages_per_seq) << a.page_shift) {
        kv_report(MHLO_CUDA_KV_ERROR_LENGTH);
        s.length = 0;
    }
    return s;
}

// Page i of sequence b, -1 when the table's entry is no page of the cache.
__device__ __forceinline__ int32_t kv_page(const KvArgs& a, int32_t b, int32_t i) {
    const int32_t page = a.page_table[b * a.table_stride + i];
    if (page >= 0 && page < a.pages) return page;
    kv_report(MHLO_CUDA_KV_ERROR_PAGE);
    return -1;
}

// The last sequence whose first(b) <= x, for an ascending first with first(0) <= x: a warp narrows the range 32-fold a step.
template <typename First>
__device__ __forceinline__ int32_t kv_search(int32_t seqs, int64_t x, First first) {
    const int32_t lane = threadIdx.x & 31;
    int32_t lo = 0, width = seqs;  // the answer is in [lo, lo + width)
    while (width > 1) {
        const int32_t step = (width + 31) / 32;
        const int32_t b = lo + lane * step;
        const bool at = lane == 0 || (lane * step < width && first(b) <= x);
        const uint32_t reached = __ballot_sync(0xffffffffu, at);
        const int32_t last = 31 - __clz(reached);
        width = min(step, width - last * step);
        lo += last * step;
    }
    return lo;
}

}  // namespace
}  // namespace mhlo
