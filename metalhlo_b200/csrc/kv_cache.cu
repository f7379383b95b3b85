// The paged key/value cache in 8 bits: appending tokens (with the rotation of keys and queries by their positions) and reading
// blocks back as dense values.
//
// A block (page of P tokens, head) has one scale s and int8 codes c, value = s c. Appending: m = max |x| over the new tokens of the
// block, s' = max(s, m (1 / 127)) (s = 0 where slot 0 is among them), earlier codes become round(c (s / s')) when s' > s, new codes
// round(x (1 / s')). One CTA owns a block, so the maximum, the rewriting and the new codes need no atomics and the result does
// not depend on the order in which CTAs run.
//
// Rotation: pair (a, b) of a position with cosine c and sine s becomes (a c - b s, b c + a s). Products and sums are rounded one by
// one (no contraction to FMA), so that codes next to the border of two steps do not depend on how a compiler fuses them.
#include <algorithm>

#include "kv_cache.cuh"

namespace mhlo {
namespace {

template <typename T>
struct AppendParams {
    KvArgs kv;
    const T* k;
    const T* v;
    const T* q;
    T* q_out;
    int64_t ks[2], vs[2], qs[2], os[2];
    const float* rope;
    int64_t rope_positions;
    int32_t rotary_dim, interleaved, q_heads;
    int64_t blocks;  // CTAs that append; the CTAs behind them rotate queries
};

// One element of a rotated row. x: the row.
template <typename T>
__device__ __forceinline__ float rotated(const T* x, int d, const float* rope, int rotary_dim, int interleaved) {
    const float own = VecTraits<T>::to_float(x[d]);
    if (rope == nullptr || d >= rotary_dim) return own;
    const int half = rotary_dim >> 1;
    const int i = interleaved ? d >> 1 : d < half ? d : d - half;
    const bool second = interleaved ? d & 1 : d >= half;
    const float other = VecTraits<T>::to_float(x[interleaved ? d ^ 1 : second ? d - half : d + half]);
    const float c = rope[i], s = rope[half + i];
    return second ? __fadd_rn(__fmul_rn(own, c), __fmul_rn(other, s)) : __fsub_rn(__fmul_rn(own, c), __fmul_rn(other, s));
}

template <typename T>
__device__ __forceinline__ const float* rope_row(const AppendParams<T>& p, int32_t position) {
    if (p.rope == nullptr) return nullptr;
    if (position >= p.rope_positions) {
        kv_report(MHLO_CUDA_KV_ERROR_POSITION);
        position = static_cast<int32_t>(p.rope_positions - 1);
    }
    return p.rope + static_cast<int64_t>(position) * p.rotary_dim;
}

constexpr int kAppendThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendParams<T> p) {
    const KvArgs& a = p.kv;
    const int page_tokens = 1 << a.page_shift, dim = a.head_dim;
    if (blockIdx.x >= p.blocks) {  // a row of queries
        const int32_t row = static_cast<int32_t>(blockIdx.x - p.blocks);
        int32_t b = row;
        if (a.starts != nullptr) b = kv_search(a.seqs, row, [&](int32_t i) { return static_cast<int64_t>(a.starts[i]); });
        const KvSequence s = kv_sequence(a, b);
        if (s.length == 0 || row < s.first || row >= s.first + s.count) return;
        const float* rope = rope_row(p, s.position(row));
        for (int i = threadIdx.x; i < p.q_heads * (dim / 16); i += kAppendThreads) {
            const int h = i / (dim / 16), unit = i % (dim / 16), half = p.rotary_dim >> 1;
            const T* x = p.q + row * p.qs[0] + h * p.qs[1];
            T* y = p.q_out + row * p.os[0] + h * p.os[1];
            float out[16];
            int at[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {  // both elements of each pair in one thread: y may be x
                at[e] = unit * 16 + e;
                if (!p.interleaved && unit * 16 < p.rotary_dim) at[e] = unit * 8 + (e & 7) + (e < 8 ? 0 : half);
                out[e] = rotated(x, at[e], rope, p.rotary_dim, p.interleaved);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) y[at[e]] = VecTraits<T>::from_float(out[e]);
        }
        return;
    }
    // block `slot` of the sequences' touched blocks. A sequence has n / P + 2 slots at least, as many as n tokens can touch:
    // slot of its first block = floor(first row / P) + 2 b.
    const int32_t head = static_cast<int32_t>(blockIdx.x % a.heads);
    const int64_t slot = blockIdx.x / a.heads;
    int32_t b, nth = 0;
    if (a.starts == nullptr) {
        b = static_cast<int32_t>(slot);
    } else {
        auto first = [&](int32_t i) { return static_cast<int64_t>(a.starts[i] >> a.page_shift) + 2 * i; };
        b = kv_search(a.seqs, slot, first);
        nth = static_cast<int32_t>(slot - first(b));
    }
    const KvSequence s = kv_sequence(a, b);
    if (s.length == 0 || s.count == 0 || nth < 0) return;
    const int32_t page_index = ((s.length - s.count) >> a.page_shift) + nth;
    const int32_t from = max(s.length - s.count, page_index << a.page_shift), to = min(s.length, (page_index + 1) << a.page_shift);
    if (from >= to) return;
    const int32_t page = kv_page(a, b, page_index);
    if (page < 0) return;
    const int32_t slot0 = from & (page_tokens - 1), n = to - from, row0 = from - (s.length - s.count) + s.first;
    const int64_t block = static_cast<int64_t>(page) * a.heads + head;
    __shared__ uint32_t largest[2][kAppendThreads / 32];
    for (int which = 0; which < 2; ++which) {
        const T* x = which == 0 ? p.k + row0 * p.ks[0] + head * p.ks[1] : p.v + row0 * p.vs[0] + head * p.vs[1];
        const int64_t pitch = which == 0 ? p.ks[0] : p.vs[0];
        int8_t* codes = (which == 0 ? a.k_codes : a.v_codes) + block * page_tokens * dim;
        float* scales = (which == 0 ? a.k_scales : a.v_scales) + block;
        uint32_t m = 0;  // magnitudes as bits: ordered like the numbers, infinity and NaN above all
        auto value = [&](int i) {
            const int t = i / dim, d = i % dim;
            if (which == 1) return VecTraits<T>::to_float(x[t * pitch + d]);
            return rotated(x + t * pitch, d, rope_row(p, from + t), p.rotary_dim, p.interleaved);
        };
        for (int i = threadIdx.x; i < n * dim; i += kAppendThreads) m = max(m, __float_as_uint(value(i)) & 0x7fffffffu);
        m = __reduce_max_sync(0xffffffffu, m);
        if ((threadIdx.x & 31) == 0) largest[which][threadIdx.x >> 5] = m;
        const float before = slot0 == 0 ? 0.f : *scales;
        __syncthreads();
        for (int w = 0; w < kAppendThreads / 32; ++w) m = max(m, largest[which][w]);
        float scale = __fmul_rn(__uint_as_float(m), 1.f / 127.f);
        if (scale < 1.17549435e-38f) scale = 0.f;
        scale = before > scale || before != before ? before : scale;
        if (m >= 0x7f800000u) scale = __uint_as_float(0x7fffffffu);
        if (threadIdx.x == 0) *scales = scale;
        if (scale > before) {
            const float ratio = __fdiv_rn(before, scale);
            for (int i = threadIdx.x; i < slot0 * dim; i += kAppendThreads) codes[i] = static_cast<int8_t>(__float2int_rn(__fmul_rn(static_cast<float>(codes[i]), ratio)));
        }
        const float step = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;  // NaN scales: codes 0
        for (int i = threadIdx.x; i < n * dim; i += kAppendThreads) {
            const int c = step > 0.f ? __float2int_rn(__fmul_rn(value(i), step)) : 0;
            codes[slot0 * dim + i] = static_cast<int8_t>(min(127, max(-127, c)));
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(128) read_kernel(const __grid_constant__ KvArgs a, T* k_out, T* v_out, int64_t s_seq, int64_t s_token, int64_t s_head,
                                                   int64_t max_tokens, int64_t pieces) {
    const int page_tokens = 1 << a.page_shift, dim = a.head_dim;
    const int32_t head = static_cast<int32_t>(blockIdx.x % a.heads);
    const int64_t unit = blockIdx.x / a.heads;
    const int32_t b = static_cast<int32_t>(unit / pieces), i0 = static_cast<int32_t>(unit % pieces);
    int32_t length = a.lengths[b];
    if (length < 0 || length > static_cast<int64_t>(a.pages_per_seq) << a.page_shift) {
        kv_report(MHLO_CUDA_KV_ERROR_LENGTH);
        length = 0;
    }
    const int64_t first = static_cast<int64_t>(i0) << a.page_shift;
    const int32_t page = first < length ? kv_page(a, b, i0) : -1;
    const int64_t block = static_cast<int64_t>(page) * a.heads + head;
    for (int which = 0; which < 2; ++which) {
        T* out = which == 0 ? k_out : v_out;
        if (out == nullptr) continue;
        out += b * s_seq + head * s_head;
        const float scale = page < 0 ? 0.f : (which == 0 ? a.k_scales : a.v_scales)[block];
        const int8_t* codes = (which == 0 ? a.k_codes : a.v_codes) + block * page_tokens * dim;
        for (int i = threadIdx.x; i < page_tokens * dim; i += 128) {
            const int64_t token = first + i / dim;
            if (token >= max_tokens) break;
            const float x = page >= 0 && token < length ? __fmul_rn(static_cast<float>(codes[i]), scale) : 0.f;
            out[token * s_token + i % dim] = VecTraits<T>::from_float(x);
        }
    }
}

template <typename T>
int append(const KvArgs& kv, const void* k, const int64_t* ks, const void* v, const int64_t* vs, const void* q, const int64_t* qs, void* q_out,
           const int64_t* os, int64_t q_heads, const float* rope, int64_t rope_positions, int64_t rotary_dim, int32_t interleaved, cudaStream_t stream) {
    AppendParams<T> p;
    p.kv = kv;
    p.k = static_cast<const T*>(k);
    p.v = static_cast<const T*>(v);
    p.q = static_cast<const T*>(q);
    p.q_out = static_cast<T*>(q_out);
    for (int i = 0; i < 2; ++i) {
        p.ks[i] = ks[i];
        p.vs[i] = vs[i];
        p.qs[i] = q ? qs[i] : 0;
        p.os[i] = q ? os[i] : 0;
    }
    p.rope = rope;
    p.rope_positions = rope_positions;
    p.rotary_dim = static_cast<int32_t>(rope ? rotary_dim : 0);
    p.interleaved = interleaved;
    p.q_heads = static_cast<int32_t>(q_heads);
    p.blocks = (kv.starts ? (static_cast<int64_t>(kv.tokens) >> kv.page_shift) + 2 * static_cast<int64_t>(kv.seqs) : kv.seqs) * kv.heads;
    const int64_t grid = p.blocks + (q ? kv.tokens : 0);
    if (grid > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "kv_cache_append: too many blocks");
    append_kernel<T><<<static_cast<unsigned>(grid), kAppendThreads, 0, stream>>>(p);
    MHLO_CUDA_CHECK_LAUNCH("kv_cache_append");
    return MHLO_CUDA_OK;
}

template <typename T>
int read(const KvArgs& kv, int64_t max_tokens, void* k_out, void* v_out, const int64_t* strides, cudaStream_t stream) {
    const int64_t pieces = (max_tokens + (int64_t{1} << kv.page_shift) - 1) >> kv.page_shift, grid = pieces * kv.heads * kv.seqs;
    if (grid > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "kv_cache_read: too many blocks");
    read_kernel<T><<<static_cast<unsigned>(grid), 128, 0, stream>>>(kv, static_cast<T*>(k_out), static_cast<T*>(v_out), strides[0], strides[1], strides[2],
                                                                    max_tokens, pieces);
    MHLO_CUDA_CHECK_LAUNCH("kv_cache_read");
    return MHLO_CUDA_OK;
}

}  // namespace

int kv_cache_device_error() { return take_kv_error(); }

int kv_args(const char* what, const mhlo_cuda_kv_cache* cache, const mhlo_cuda_kv_batch* batch, KvArgs* out) {
    if (!cache || !batch) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null cache or batch", what);
    if (!cache->k_codes || !cache->v_codes || !cache->k_scales || !cache->v_scales) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null pointer in the cache", what);
    if (!aligned16(cache->k_codes) || !aligned16(cache->v_codes)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: codes are not 16-byte aligned", what);
    if (cache->pages < 1 || cache->pages > 0x7fffffff || cache->heads < 1 || cache->heads > 65535)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld pages of %lld heads", what, static_cast<long long>(cache->pages), static_cast<long long>(cache->heads));
    if (cache->page_tokens != 16 && cache->page_tokens != 32 && cache->page_tokens != 64 && cache->page_tokens != 128)
        return fail(MHLO_CUDA_UNSUPPORTED, "%s: %lld tokens in a page (16, 32, 64 or 128)", what, static_cast<long long>(cache->page_tokens));
    if (cache->head_dim < 16 || cache->head_dim > 256 || cache->head_dim % 16 != 0)
        return fail(MHLO_CUDA_UNSUPPORTED, "%s: head dimension %lld (a multiple of 16 up to 256)", what, static_cast<long long>(cache->head_dim));
    if (batch->seqs < 0 || batch->seqs > (1 << 24) || batch->tokens < 0 || batch->tokens > (1 << 30) || batch->pages_per_seq < 0 ||
        batch->pages_per_seq > (int64_t{1} << 30) / cache->page_tokens || batch->table_stride < batch->pages_per_seq)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld sequences, %lld tokens, %lld pages a sequence, table rows %lld apart", what,
                    static_cast<long long>(batch->seqs), static_cast<long long>(batch->tokens), static_cast<long long>(batch->pages_per_seq),
                    static_cast<long long>(batch->table_stride));
    if (batch->seqs > 0 && (!batch->lengths || (batch->pages_per_seq > 0 && !batch->page_table))) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null lengths or page table", what);
    out->k_codes = cache->k_codes;
    out->v_codes = cache->v_codes;
    out->k_scales = cache->k_scales;
    out->v_scales = cache->v_scales;
    out->page_table = batch->page_table;
    out->lengths = batch->lengths;
    out->starts = batch->token_starts;
    out->table_stride = batch->table_stride;
    out->pages = static_cast<int32_t>(cache->pages);
    out->heads = static_cast<int32_t>(cache->heads);
    out->head_dim = static_cast<int32_t>(cache->head_dim);
    out->page_shift = cache->page_tokens == 16 ? 4 : cache->page_tokens == 32 ? 5 : cache->page_tokens == 64 ? 6 : 7;
    out->seqs = static_cast<int32_t>(batch->seqs);
    out->pages_per_seq = static_cast<int32_t>(batch->pages_per_seq);
    out->tokens = static_cast<int32_t>(batch->tokens);
    return MHLO_CUDA_OK;
}

int kv_row_strides(const char* what, const char* name, const int64_t* strides) {
    if (!strides) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null strides of %s", what, name);
    if (strides[0] < 0 || strides[1] < 0) return fail(MHLO_CUDA_UNSUPPORTED, "%s: negative strides of %s", what, name);
    return MHLO_CUDA_OK;
}

}  // namespace mhlo

using namespace mhlo;

extern "C" {

int mhlo_cuda_kv_cache_append(int32_t dtype, const mhlo_cuda_kv_cache* cache, const mhlo_cuda_kv_batch* batch, const void* k_dev, const int64_t k_strides[2],
                              const void* v_dev, const int64_t v_strides[2], const void* q_dev, const int64_t q_strides[2], void* q_out_dev,
                              const int64_t q_out_strides[2], int64_t q_heads, const float* rope_dev, int64_t rope_positions, int64_t rotary_dim,
                              int32_t interleaved, mhlo_cuda_stream_t stream) {
    static const char* const what = "kv_cache_append";
    if (dtype != MHLO_DT_F16 && dtype != MHLO_DT_BF16 && dtype != MHLO_DT_F32) return fail(MHLO_CUDA_UNSUPPORTED, "%s: dtype %d", what, dtype);
    if (rope_dev != nullptr) {
        if (!cache || rotary_dim < 16 || rotary_dim % 16 != 0 || rotary_dim > cache->head_dim)
            return fail(MHLO_CUDA_UNSUPPORTED, "%s: rotation of %lld elements (a multiple of 16 up to the head dimension)", what, static_cast<long long>(rotary_dim));
        if (rope_positions < 1) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: a rotation table without positions", what);
        if (!aligned16(rope_dev)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: the rotation table is not 16-byte aligned", what);
    } else if (q_dev != nullptr) {
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: queries without a rotation table", what);
    }
    KvArgs kv;
    if (int st = kv_args(what, cache, batch, &kv)) return st;
    if (batch->tokens == 0 || batch->seqs == 0) return MHLO_CUDA_OK;
    if (!batch->token_starts && batch->tokens != batch->seqs)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld tokens of %lld sequences need token_starts", what, static_cast<long long>(batch->tokens), static_cast<long long>(batch->seqs));
    if (!k_dev || !v_dev) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null keys or values", what);
    if (int st = kv_row_strides(what, "k", k_strides)) return st;
    if (int st = kv_row_strides(what, "v", v_strides)) return st;
    if (q_dev != nullptr) {
        if (!q_out_dev || q_heads < 1 || q_heads > 65535) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null result or %lld heads of the queries", what, static_cast<long long>(q_heads));
        if (int st = kv_row_strides(what, "q", q_strides)) return st;
        if (int st = kv_row_strides(what, "q_out", q_out_strides)) return st;
        if (q_dev == q_out_dev && (q_strides[0] != q_out_strides[0] || q_strides[1] != q_out_strides[1]))
            return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: queries rotated in place need one set of strides", what);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MHLO_DT_F32)
        return append<float>(kv, k_dev, k_strides, v_dev, v_strides, q_dev, q_strides, q_out_dev, q_out_strides, q_heads, rope_dev, rope_positions, rotary_dim, interleaved, st);
    if (dtype == MHLO_DT_F16)
        return append<__half>(kv, k_dev, k_strides, v_dev, v_strides, q_dev, q_strides, q_out_dev, q_out_strides, q_heads, rope_dev, rope_positions, rotary_dim, interleaved, st);
    return append<__nv_bfloat16>(kv, k_dev, k_strides, v_dev, v_strides, q_dev, q_strides, q_out_dev, q_out_strides, q_heads, rope_dev, rope_positions, rotary_dim, interleaved, st);
}

int mhlo_cuda_kv_cache_read(int32_t dtype, const mhlo_cuda_kv_cache* cache, const mhlo_cuda_kv_batch* batch, int64_t max_tokens, void* k_out_dev,
                            void* v_out_dev, const int64_t out_strides[3], mhlo_cuda_stream_t stream) {
    static const char* const what = "kv_cache_read";
    if (dtype != MHLO_DT_F16 && dtype != MHLO_DT_BF16 && dtype != MHLO_DT_F32) return fail(MHLO_CUDA_UNSUPPORTED, "%s: dtype %d", what, dtype);
    KvArgs kv;
    if (int st = kv_args(what, cache, batch, &kv)) return st;
    if (max_tokens < 0 || max_tokens > (int64_t{1} << 30)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld tokens", what, static_cast<long long>(max_tokens));
    if (batch->seqs == 0 || max_tokens == 0 || (!k_out_dev && !v_out_dev)) return MHLO_CUDA_OK;
    if (int st = kv_row_strides(what, "the result", out_strides)) return st;
    if (out_strides[2] < 0) return fail(MHLO_CUDA_UNSUPPORTED, "%s: negative strides of the result", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MHLO_DT_F32) return read<float>(kv, max_tokens, k_out_dev, v_out_dev, out_strides, st);
    if (dtype == MHLO_DT_F16) return read<__half>(kv, max_tokens, k_out_dev, v_out_dev, out_strides, st);
    return read<__nv_bfloat16>(kv, max_tokens, k_out_dev, v_out_dev, out_strides, st);
}

}  // extern "C"
