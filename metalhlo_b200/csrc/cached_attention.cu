// Attention of new tokens over the paged 8-bit key/value cache: o = softmax(scale q k^T) v with k = ks c, v = vs c.
//
// One CTA per (row, query head): its warps take keys in turn, a lane holds head_dim / 32 elements of q and o, and every warp keeps
// a running maximum, sum and output that are joined at the end.
#include <algorithm>

#include "kv_cache.cuh"

namespace mhlo {
namespace {

template <typename T>
struct CachedParams {
    KvArgs kv;
    const T* q;
    T* o;
    float* lse;
    int64_t qs[2], os[2];
    int32_t q_heads, group;
    float scale;
};

constexpr int kRowThreads = 128, kRowWarps = kRowThreads / 32;

template <typename T>
__global__ void __launch_bounds__(kRowThreads) cached_rows_kernel(const __grid_constant__ CachedParams<T> p) {
    const KvArgs& a = p.kv;
    const int32_t h = static_cast<int32_t>(blockIdx.x % p.q_heads), row = static_cast<int32_t>(blockIdx.x / p.q_heads);
    int32_t b = row;
    if (a.starts != nullptr) b = kv_search(a.seqs, row, [&](int32_t i) { return static_cast<int64_t>(a.starts[i]); });
    const KvSequence s = kv_sequence(a, b);
    if (row < s.first || row >= s.first + s.count) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = a.head_dim, each = dim / 32, head = h / p.group;
    const int32_t keys = s.length == 0 ? 0 : s.position(row) + 1;
    float q[8], o[8], m = -INFINITY, l = 0.f;
    for (int i = 0; i < each; ++i) {
        q[i] = VecTraits<T>::to_float(p.q[row * p.qs[0] + h * p.qs[1] + lane + 32 * i]);
        o[i] = 0.f;
    }
    for (int32_t j = warp; j < keys; j += kRowWarps) {
        const int32_t page = kv_page(a, b, j >> a.page_shift);
        if (page < 0) continue;
        const int64_t block = static_cast<int64_t>(page) * a.heads + head, at = ((block << a.page_shift) + (j & ((1 << a.page_shift) - 1))) * dim + lane;
        float z = 0.f;
        for (int i = 0; i < each; ++i) z += q[i] * static_cast<float>(a.k_codes[at + 32 * i]);
        z = warp_reduce<SumOp>(z) * a.k_scales[block] * p.scale;
        const float top = fmaxf(m, z), keep = m == top ? 1.f : expf(m - top), w = z == top ? 1.f : expf(z - top);
        m = top;
        l = l * keep + w;
        for (int i = 0; i < each; ++i) o[i] = o[i] * keep + w * a.v_scales[block] * static_cast<float>(a.v_codes[at + 32 * i]);
    }
    __shared__ float sm[kRowWarps], sl[kRowWarps], so[kRowWarps][256];
    if (lane == 0) sm[warp] = m, sl[warp] = l;
    for (int i = 0; i < each; ++i) so[warp][lane + 32 * i] = o[i];
    __syncthreads();
    float top = -INFINITY, total = 0.f;
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < kRowWarps; ++w) total += sl[w] * (sm[w] == top ? 1.f : expf(sm[w] - top));
    for (int d = threadIdx.x; d < dim; d += kRowThreads) {
        float sum = 0.f;
        for (int w = 0; w < kRowWarps; ++w) sum += so[w][d] * (sm[w] == top ? 1.f : expf(sm[w] - top));
        p.o[row * p.os[0] + h * p.os[1] + d] = VecTraits<T>::from_float(total == 0.f ? 0.f : sum / total);
    }
    if (p.lse != nullptr && threadIdx.x == 0) p.lse[static_cast<int64_t>(row) * p.q_heads + h] = total == 0.f ? -INFINITY : top + logf(total);
}

template <typename T>
int launch(const KvArgs& kv, const void* q, const int64_t* qs, int64_t q_heads, float scale, void* o, const int64_t* os, float* lse, cudaStream_t stream) {
    CachedParams<T> p;
    p.kv = kv;
    p.q = static_cast<const T*>(q);
    p.o = static_cast<T*>(o);
    p.lse = lse;
    for (int i = 0; i < 2; ++i) p.qs[i] = qs[i], p.os[i] = os[i];
    p.q_heads = static_cast<int32_t>(q_heads);
    p.group = static_cast<int32_t>(q_heads / kv.heads);
    p.scale = scale;
    if (kv.tokens * q_heads > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "cached_attention: too many rows");
    cached_rows_kernel<T><<<static_cast<unsigned>(kv.tokens * q_heads), kRowThreads, 0, stream>>>(p);
    MHLO_CUDA_CHECK_LAUNCH("cached_attention");
    return MHLO_CUDA_OK;
}

}  // namespace

int cached_attention_device_error() { return take_kv_error(); }

}  // namespace mhlo

using namespace mhlo;

extern "C" {

int64_t mhlo_cuda_cached_attention_scratch_bytes(const mhlo_cuda_kv_cache* cache, const mhlo_cuda_kv_batch* batch, int64_t q_heads) {
    if (!cache || !batch || q_heads < 1) return 0;
    return 0;
}

int mhlo_cuda_cached_attention(int32_t dtype, const void* q_dev, const int64_t q_strides[2], const mhlo_cuda_kv_cache* cache, const mhlo_cuda_kv_batch* batch,
                               int64_t q_heads, float scale, void* o_dev, const int64_t o_strides[2], float* lse_dev, void* scratch_dev, int64_t scratch_bytes,
                               mhlo_cuda_stream_t stream) {
    static const char* const what = "cached_attention";
    if (dtype != MHLO_DT_F16 && dtype != MHLO_DT_BF16 && dtype != MHLO_DT_F32) return fail(MHLO_CUDA_UNSUPPORTED, "%s: dtype %d", what, dtype);
    KvArgs kv;
    if (int st = kv_args(what, cache, batch, &kv)) return st;
    if (kv.head_dim != 64 && kv.head_dim != 96 && kv.head_dim != 128 && kv.head_dim != 256)
        return fail(MHLO_CUDA_UNSUPPORTED, "%s: head dimension %d (64, 96, 128 or 256)", what, kv.head_dim);
    if (q_heads < 1 || q_heads > 65535 || q_heads % kv.heads != 0)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld query heads over %d heads", what, static_cast<long long>(q_heads), kv.heads);
    if (!(scale > 0.f) || scale > 3.402823e38f) return fail(MHLO_CUDA_UNSUPPORTED, "%s: the scale has to be positive and finite", what);
    if (batch->tokens == 0 || batch->seqs == 0) return MHLO_CUDA_OK;
    if (!batch->token_starts && batch->tokens != batch->seqs)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld tokens of %lld sequences need token_starts", what, static_cast<long long>(batch->tokens), static_cast<long long>(batch->seqs));
    if (!q_dev || !o_dev) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null queries or result", what);
    if (int st = kv_row_strides(what, "q", q_strides)) return st;
    if (int st = kv_row_strides(what, "o", o_strides)) return st;
    if (q_dev == o_dev && (q_strides[0] != o_strides[0] || q_strides[1] != o_strides[1]))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: a result in place of the queries needs their strides", what);
    const int64_t need = mhlo_cuda_cached_attention_scratch_bytes(cache, batch, q_heads);
    if (need > 0 && (!scratch_dev || scratch_bytes < need || !aligned16(scratch_dev)))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: needs %lld bytes of 16-byte aligned scratch", what, static_cast<long long>(need));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == MHLO_DT_F32) return launch<float>(kv, q_dev, q_strides, q_heads, scale, o_dev, o_strides, lse_dev, st);
    if (dtype == MHLO_DT_F16) return launch<__half>(kv, q_dev, q_strides, q_heads, scale, o_dev, o_strides, lse_dev, st);
    return launch<__nv_bfloat16>(kv, q_dev, q_strides, q_heads, scale, o_dev, o_strides, lse_dev, st);
}

}  // extern "C"
