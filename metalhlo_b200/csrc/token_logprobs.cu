// Log probabilities of given tokens, entropy, the largest alternatives, and their gradient with respect to the logits.
//
// With z = scale x and m = max z: S = sum exp(z - m), T = sum exp(z - m) (z - m), lse = m + log S, entropy = log S - T / S. A logit
// of -infinity has probability 0 and no part in T.
#include <algorithm>

#include "common.cuh"

namespace mhlo {
namespace {

constexpr int kThreads = 512;

template <typename T>
struct LogprobParams {
    const T* x;
    int64_t row_stride, vocab;
    float scale;
    const void* targets;
    int32_t wide_targets;  // I64
    float* logprobs;
    float* entropy;
    float* lse;
    int32_t top_k;
    float* top_logprobs;
    int32_t* top_ids;
};

__device__ __forceinline__ int64_t target_of(const void* targets, int32_t wide, int64_t row) {
    return wide ? static_cast<const int64_t*>(targets)[row] : static_cast<const int32_t*>(targets)[row];
}

// Logits in the order of the alternatives: NaN above all, -0 = +0.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const __grid_constant__ LogprobParams<T> p) {
    __shared__ float scratch[3][32];
    __shared__ unsigned long long best[kThreads / 32];
    const int64_t row = blockIdx.x;
    const T* x = p.x + row * p.row_stride;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY;
    for (int64_t i = threadIdx.x; i < p.vocab; i += kThreads) m = fmaxf(m, VecTraits<T>::to_float(x[i]) * p.scale);
    m = cta_reduce<MaxOp>(m, scratch[0]);
    float s = 0.f, t = 0.f;
    for (int64_t i = threadIdx.x; i < p.vocab; i += kThreads) {
        const float d = VecTraits<T>::to_float(x[i]) * p.scale - m, e = expf(d);
        s += e;
        t += e * fmaxf(d, -200.f);
    }
    s = cta_reduce<SumOp>(s, scratch[1]);
    t = cta_reduce<SumOp>(t, scratch[2]);
    const float lse = m + logf(s);
    if (threadIdx.x == 0) {
        if (p.lse) p.lse[row] = lse;
        if (p.entropy) p.entropy[row] = logf(s) - t / s;
        if (p.targets) {
            const int64_t id = target_of(p.targets, p.wide_targets, row);
            p.logprobs[row] = id < 0 ? 0.f : id >= p.vocab ? NAN : VecTraits<T>::to_float(x[id]) * p.scale - lse;
        }
    }
    unsigned long long below = ~0ull;  // the last alternative taken
    for (int k = 0; k < p.top_k; ++k) {
        unsigned long long mine = 0;
        for (int64_t i = threadIdx.x; i < p.vocab; i += kThreads) {
            const unsigned long long key = static_cast<unsigned long long>(order_of(VecTraits<T>::to_float(x[i]))) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
            if (key < below && key > mine) mine = key;
        }
        for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        __syncthreads();
        if (lane == 0) best[warp] = mine;
        __syncthreads();
        for (int w = 0; w < kThreads / 32; ++w) mine = max(mine, best[w]);
        below = mine;
        if (threadIdx.x == 0) {
            const uint32_t id = 0xffffffffu - static_cast<uint32_t>(mine);
            p.top_ids[row * p.top_k + k] = static_cast<int32_t>(id);
            p.top_logprobs[row * p.top_k + k] = VecTraits<T>::to_float(x[id]) * p.scale - lse;
        }
    }
}

template <typename T>
struct GradParams {
    const T* x;
    int64_t row_stride, vocab;
    float scale;
    const void* targets;
    int32_t wide_targets;
    const float* lse;
    const float* entropy;
    const float* g;
    const float* e;
    int32_t top_k;
    const int32_t* top_ids;
    const float* t;
    T* dx;
    int64_t dx_row_stride;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_grad_kernel(const __grid_constant__ GradParams<T> p) {
    __shared__ float weight[MHLO_CUDA_TOP_LOGPROBS_MAX];
    __shared__ int32_t ids[MHLO_CUDA_TOP_LOGPROBS_MAX];
    const int64_t row = blockIdx.x;
    const T* x = p.x + row * p.row_stride;
    T* dx = p.dx + row * p.dx_row_stride;
    int64_t target = -1;
    float g = 0.f;
    if (p.g && p.targets) {
        target = target_of(p.targets, p.wide_targets, row);
        g = target < 0 ? 0.f : target >= p.vocab ? NAN : p.g[row];
    }
    if (threadIdx.x < p.top_k) {
        const int32_t id = p.top_ids[row * p.top_k + threadIdx.x];
        ids[threadIdx.x] = id;
        weight[threadIdx.x] = id < 0 ? 0.f : id >= p.vocab ? NAN : p.t[row * p.top_k + threadIdx.x];
    }
    __syncthreads();
    float all = g;
    for (int k = 0; k < p.top_k; ++k) all += weight[k];
    const float lse = p.lse[row], e = p.e ? p.e[row] : 0.f, h = p.e ? p.entropy[row] : 0.f;
    for (int64_t i = threadIdx.x; i < p.vocab; i += kThreads) {
        const float logp = VecTraits<T>::to_float(x[i]) * p.scale - lse, pr = expf(logp);
        float d = -pr * (all + e * (fmaxf(logp, -200.f) + h));
        if (i == target) d += g;
        for (int k = 0; k < p.top_k; ++k) d += ids[k] == i ? weight[k] : 0.f;
        dx[i] = VecTraits<T>::from_float(d * p.scale);
    }
}

int check_rows(const char* what, int32_t dtype, const void* x, int64_t row_stride, int64_t rows, int64_t vocab, float scale, const void* targets,
               int32_t target_dtype, int32_t top_k) {
    if (dtype != MHLO_DT_F16 && dtype != MHLO_DT_BF16 && dtype != MHLO_DT_F32) return fail(MHLO_CUDA_UNSUPPORTED, "%s: dtype %d", what, dtype);
    if (rows < 0 || rows > 0x7fffffff || vocab < 1 || vocab > 0x7fffffff || row_stride < vocab)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld rows of %lld logits, %lld apart", what, static_cast<long long>(rows), static_cast<long long>(vocab), static_cast<long long>(row_stride));
    if (!(scale > 0.f) || scale > 3.402823e38f) return fail(MHLO_CUDA_UNSUPPORTED, "%s: the scale has to be positive and finite", what);
    if (targets && target_dtype != MHLO_DT_I32 && target_dtype != MHLO_DT_I64) return fail(MHLO_CUDA_UNSUPPORTED, "%s: targets of dtype %d (I32 or I64)", what, target_dtype);
    if (top_k < 0 || top_k > MHLO_CUDA_TOP_LOGPROBS_MAX || top_k > vocab) return fail(MHLO_CUDA_UNSUPPORTED, "%s: %d alternatives of %lld", what, top_k, static_cast<long long>(vocab));
    if (rows > 0 && !x) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null logits", what);
    return MHLO_CUDA_OK;
}

template <typename T>
int launch(const void* x, LogprobParams<T> p, int64_t rows, cudaStream_t stream) {
    p.x = static_cast<const T*>(x);
    logprobs_kernel<T><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(p);
    MHLO_CUDA_CHECK_LAUNCH("token_logprobs");
    return MHLO_CUDA_OK;
}

template <typename T>
int launch_grad(const void* x, void* dx, GradParams<T> p, int64_t rows, cudaStream_t stream) {
    p.x = static_cast<const T*>(x);
    p.dx = static_cast<T*>(dx);
    logprobs_grad_kernel<T><<<static_cast<unsigned>(rows), kThreads, 0, stream>>>(p);
    MHLO_CUDA_CHECK_LAUNCH("token_logprobs_grad");
    return MHLO_CUDA_OK;
}

}  // namespace
}  // namespace mhlo

using namespace mhlo;

extern "C" {

int mhlo_cuda_token_logprobs(int32_t dtype, const void* x_dev, int64_t row_stride, int64_t rows, int64_t vocab, float scale, const void* targets_dev,
                             int32_t target_dtype, float* logprobs_dev, float* entropy_dev, float* lse_dev, int32_t top_k, float* top_logprobs_dev,
                             int32_t* top_ids_dev, mhlo_cuda_stream_t stream) {
    static const char* const what = "token_logprobs";
    if (int st = check_rows(what, dtype, x_dev, row_stride, rows, vocab, scale, targets_dev, target_dtype, top_k)) return st;
    if (rows == 0) return MHLO_CUDA_OK;
    if ((targets_dev == nullptr) != (logprobs_dev == nullptr)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: targets and their log probabilities go together", what);
    if (top_k > 0 && (!top_logprobs_dev || !top_ids_dev)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null result for the alternatives", what);
    auto run = [&](auto zero) {
        using T = decltype(zero);
        LogprobParams<T> p{nullptr, row_stride, vocab, scale, targets_dev, target_dtype == MHLO_DT_I64, logprobs_dev, entropy_dev, lse_dev, top_k, top_logprobs_dev, top_ids_dev};
        return launch<T>(x_dev, p, rows, static_cast<cudaStream_t>(stream));
    };
    if (dtype == MHLO_DT_F32) return run(float{});
    if (dtype == MHLO_DT_F16) return run(__half{});
    return run(__nv_bfloat16{});
}

int mhlo_cuda_token_logprobs_grad(int32_t dtype, const void* x_dev, int64_t row_stride, int64_t rows, int64_t vocab, float scale, const void* targets_dev,
                                  int32_t target_dtype, const float* lse_dev, const float* entropy_dev, const float* grad_logprobs_dev,
                                  const float* grad_entropy_dev, int32_t top_k, const int32_t* top_ids_dev, const float* grad_top_dev, void* dx_dev,
                                  int64_t dx_row_stride, mhlo_cuda_stream_t stream) {
    static const char* const what = "token_logprobs_grad";
    if (int st = check_rows(what, dtype, x_dev, row_stride, rows, vocab, scale, targets_dev, target_dtype, top_k)) return st;
    if (rows == 0) return MHLO_CUDA_OK;
    if (!lse_dev || !dx_dev) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null lse or result", what);
    if (grad_logprobs_dev && !targets_dev) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: a gradient of log probabilities without targets", what);
    if (grad_entropy_dev && !entropy_dev) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: a gradient of the entropy without the entropy", what);
    if (grad_top_dev && (top_k == 0 || !top_ids_dev)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: a gradient of alternatives without their ids", what);
    if (dx_row_stride < vocab || (dx_dev == x_dev && dx_row_stride != row_stride))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: rows of the result %lld apart", what, static_cast<long long>(dx_row_stride));
    auto run = [&](auto zero) {
        using T = decltype(zero);
        GradParams<T> p{nullptr, row_stride, vocab, scale, targets_dev, target_dtype == MHLO_DT_I64, lse_dev, entropy_dev, grad_logprobs_dev, grad_entropy_dev,
                        grad_top_dev ? top_k : 0, top_ids_dev, grad_top_dev, nullptr, dx_row_stride};
        return launch_grad<T>(x_dev, dx_dev, p, rows, static_cast<cudaStream_t>(stream));
    };
    if (dtype == MHLO_DT_F32) return run(float{});
    if (dtype == MHLO_DT_F16) return run(__half{});
    return run(__nv_bfloat16{});
}

}  // extern "C"
