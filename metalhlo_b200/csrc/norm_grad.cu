// Gradients of layer norm and RMS norm over [rows, hidden]: with y = (x - mean) r, r = 1 / sqrt(var + eps) (RMS norm: mean = 0) and
// t = dy gamma,
//   dx = r (t - mean(t) - y mean(t y)) (RMS norm without mean(t)), dgamma = sum over rows of dy y, dbeta = sum over rows of dy.
// Mean and r are taken from x again, which has to be read anyway: nothing has to be kept of the forward half.
//
// Bound by HBM: x, dy (and the gradient of the residual stream) read once, dx written once. Rows of up to 512 elements are a warp's, held in its
// registers; longer ones a CTA's: x and dy arrive in shared memory by bulk copies some rows ahead, so that the registers are left for the sums
// of the thread's own columns over all rows of its CTA. The join of those over the CTAs is a second launch, in a fixed order. Each warp takes its
// own mean first and sums what deviates from that; the warps' sums are joined with one barrier a row, without differences of large
// numbers.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "tc_ptx.cuh"

namespace mhlo {
namespace {

template <typename T>
struct NormGradParams {
    const T *x, *gamma, *dy, *residual;
    T* dx;
    float* partial;  // [CTAs][2][hidden] (RMS norm: [CTAs][hidden]): sums of dy y, and of dy; null: not wanted
    int64_t rows;
    int32_t hidden;
    float eps;
};

__device__ __forceinline__ float sum32(float v) { return warp_reduce<SumOp>(v); }

// W elements side by side; where they are not on the 16-byte grid, one.
template <typename T, int W>
__device__ __forceinline__ void load(const T* p, float* f) {
    if constexpr (W == 1) *f = VecTraits<T>::to_float(*p);
    else VecTraits<T>::unpack(*reinterpret_cast<const uint4*>(p), f);
}
// The same as it is in memory, for what waits in registers.
template <typename T, int W>
struct Raw {
    typename std::conditional<W == 1, T, uint4>::type raw;
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (W == 1) raw = *p;
        else raw = ld_stream16(p);
    }
    __device__ __forceinline__ void unpack(float* f) const {
        if constexpr (W == 1) *f = VecTraits<T>::to_float(raw);
        else VecTraits<T>::unpack(raw, f);
    }
};
template <typename T, int W>
__device__ __forceinline__ void store(T* p, const float* f) {
    if constexpr (W == 1) *p = VecTraits<T>::from_float(*f);
    else st_stream16(p, VecTraits<T>::pack(f));
}

// A row a warp, W elements to a chunk, N chunks a lane.
constexpr int kWarpThreads = 256;
template <typename T, int W, int N, bool RMS>
__global__ void __launch_bounds__(kWarpThreads, 2) norm_grad_warp_kernel(const __grid_constant__ NormGradParams<T> p) {
    constexpr int E = W * N, kWarps = kWarpThreads / 32;
    extern __shared__ float columns[];  // as partial, the CTA's sums
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float over_hidden = 1.f / static_cast<float>(p.hidden);
    grid_dependency_wait();
    grid_dependency_release();
    int32_t at[N];
    float gamma[E], of_gamma[E], of_beta[E];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        at[n] = (n * 32 + lane) * W;
#pragma unroll
        for (int e = 0; e < W; ++e) gamma[n * W + e] = 1.f, of_gamma[n * W + e] = of_beta[n * W + e] = 0.f;
        if (p.gamma != nullptr && at[n] < p.hidden) load<T, W>(p.gamma + at[n], gamma + n * W);
    }
    const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps;
    Raw<T, W> next_x[N], next_dy[N];
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (r < p.rows && at[n] < p.hidden) {
                next_x[n].load(p.x + r * p.hidden + at[n]);
                next_dy[n].load(p.dy + r * p.hidden + at[n]);
            }
    };
    int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    fetch(row);
    for (; row < p.rows; row += step) {
        float x[E], dy[E];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            next_x[n].unpack(x + n * W);
            next_dy[n].unpack(dy + n * W);
            if (at[n] >= p.hidden) {
#pragma unroll
                for (int e = n * W; e < n * W + W; ++e) x[e] = dy[e] = 0.f;
            }
        }
        fetch(row + step);
        float mean = 0.f;
        if (!RMS) {
#pragma unroll
            for (int e = 0; e < E; ++e) mean += x[e];
            mean = sum32(mean) * over_hidden;
        }
        float squares = 0.f, sum_t = 0.f, sum_td = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bool has = at[n] < p.hidden;
#pragma unroll
            for (int e = n * W; e < n * W + W; ++e) {
                if (!RMS) x[e] = has ? x[e] - mean : 0.f;
                const float t = dy[e] * gamma[e];
                squares = fmaf(x[e], x[e], squares);
                sum_t += t;
                sum_td = fmaf(t, x[e], sum_td);
            }
        }
        squares = sum32(squares);
        sum_t = RMS ? 0.f : sum32(sum_t);
        sum_td = sum32(sum_td);
        const float r = rsqrtf(fmaf(squares, over_hidden, p.eps)), c1 = sum_t * over_hidden, c2 = sum_td * r * over_hidden;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (at[n] < p.hidden) {
                float out[W];
#pragma unroll
                for (int e = 0; e < W; ++e) out[e] = 0.f;
                if (p.residual != nullptr) load<T, W>(p.residual + row * p.hidden + at[n], out);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const int i = n * W + e;
                    const float y = x[i] * r;
                    of_gamma[i] = fmaf(dy[i], y, of_gamma[i]);
                    if (!RMS) of_beta[i] += dy[i];
                    out[e] = fmaf(r, fmaf(-y, c2, fmaf(dy[i], gamma[i], -c1)), out[e]);
                }
                store<T, W>(p.dx + row * p.hidden + at[n], out);
            }
        }
    }
    if (p.partial == nullptr) return;
    for (int w = 0; w < kWarps; ++w) {  // one warp after the other: a fixed order
        if (warp == w) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int e = 0; e < W; ++e)
                    if (at[n] < p.hidden) {
                        float *const g = columns + at[n] + e, *const b = g + p.hidden;
                        *g = of_gamma[n * W + e] + (w == 0 ? 0.f : *g);
                        if (!RMS) *b = of_beta[n * W + e] + (w == 0 ? 0.f : *b);
                    }
        }
        __syncthreads();
    }
    const int width = (RMS ? 1 : 2) * p.hidden;
    float* const to = p.partial + static_cast<int64_t>(blockIdx.x) * width;
    for (int i = tid; i < width; i += kWarpThreads) to[i] = columns[i];
}

// A row a CTA, 16 elements a thread. A stage of the ring holds a row of x and one of dy, each from the 16-byte boundary below its start on.
constexpr int kEach = 16, kMostThreads = 1024;
template <typename T>
__host__ __device__ constexpr int ring_bytes(int hidden) { return (hidden * static_cast<int>(sizeof(T)) + 30) / 16 * 16; }

__device__ __forceinline__ void bulk_copy(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)), "l"(from), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

constexpr int kMostStages = 8;
template <typename T, bool VEC, bool RMS, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_grad_kernel(const __grid_constant__ NormGradParams<T> p, int32_t stages) {
    constexpr int W = VEC ? VecTraits<T>::kElems : 1, N = kEach / W;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ uint64_t full[kMostStages];
    __shared__ float4 parts[2][32];  // of a row, by warp
    __shared__ float counts[32];     // elements of a warp
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    const int row_bytes = ring_bytes<T>(p.hidden);
    const float over_hidden = 1.f / static_cast<float>(p.hidden);
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
        fence_barrier_init();
    }
    float mine = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) mine += (n * threads + tid) * W < p.hidden ? W : 0;
    const float count = sum32(mine), over_count = count > 0.f ? 1.f / count : 0.f;
    if (lane == 0) counts[warp] = count;
    __syncthreads();
    grid_dependency_wait();
    grid_dependency_release();
    // One thread: row r on its way into a stage. The bytes behind the tensor's last 16-byte boundary are not touched: they go by hand.
    auto send = [&](int64_t r, int stage) {
        if (r >= p.rows) return;
        const T* const from[2] = {p.x, p.dy};
        uint32_t bytes[2];
        uintptr_t start[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uintptr_t begin = reinterpret_cast<uintptr_t>(from[i] + r * p.hidden), end = begin + p.hidden * sizeof(T);
            start[i] = begin & ~static_cast<uintptr_t>(15);
            uint8_t* const to = ring + (stage * 2 + i) * row_bytes;
            uintptr_t upto = (end + 15) & ~static_cast<uintptr_t>(15);
            if (upto != end && r == p.rows - 1) {
                upto = end & ~static_cast<uintptr_t>(15);
                for (uintptr_t b = max(upto, begin); b < end; b += sizeof(T)) *reinterpret_cast<T*>(to + (b - start[i])) = *reinterpret_cast<const T*>(b);
            }
            bytes[i] = upto > start[i] ? static_cast<uint32_t>(upto - start[i]) : 0;
        }
        mbar_expect_tx(&full[stage], bytes[0] + bytes[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (bytes[i] > 0) bulk_copy(ring + (stage * 2 + i) * row_bytes, reinterpret_cast<const void*>(start[i]), bytes[i], &full[stage]);
    };
    int64_t row = blockIdx.x;
    if (tid == 0)
        for (int s = 0; s < stages; ++s) send(row + static_cast<int64_t>(s) * gridDim.x, s);
    float of_gamma[kEach], of_beta[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) of_gamma[e] = of_beta[e] = 0.f;
    int stage = 0;
    uint32_t phase = 0;
    for (int turn = 0; row < p.rows; row += gridDim.x, turn ^= 1) {
        Raw<T, W> residual[N];
        if (p.residual != nullptr) {
#pragma unroll
            for (int n = 0; n < N; ++n)
                if ((n * threads + tid) * W < p.hidden) residual[n].load(p.residual + row * p.hidden + (n * threads + tid) * W);
        }
        const T *const x = reinterpret_cast<const T*>(ring + stage * 2 * row_bytes + (VEC ? 0 : reinterpret_cast<uintptr_t>(p.x + row * p.hidden) & 15)),
                *const dy = reinterpret_cast<const T*>(ring + (stage * 2 + 1) * row_bytes + (VEC ? 0 : reinterpret_cast<uintptr_t>(p.dy + row * p.hidden) & 15));
        if (!mbar_wait(&full[stage], phase)) return;  // cannot be: nothing but the copies is waited for
        float mean = 0.f;
        float dev[kEach];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = (n * threads + tid) * W;
#pragma unroll
            for (int e = 0; e < W; ++e) dev[n * W + e] = 0.f;
            if (i < p.hidden) load<T, W>(x + i, dev + n * W);
#pragma unroll
            for (int e = 0; e < W; ++e) mean += dev[n * W + e];
        }
        mean = RMS ? 0.f : sum32(mean) * over_count;
        float squares = 0.f, sum_t = 0.f, sum_td = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = (n * threads + tid) * W;
            if (i < p.hidden) {
                float t[W], g[W];
                load<T, W>(dy + i, t);
                if (p.gamma != nullptr) load<T, W>(p.gamma + i, g);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    if (p.gamma != nullptr) t[e] *= g[e];
                    const float d = dev[n * W + e] - mean;
                    squares = fmaf(d, d, squares);
                    sum_t += t[e];
                    sum_td = fmaf(t[e], d, sum_td);
                }
            }
        }
        squares = sum32(squares);
        if (!RMS) sum_t = sum32(sum_t);
        sum_td = sum32(sum_td);
        if (lane == 0) parts[turn][warp] = make_float4(mean, squares, sum_t, sum_td);
        __syncthreads();
        // all have done with the row before this one
        if (tid == 0 && row >= gridDim.x) {
            const int before = stage == 0 ? stages - 1 : stage - 1;
            send(row + static_cast<int64_t>(stages - 1) * gridDim.x, before);
        }
        const bool there = lane < warps;
        const float4 w = there ? parts[turn][lane] : make_float4(0.f, 0.f, 0.f, 0.f);
        if (RMS) {
            squares = sum32(w.y);
            sum_td = sum32(w.w);
        } else {
            const float n = there ? counts[lane] : 0.f;
            mean = sum32(n * w.x) * over_hidden;
            const float d = w.x - mean;
            squares = sum32(there ? fmaf(n * d, d, w.y) : 0.f);
            sum_t = sum32(w.z);
            sum_td = sum32(there ? fmaf(w.z, d, w.w) : 0.f);
        }
        const float r = rsqrtf(fmaf(squares, over_hidden, p.eps)), c1 = RMS ? 0.f : sum_t * over_hidden, c2 = sum_td * r * over_hidden;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int i = (n * threads + tid) * W;
            if (i < p.hidden) {
                float d[W], g[W], out[W], rest[W];
                if (p.residual != nullptr) residual[n].unpack(rest);
                load<T, W>(dy + i, d);
                if (p.gamma != nullptr) load<T, W>(p.gamma + i, g);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const int k = n * W + e;
                    const float y = (dev[k] - mean) * r, t = p.gamma != nullptr ? d[e] * g[e] : d[e];
                    of_gamma[k] = fmaf(d[e], y, of_gamma[k]);
                    if (!RMS) of_beta[k] += d[e];
                    out[e] = r * fmaf(-y, c2, t - c1);
                    if (p.residual != nullptr) out[e] += rest[e];
                }
                store<T, W>(p.dx + row * p.hidden + i, out);
            }
        }
        if (++stage == stages) stage = 0, phase ^= 1;
    }
    if (p.partial == nullptr) return;
    float* const to = p.partial + static_cast<int64_t>(blockIdx.x) * (RMS ? 1 : 2) * p.hidden;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int i = (n * threads + tid) * W;
        if (i < p.hidden) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                to[i + e] = of_gamma[n * W + e];
                if (!RMS) to[p.hidden + i + e] = of_beta[n * W + e];
            }
        }
    }
}

// Sums `parts` rows of `width` columns (dgamma, then dbeta), 32 a CTA: 32 warps take every 32nd part, and are joined in order.
constexpr int kJoin = 1024;
__global__ void __launch_bounds__(kJoin) norm_grad_join_kernel(const float* partial, int32_t parts, int32_t hidden, int32_t width, float* dgamma, float* dbeta) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_wait();
    const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float sum = 0.f;
    if (column < width) {
#pragma unroll 4
        for (int32_t i = warp; i < parts; i += 32) sum += partial[static_cast<int64_t>(i) * width + column];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp != 0 || column >= width) return;
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) sum += sums[w][lane];
    if (column < hidden) {
        if (dgamma != nullptr) dgamma[column] = sum;
    } else if (dbeta != nullptr) {
        dbeta[column - hidden] = sum;
    }
}

// ---- rows that are too long for the registers of a CTA: statistics, the columns' sums and dx, a launch each --------------------------------
constexpr int kLongThreads = 512, kSplits = 64;

struct RowSums {
    float mean, r, c1, c2;
};

template <typename T, bool RMS>
__global__ void __launch_bounds__(kLongThreads) norm_grad_long_sums_kernel(const __grid_constant__ NormGradParams<T> p, RowSums* to) {
    __shared__ float scratch[3][32];
    const T *const x = p.x + blockIdx.x * static_cast<int64_t>(p.hidden), *const dy = p.dy + blockIdx.x * static_cast<int64_t>(p.hidden);
    const float over_hidden = 1.f / static_cast<float>(p.hidden);
    float mean = 0.f;
    if (!RMS) {
        float sum = 0.f;
        for (int32_t i = threadIdx.x; i < p.hidden; i += kLongThreads) sum += VecTraits<T>::to_float(x[i]);
        mean = cta_reduce<SumOp>(sum, scratch[0]) * over_hidden;
        __syncthreads();
        // what the sum's rounding left
        float rest = 0.f;
        for (int32_t i = threadIdx.x; i < p.hidden; i += kLongThreads) rest += VecTraits<T>::to_float(x[i]) - mean;
        mean += cta_reduce<SumOp>(rest, scratch[1]) * over_hidden;
        __syncthreads();
    }
    float squares = 0.f, sum_t = 0.f, sum_td = 0.f;
    for (int32_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
        const float d = VecTraits<T>::to_float(x[i]) - mean, t = VecTraits<T>::to_float(dy[i]) * (p.gamma ? VecTraits<T>::to_float(p.gamma[i]) : 1.f);
        squares = fmaf(d, d, squares);
        sum_t += t;
        sum_td = fmaf(t, d, sum_td);
    }
    squares = cta_reduce<SumOp>(squares, scratch[0]);
    sum_t = cta_reduce<SumOp>(sum_t, scratch[1]);
    sum_td = cta_reduce<SumOp>(sum_td, scratch[2]);
    if (threadIdx.x == 0) {
        const float r = rsqrtf(fmaf(squares, over_hidden, p.eps));
        to[blockIdx.x] = {mean, r, RMS ? 0.f : sum_t * over_hidden, sum_td * r * over_hidden};
    }
}

template <typename T, bool RMS>
__global__ void __launch_bounds__(256) norm_grad_long_columns_kernel(const __grid_constant__ NormGradParams<T> p, const RowSums* sums) {
    const int32_t column = blockIdx.x * 256 + threadIdx.x;
    if (column >= p.hidden) return;
    float of_gamma = 0.f, of_beta = 0.f;
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float d = VecTraits<T>::to_float(p.dy[row * p.hidden + column]);
        of_gamma = fmaf(d, (VecTraits<T>::to_float(p.x[row * p.hidden + column]) - sums[row].mean) * sums[row].r, of_gamma);
        of_beta += d;
    }
    float* const to = p.partial + static_cast<int64_t>(blockIdx.y) * (RMS ? 1 : 2) * p.hidden;
    to[column] = of_gamma;
    if (!RMS) to[p.hidden + column] = of_beta;
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads) norm_grad_long_rows_kernel(const __grid_constant__ NormGradParams<T> p, const RowSums* sums) {
    const RowSums s = sums[blockIdx.x];
    const int64_t base = blockIdx.x * static_cast<int64_t>(p.hidden);
    for (int32_t i = threadIdx.x; i < p.hidden; i += kLongThreads) {
        const float t = VecTraits<T>::to_float(p.dy[base + i]) * (p.gamma ? VecTraits<T>::to_float(p.gamma[i]) : 1.f);
        const float y = (VecTraits<T>::to_float(p.x[base + i]) - s.mean) * s.r;
        p.dx[base + i] = VecTraits<T>::from_float(fmaf(s.r, fmaf(-y, s.c2, t - s.c1), p.residual ? VecTraits<T>::to_float(p.residual[base + i]) : 0.f));
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------------
constexpr int kMostCtas = 4 * kNumSMs;  // whose sums are joined

template <bool RMS>
int join(const float* partial, int64_t parts, int64_t hidden, float* dgamma, float* dbeta, cudaStream_t stream) {
    const int64_t width = (RMS ? 1 : 2) * hidden;
    const cudaError_t e = launch_dependent(norm_grad_join_kernel, dim3(static_cast<unsigned>((width + 31) / 32)), dim3(kJoin), 0, stream, 1, true, partial,
                                           static_cast<int32_t>(parts), static_cast<int32_t>(hidden), static_cast<int32_t>(width), dgamma, dbeta);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of norm_grad failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("norm_grad");
    return MHLO_CUDA_OK;
}

template <bool RMS, typename K, typename T, typename... Args>
int launch(K kernel, const NormGradParams<T>& p, int threads, int rows_of_cta, size_t smem, float* dgamma, float* dbeta, cudaStream_t stream, Args... args) {
    int per_sm = 0;
    MHLO_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem), MHLO_CUDA_EXECUTION_FAILED);
    const int64_t grid = std::min<int64_t>((p.rows + rows_of_cta - 1) / rows_of_cta, std::min<int64_t>(kMostCtas, static_cast<int64_t>(std::max(per_sm, 1)) * kNumSMs));
    const cudaError_t e = launch_dependent(kernel, dim3(static_cast<unsigned>(grid)), dim3(static_cast<unsigned>(threads)), smem, stream, 1, grid < kNumSMs, p, args...);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of norm_grad failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("norm_grad");
    return p.partial == nullptr ? MHLO_CUDA_OK : join<RMS>(p.partial, grid, p.hidden, dgamma, dbeta, stream);
}

template <typename T, int W, int N, bool RMS>
int warp_rows(const NormGradParams<T>& p, float* dgamma, float* dbeta, cudaStream_t stream) {
    return launch<RMS>(norm_grad_warp_kernel<T, W, N, RMS>, p, kWarpThreads, kWarpThreads / 32, 2 * static_cast<size_t>(p.hidden) * sizeof(float), dgamma, dbeta, stream);
}

// Shared memory of an SM for the rings of all its CTAs.
constexpr int kRingBytes = 220 * 1024;

template <typename T, bool VEC, bool RMS, int THREADS>
int cta_rows_of(const NormGradParams<T>& p, int threads, float* dgamma, float* dbeta, cudaStream_t stream) {
    const int stage = 2 * ring_bytes<T>(p.hidden);
    // as many CTAs as have 512 threads between them, and stages as there is room for
    const int ctas = std::max(1, 512 / threads);
    const int stages = std::max(2, std::min(kMostStages, kRingBytes / ctas / stage));
    static std::atomic<bool> allowed[64];
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(norm_grad_kernel<T, VEC, RMS, THREADS>), kRingBytes, allowed)) return st;
    return launch<RMS>(norm_grad_kernel<T, VEC, RMS, THREADS>, p, threads, 1, static_cast<size_t>(stages) * stage, dgamma, dbeta, stream, stages);
}
// A build for each number of registers that a thread can have: 128, 80, 64.
template <typename T, bool VEC, bool RMS>
int cta_rows(const NormGradParams<T>& p, float* dgamma, float* dbeta, cudaStream_t stream) {
    const int threads = ((p.hidden + kEach - 1) / kEach + 31) / 32 * 32;
    if (threads <= 512) return cta_rows_of<T, VEC, RMS, 512>(p, threads, dgamma, dbeta, stream);
    if (threads <= 768) return cta_rows_of<T, VEC, RMS, 768>(p, threads, dgamma, dbeta, stream);
    return cta_rows_of<T, VEC, RMS, kMostThreads>(p, threads, dgamma, dbeta, stream);
}

template <typename T, bool RMS>
int long_rows(NormGradParams<T> p, void* scratch, float* dgamma, float* dbeta, cudaStream_t stream) {
    RowSums* const sums = static_cast<RowSums*>(scratch);
    const unsigned rows = static_cast<unsigned>(p.rows);
    norm_grad_long_sums_kernel<T, RMS><<<rows, kLongThreads, 0, stream>>>(p, sums);
    MHLO_CUDA_CHECK_LAUNCH("norm_grad");
    if (p.partial != nullptr) {
        p.partial = reinterpret_cast<float*>(sums + p.rows);
        const int64_t splits = std::min<int64_t>(kSplits, p.rows);
        norm_grad_long_columns_kernel<T, RMS><<<dim3(static_cast<unsigned>((p.hidden + 255) / 256), static_cast<unsigned>(splits)), 256, 0, stream>>>(p, sums);
        MHLO_CUDA_CHECK_LAUNCH("norm_grad");
        if (int st = join<RMS>(p.partial, splits, p.hidden, dgamma, dbeta, stream)) return st;
    }
    norm_grad_long_rows_kernel<T><<<rows, kLongThreads, 0, stream>>>(p, sums);
    MHLO_CUDA_CHECK_LAUNCH("norm_grad");
    return MHLO_CUDA_OK;
}

template <typename T, bool RMS>
int norm_grad(const NormGradParams<T>& p, void* scratch, float* dgamma, float* dbeta, cudaStream_t stream) {
    constexpr int V = VecTraits<T>::kElems;
    const bool vec = p.hidden % V == 0 && aligned16(p.x) && aligned16(p.dy) && aligned16(p.dx) && (!p.gamma || aligned16(p.gamma)) && (!p.residual || aligned16(p.residual));
    if (vec && p.hidden <= 32 * V) return warp_rows<T, V, 1, RMS>(p, dgamma, dbeta, stream);
    if (vec && p.hidden <= 64 * V) return warp_rows<T, V, 2, RMS>(p, dgamma, dbeta, stream);
    if (!vec && p.hidden <= 256) return warp_rows<T, 1, 8, RMS>(p, dgamma, dbeta, stream);
    if (p.hidden <= kEach * kMostThreads && 4 * ring_bytes<T>(p.hidden) <= kRingBytes)  // two stages
        return vec ? cta_rows<T, true, RMS>(p, dgamma, dbeta, stream) : cta_rows<T, false, RMS>(p, dgamma, dbeta, stream);
    return long_rows<T, RMS>(p, scratch, dgamma, dbeta, stream);
}

int64_t scratch_bytes(int64_t rows, int64_t hidden) {
    const int64_t joined = std::min<int64_t>(rows, kMostCtas) * 2 * hidden * 4;
    return rows * static_cast<int64_t>(sizeof(RowSums)) + joined;
}

int entry(const char* what, bool rms, int32_t dtype, const void* x, const void* gamma, const void* dy, const void* residual, void* dx, float* dgamma, float* dbeta, int64_t rows,
          int64_t hidden, float eps, void* scratch, int64_t bytes, cudaStream_t stream) {
    if (dtype != MHLO_DT_F16 && dtype != MHLO_DT_BF16 && dtype != MHLO_DT_F32) return fail(MHLO_CUDA_UNSUPPORTED, "%s: dtype %d", what, dtype);
    if (rows < 0 || hidden < 1 || rows > 0x7fffffff || hidden > (1 << 24))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld rows of %lld elements", what, static_cast<long long>(rows), static_cast<long long>(hidden));
    if (!(eps >= 0.f)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: eps %g", what, eps);
    const bool sums = dgamma != nullptr || dbeta != nullptr;
    if (rows == 0) {
        if (dgamma) MHLO_CUDA_TRY(cudaMemsetAsync(dgamma, 0, hidden * 4, stream), MHLO_CUDA_EXECUTION_FAILED);
        if (dbeta) MHLO_CUDA_TRY(cudaMemsetAsync(dbeta, 0, hidden * 4, stream), MHLO_CUDA_EXECUTION_FAILED);
        return MHLO_CUDA_OK;
    }
    if (!x || !dy || !dx) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null x, dy or dx", what);
    if (!scratch || !aligned16(scratch) || bytes < scratch_bytes(rows, hidden))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld bytes of scratch, %lld needed, on 16 bytes", what, static_cast<long long>(bytes),
                    static_cast<long long>(scratch_bytes(rows, hidden)));
    auto run = [&](auto t) {
        using T = decltype(t);
        NormGradParams<T> p;
        p.x = static_cast<const T*>(x);
        p.gamma = static_cast<const T*>(gamma);
        p.dy = static_cast<const T*>(dy);
        p.residual = static_cast<const T*>(residual);
        p.dx = static_cast<T*>(dx);
        p.partial = sums ? static_cast<float*>(scratch) : nullptr;
        p.rows = rows;
        p.hidden = static_cast<int32_t>(hidden);
        p.eps = eps;
        return rms ? norm_grad<T, true>(p, scratch, dgamma, dbeta, stream) : norm_grad<T, false>(p, scratch, dgamma, dbeta, stream);
    };
    switch (dtype) {
        case MHLO_DT_F32: return run(float{});
        case MHLO_DT_F16: return run(__half{});
        default: return run(__nv_bfloat16{});
    }
}

}  // namespace
}  // namespace mhlo

using namespace mhlo;

extern "C" {

int64_t mhlo_cuda_norm_grad_scratch_bytes(int64_t rows, int64_t hidden) {
    return rows < 0 || hidden < 1 || rows > 0x7fffffff || hidden > (1 << 24) ? 0 : scratch_bytes(rows, hidden);
}

int mhlo_cuda_layer_norm_grad(int32_t dtype, const void* x_dev, const void* gamma_dev, const void* dy_dev, const void* residual_grad_dev, void* dx_dev, float* dgamma_dev,
                              float* dbeta_dev, int64_t rows, int64_t hidden, float eps, void* scratch_dev, int64_t scratch_bytes, mhlo_cuda_stream_t stream) {
    return entry("layer_norm_grad", false, dtype, x_dev, gamma_dev, dy_dev, residual_grad_dev, dx_dev, dgamma_dev, dbeta_dev, rows, hidden, eps, scratch_dev, scratch_bytes,
                 static_cast<cudaStream_t>(stream));
}

int mhlo_cuda_rms_norm_grad(int32_t dtype, const void* x_dev, const void* gamma_dev, const void* dy_dev, const void* residual_grad_dev, void* dx_dev, float* dgamma_dev,
                            int64_t rows, int64_t hidden, float eps, void* scratch_dev, int64_t scratch_bytes, mhlo_cuda_stream_t stream) {
    return entry("rms_norm_grad", true, dtype, x_dev, gamma_dev, dy_dev, residual_grad_dev, dx_dev, dgamma_dev, nullptr, rows, hidden, eps, scratch_dev, scratch_bytes,
                 static_cast<cudaStream_t>(stream));
}

}  // extern "C"
