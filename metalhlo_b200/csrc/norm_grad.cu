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
// bf16, [32768, 4096] with a residual's gradient: 226-238 us (4.5 to 4.8 TB/s; a row is 4400 instructions of its warps, 57 % of the issue slots, and 16 elements of
// x, dy, gamma and two sums fill 128 registers, so 16 warps share an SM). 8 elements a thread and twice the warps took 378 us, a row at a time in three CTAs 350,
// one element at a time instead of pairs 276. fp32, [4096, 5120]: 50 us (5 TB/s), 6 of them the join. f16, [1021, 769] off the 16-byte grid: 13 us, two launches.
#include <algorithm>
#include <type_traits>

#include "kv_cache.cuh"
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

// Read once, and not through the path for constants (ld.global.nc): the call may write its result over the tensor.
__device__ __forceinline__ uint4 ld_once16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

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
        else raw = ld_once16(p);
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

// A row a CTA, E elements a thread. A stage of the ring holds a row of x and one of dy, each from the 16-byte boundary below its start on.
constexpr int kMostThreads = 1024;
template <typename T>
__host__ __device__ constexpr int ring_bytes(int hidden) { return (hidden * static_cast<int>(sizeof(T)) + 30) / 16 * 16; }

__device__ __forceinline__ void bulk_copy(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(to)), "l"(from), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// Shuffles are what a row costs most of (one a clock and SM): sums of several values are taken together, the lanes that have `bit` going on with b, the
// others with a.
__device__ __forceinline__ float fold(float a, float b, int bit) {
    const bool upper = (threadIdx.x & bit) != 0;
    return (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, bit);
}
__device__ __forceinline__ float add_across(float v, int bit) { return v + __shfl_xor_sync(0xffffffffu, v, bit); }

// Sums over the warp of one value a row, in all lanes.
template <int R>
__device__ __forceinline__ void sum_rows(float (&v)[R]) {
    if constexpr (R == 1) {
        v[0] = sum32(v[0]);
    } else {
        float x = fold(v[0], v[1], 16);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) x = add_across(x, o);
        const float y = __shfl_xor_sync(0xffffffffu, x, 16);
        const bool upper = (threadIdx.x & 16) != 0;
        v[0] = upper ? y : x;
        v[1] = upper ? x : y;
    }
}

// Sums over the warp of three values a row, to where they are wanted: parts[row][warp] = {mean, a, b, c}.
template <int R>
__device__ __forceinline__ void leave_sums(float4 (*parts)[32], const float (&mean)[R], const float (&a)[R], const float (&b)[R], const float (&c)[R]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float x, y, z;
    if constexpr (R == 2) x = fold(a[0], a[1], 16), y = fold(b[0], b[1], 16), z = fold(c[0], c[1], 16);
    else x = add_across(a[0], 16), y = add_across(b[0], 16), z = add_across(c[0], 16);
    x = fold(x, y, 8);
    z = add_across(z, 8);
    x = fold(x, z, 4);
    x = add_across(add_across(x, 2), 1);
    // lanes 0, 8, 4 of a row's half: a, b, c
    const int row = R == 2 ? lane >> 4 : 0, which = lane & 15;
    if ((R == 2 || lane < 16) && (which & 3) == 0) {
        float* const to = reinterpret_cast<float*>(&parts[row][warp]);
        to[which == 0 ? 1 : which == 8 ? 2 : which == 4 ? 3 : 0] = which == 12 ? (R == 2 && row == 1 ? mean[R - 1] : mean[0]) : x;
    }
}

__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// A thread's elements of a row go in units of pairs, for two of which one instruction does: a 16-byte vector (VEC), or two elements by themselves,
// threads apart.
template <typename T, bool VEC>
struct Unit {
    static constexpr int kElems = VEC ? VecTraits<T>::kElems : 2, kPairs = kElems / 2;
    using Held = typename std::conditional<VEC, uint4, T[2]>::type;  // as it is in memory
    int at[VEC ? 1 : 2];
    bool has[VEC ? 1 : 2];
    __device__ __forceinline__ Unit(int u, int tid, int threads, int hidden) {
#pragma unroll
        for (int i = 0; i < (VEC ? 1 : 2); ++i) {
            at[i] = VEC ? (u * threads + tid) * kElems : (2 * u + i) * threads + tid;
            has[i] = at[i] < hidden;
        }
    }
    __device__ __forceinline__ void hold(const T* row, Held& h) const {
        if constexpr (VEC) {
            if (has[0]) h = ld_once16(row + at[0]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (has[i]) h[i] = row[at[i]];
        }
    }
    __device__ __forceinline__ void unpack(const Held& h, float2* v) const {
        if constexpr (VEC) VecTraits<T>::unpack2(h, v);
        else *v = make_float2(VecTraits<T>::to_float(h[0]), VecTraits<T>::to_float(h[1]));
    }
    // Elements behind the row's end: not to be looked at (VEC), zero.
    __device__ __forceinline__ void load(const T* row, float2* v) const {
        if constexpr (VEC) VecTraits<T>::unpack2(*reinterpret_cast<const uint4*>(row + at[0]), v);
        else *v = make_float2(has[0] ? VecTraits<T>::to_float(row[at[0]]) : 0.f, has[1] ? VecTraits<T>::to_float(row[at[1]]) : 0.f);
    }
    __device__ __forceinline__ bool any() const { return has[0]; }
    __device__ __forceinline__ float2 only(float2 v) const {
        if constexpr (!VEC) v = make_float2(has[0] ? v.x : 0.f, has[1] ? v.y : 0.f);
        return v;
    }
    __device__ __forceinline__ void store(T* row, const float2* v) const {
        if constexpr (VEC) {
            st_stream16(row + at[0], VecTraits<T>::pack2(v));
        } else {
            if (has[0]) row[at[0]] = VecTraits<T>::from_float(v->x);
            if (has[1]) row[at[1]] = VecTraits<T>::from_float(v->y);
        }
    }
    __device__ __forceinline__ void store_sums(float* row, const float2* v) const {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            if (VEC || has[0]) row[at[0] + 2 * k] = v[k].x;
            if (VEC) row[at[0] + 2 * k + 1] = v[k].y;
            else if (has[VEC ? 0 : 1]) row[at[VEC ? 0 : 1]] = v[k].y;
        }
    }
};

constexpr int kMostStages = 12;
constexpr int kWaitError = 40;  // a copy did not come: what the call leaves is not its result
// A copy did not come. Those still under way end, if they do, before the CTA does. slot, parity: of the row that did not come; rows: that are left from it on.
__device__ __noinline__ void give_up(uint64_t* full, int stages, int slot, uint32_t parity, int64_t rows, int64_t step) {
    kv_report(kWaitError);
    for (int k = 1; k < stages && k * step < rows; ++k) {
        if (++slot == stages) slot = 0, parity ^= 1;
        if (!mbar_wait(&full[slot], parity)) return;
    }
}

// E: elements of a thread. R: rows at once, which share a barrier and the latency of the reductions.
template <typename T, bool VEC, bool RMS, int E, int R, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) norm_grad_kernel(const __grid_constant__ NormGradParams<T> p, int32_t stages) {
    using U = Unit<T, VEC>;
    constexpr int N = E / U::kElems, P = U::kPairs;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ uint64_t full[kMostStages];
    __shared__ float4 parts[2][R][32];  // of a row, by warp: mean, squares, t, t times deviation
    __shared__ float counts[32];        // elements of a warp
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    const int row_bytes = ring_bytes<T>(p.hidden);
    const float over_hidden = 1.f / static_cast<float>(p.hidden);
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
        fence_barrier_init();
    }
    float mine = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const U u(n, tid, threads, p.hidden);
        mine += VEC ? (u.has[0] ? U::kElems : 0) : u.has[0] + u.has[VEC ? 0 : 1];
    }
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
    const int64_t step = gridDim.x;
    if (tid == 0)
        for (int s = 0; s < stages; ++s) send(row + s * step, s);
    float2 gamma[E / 2], of_gamma[E / 2], of_beta[E / 2];
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
        gamma[k] = twice(1.f);
        of_gamma[k] = of_beta[k] = twice(0.f);
    }
    if (p.gamma != nullptr) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const U u(n, tid, threads, p.hidden);
            if (u.any()) u.load(p.gamma, gamma + n * P);
        }
    }
    int stage = 0;
    uint32_t phase = 0;
    for (int turn = 0; row < p.rows; row += R * step, turn ^= 1) {
        const T *x[R], *dy[R];
        float mean[R], squares[R], sum_t[R], sum_td[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t r = row + i * step;
            const int at = stage + i < stages ? stage + i : stage + i - stages;
            x[i] = reinterpret_cast<const T*>(ring + at * 2 * row_bytes + (VEC ? 0 : reinterpret_cast<uintptr_t>(p.x + r * p.hidden) & 15));
            dy[i] = reinterpret_cast<const T*>(ring + (at * 2 + 1) * row_bytes + (VEC ? 0 : reinterpret_cast<uintptr_t>(p.dy + r * p.hidden) & 15));
            if (r < p.rows && !mbar_wait(&full[at], phase ^ (stage + i < stages ? 0u : 1u))) return give_up(full, stages, at, phase ^ (stage + i < stages ? 0u : 1u), p.rows - r, step);
            mean[i] = 0.f;
            if (!RMS && r < p.rows) {
                float2 sum = twice(0.f);
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const U u(n, tid, threads, p.hidden);
                    if (!u.any()) continue;
                    float2 v[P];
                    u.load(x[i], v);
#pragma unroll
                    for (int k = 0; k < P; ++k) sum = __fadd2_rn(sum, v[k]);
                }
                mean[i] = sum.x + sum.y;
            }
        }
        if (!RMS) {
            sum_rows<R>(mean);
#pragma unroll
            for (int i = 0; i < R; ++i) mean[i] *= over_count;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float2 sq = twice(0.f), st = twice(0.f), std = twice(0.f);
            const float2 minus_mean = twice(-mean[i]);
            if (row + i * step < p.rows) {
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const U u(n, tid, threads, p.hidden);
                    if (!u.any()) continue;
                    float2 v[P], t[P];
                    u.load(x[i], v);
                    u.load(dy[i], t);
#pragma unroll
                    for (int k = 0; k < P; ++k) {
                        const float2 d = RMS ? v[k] : u.only(__fadd2_rn(v[k], minus_mean)), tg = __fmul2_rn(t[k], gamma[n * P + k]);
                        sq = __ffma2_rn(d, d, sq);
                        if (!RMS) st = __fadd2_rn(st, tg);
                        std = __ffma2_rn(tg, d, std);
                    }
                }
            }
            squares[i] = sq.x + sq.y;
            sum_t[i] = st.x + st.y;
            sum_td[i] = std.x + std.y;
        }
        leave_sums<R>(parts[turn], mean, squares, sum_t, sum_td);
        typename U::Held residual[R][N];
        if (p.residual != nullptr) {
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int n = 0; n < N; ++n)
                    if (row + i * step < p.rows) U(n, tid, threads, p.hidden).hold(p.residual + (row + i * step) * p.hidden, residual[i][n]);
        }
        __syncthreads();
        // all have done with the rows before these
        if (tid == 0 && row >= R * step) {
#pragma unroll
            for (int i = R; i > 0; --i) send(row + (stages - i) * step, stage >= i ? stage - i : stage - i + stages);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int64_t r = row + i * step;
            if (r >= p.rows) continue;
            // The warps' sums around their own means, joined around the first one's: differences of means are small, or at most as large as the
            // row's whole deviation.
            const float base = parts[turn][i][0].x;
            float sq = 0.f, td = 0.f, sum = 0.f, far = 0.f, far2 = 0.f;
            for (int w = 0; w < warps; ++w) {
                const float4 v = parts[turn][i][w];
                sq += v.y;
                td += v.w;
                if (!RMS) {
                    const float d = v.x - base, nd = counts[w] * d;
                    far += nd;
                    far2 = fmaf(nd, d, far2);
                    sum += v.z;
                    td = fmaf(v.z, d, td);
                }
            }
            const float shift = far * over_hidden, c1 = sum * over_hidden;
            if (!RMS) {
                sq += fmaf(-far, shift, far2);
                sq = sq < 0.f ? 0.f : sq;  // not fmaxf, which makes a number of a NaN
                td = fmaf(-shift, sum, td);
            }
            const float rs = rsqrtf(fmaf(sq, over_hidden, p.eps)), c2 = td * rs * over_hidden;
            const float2 rs2 = twice(rs), minus_mean = twice(-(base + shift)), minus_c1 = twice(-rs * c1), minus_c2 = twice(-rs * c2);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const U u(n, tid, threads, p.hidden);
                if (!u.any()) continue;
                float2 v[P], d[P], out[P];
                u.load(x[i], v);
                u.load(dy[i], d);
                if (p.residual != nullptr) {
                    u.unpack(residual[i][n], out);
                } else {
#pragma unroll
                    for (int k = 0; k < P; ++k) out[k] = twice(0.f);
                }
#pragma unroll
                for (int k = 0; k < P; ++k) {
                    const float2 y = __fmul2_rn(RMS ? v[k] : __fadd2_rn(v[k], minus_mean), rs2), t = __fmul2_rn(d[k], gamma[n * P + k]);
                    of_gamma[n * P + k] = __ffma2_rn(d[k], y, of_gamma[n * P + k]);
                    if (!RMS) {
                        of_beta[n * P + k] = __fadd2_rn(of_beta[n * P + k], d[k]);
                        out[k] = __fadd2_rn(out[k], minus_c1);
                    }
                    out[k] = __ffma2_rn(t, rs2, __ffma2_rn(y, minus_c2, out[k]));
                }
                u.store(p.dx + r * p.hidden, out);
            }
        }
        stage += R;
        if (stage >= stages) stage -= stages, phase ^= 1;
    }
    if (p.partial == nullptr) return;
    float* const to = p.partial + static_cast<int64_t>(blockIdx.x) * (RMS ? 1 : 2) * p.hidden;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const U u(n, tid, threads, p.hidden);
        if (!u.any()) continue;
        u.store_sums(to, of_gamma + n * P);
        if (!RMS) u.store_sums(to + p.hidden, of_beta + n * P);
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
#pragma unroll 8
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

// per_sm: CTAs that an SM takes.
template <bool RMS, typename K, typename T, typename... Args>
int launch(K kernel, const NormGradParams<T>& p, int threads, int rows_of_cta, size_t smem, int per_sm, float* dgamma, float* dbeta, cudaStream_t stream, Args... args) {
    const int64_t grid = std::min<int64_t>((p.rows + rows_of_cta - 1) / rows_of_cta, std::min<int64_t>(kMostCtas, static_cast<int64_t>(per_sm) * kNumSMs));
    const cudaError_t e = launch_dependent(kernel, dim3(static_cast<unsigned>(grid)), dim3(static_cast<unsigned>(threads)), smem, stream, 1, grid < kNumSMs, p, args...);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of norm_grad failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("norm_grad");
    return p.partial == nullptr ? MHLO_CUDA_OK : join<RMS>(p.partial, grid, p.hidden, dgamma, dbeta, stream);
}

template <typename T, int W, int N, bool RMS>
int warp_rows(const NormGradParams<T>& p, float* dgamma, float* dbeta, cudaStream_t stream) {
    return launch<RMS>(norm_grad_warp_kernel<T, W, N, RMS>, p, kWarpThreads, kWarpThreads / 32, 2 * static_cast<size_t>(p.hidden) * sizeof(float), 2, dgamma, dbeta, stream);
}

// Shared memory of an SM for the rings of all its CTAs.
constexpr int kRingBytes = 220 * 1024;

template <typename T, bool VEC, bool RMS, int E, int R, int THREADS, int CTAS>
int cta_rows_of(const NormGradParams<T>& p, float* dgamma, float* dbeta, cudaStream_t stream) {
    auto kernel = norm_grad_kernel<T, VEC, RMS, E, R, THREADS, CTAS>;
    const int threads = ((p.hidden + E - 1) / E + 31) / 32 * 32, stage = 2 * ring_bytes<T>(p.hidden);
    // as many CTAs as the registers take, and stages as there is room for
    const int ctas = std::max(1, THREADS * CTAS / threads);
    const int stages = std::max(2 * R, std::min(kMostStages, kRingBytes / ctas / stage));  // the rows at hand, and the next ones
    static std::atomic<bool> allowed[64];
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), kRingBytes, allowed)) return st;
    return launch<RMS>(kernel, p, threads, 1, static_cast<size_t>(stages) * stage, std::min(ctas, std::max(1, kRingBytes / (stages * stage))), dgamma, dbeta, stream, stages);
}
// 512 threads an SM, of 128 registers, up to 8192 elements.
template <typename T, bool VEC, bool RMS>
int cta_rows(const NormGradParams<T>& p, float* dgamma, float* dbeta, cudaStream_t stream) {
    constexpr int R = VEC && sizeof(T) == 2 ? 2 : 1;  // four rows of x and dy in fp32 would not fit
    if (p.hidden <= 16 * 128) return cta_rows_of<T, VEC, RMS, 16, R, 128, 4>(p, dgamma, dbeta, stream);
    if (p.hidden <= 16 * 256) return cta_rows_of<T, VEC, RMS, 16, R, 256, 2>(p, dgamma, dbeta, stream);
    if (p.hidden <= 16 * 512) return cta_rows_of<T, VEC, RMS, 16, R, 512, 1>(p, dgamma, dbeta, stream);
    if (p.hidden <= 16 * 768) return cta_rows_of<T, VEC, RMS, 16, 1, 768, 1>(p, dgamma, dbeta, stream);
    return cta_rows_of<T, VEC, RMS, 16, 1, 1024, 1>(p, dgamma, dbeta, stream);
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

// By the width, as a batch has many rows; layer norm, bf16, both sides in us, for 8192 / 1000 / 64 rows. A row a warp or a CTA at 512 elements: 17 and 23 / 12 and 9 / 11 and 5 (255
// off the grid: 13 and 33 / 9 and 10 / 8 and 6). A row a CTA of 640 to 1024 threads, of 80 to 64 registers that spill, or three launches: 8200 elements 224 and 289 / 39 and 36 / 16 and
// 17, 12 288 268 and 408 / 54 and 47 / 24 and 21, 16 384 453 and 529 / 90 and 63 / 35 and 25; RMS norm 119 and 264 / 25 and 30 / 10 and 14, 148 and 379 / 33 and 39 / 14 and 18, 242 and
// 499 / 46 and 55 / 18 and 20.
template <typename T, bool RMS>
int norm_grad(const NormGradParams<T>& p, void* scratch, float* dgamma, float* dbeta, cudaStream_t stream) {
    constexpr int V = VecTraits<T>::kElems;
    const bool vec = p.hidden % V == 0 && aligned16(p.x) && aligned16(p.dy) && aligned16(p.dx) && (!p.gamma || aligned16(p.gamma)) && (!p.residual || aligned16(p.residual));
    if (vec && p.hidden <= 32 * V) return warp_rows<T, V, 1, RMS>(p, dgamma, dbeta, stream);
    if (vec && p.hidden <= 64 * V) return warp_rows<T, V, 2, RMS>(p, dgamma, dbeta, stream);
    if (!vec && p.hidden <= 256) return warp_rows<T, 1, 8, RMS>(p, dgamma, dbeta, stream);
    if (p.hidden <= 16 * kMostThreads && 4 * ring_bytes<T>(p.hidden) <= kRingBytes)  // two stages
        return vec ? cta_rows<T, true, RMS>(p, dgamma, dbeta, stream) : cta_rows<T, false, RMS>(p, dgamma, dbeta, stream);
    return long_rows<T, RMS>(p, scratch, dgamma, dbeta, stream);
}

int64_t scratch_bytes(int64_t rows, int64_t hidden) {
    const int64_t parts = hidden > 16 * kMostThreads ? kSplits : kMostCtas;  // such rows are not a CTA's
    const int64_t joined = std::min(rows, parts) * 2 * hidden * 4;
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

int norm_grad_device_error() { return take_kv_error(); }
bool norm_grad_error_store(int code) { return cudaMemcpyToSymbol(g_kv_error, &code, sizeof code) == cudaSuccess; }

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
