// Log probabilities of given tokens, entropy, the largest alternatives, and their gradient with respect to the logits.
//
// With z = scale x and m = max x: d_i = (x_i - m) scale log2(e), S = sum 2^d, T = sum 2^d d, so lse = scale m + log S and entropy =
// log S - log(2) T / S. A logit of -infinity has probability 0 and no part in T. Differences to the maximum are taken before the
// scale: rows at the lowest value of their type neither overflow nor lose their digits.
//
// One pass. A thread has 4 vectors of 16 bytes in flight and keeps a running maximum with its S and T; when a batch of its vectors
// holds a larger logit, S and T move to it (T' = f (T + S delta), S' = f S with f = 2^delta). Everything is joined at the end of the
// row. Per element that is about five instructions and one exponential (16 a clock and SM), against 11 16-bit elements a clock and
// SM that the memory delivers. [4096, 50257] bf16: 77 us in a graph, 5.3 TB/s, 80 in calls one behind the other; ncu counts 70 % of issue
// slots and 67 % of the exponential unit. Gradient (read, exponential, write): 132 us in a graph, 6.2 TB/s, 135 in calls.
//
// Alternatives come out of the same pass. Keys are 64 bits, the logit's order above the complement of its place, so no two are equal
// and ties go to the lowest id. After the first batch a key that k threads' maxima reach bounds the k-th largest key from below; from
// then on vectors whose maximum reaches the bound, some dozens to a few hundred of a row, are noted on a list, and the
// threads do not wait for one another (looking through a vector at once cost its warp more than the exponentials). At the end what k
// maxima on the list reach is a bound again, and the keys of the vectors that reach it, hardly more than k, are ranked. Rows
// that overflow the list (rising logits) are gone over once more a vector a thread, with single keys on the list: when it
// overflows, it is cut to its k largest and the bound raised by the new vectors' own maxima: then hardly more than k threads have
// anything to add.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace mhlo {
namespace {

typedef unsigned long long Key;

constexpr int kBatch = 4;     // vectors of a thread in flight
// What the lists hold: keys (those of a batch at least, for as many threads as there may be alternatives) and vectors. A warp by itself
// has short rows and needs little.
template <int THREADS>
struct Lists {
    static constexpr int kKeys = THREADS < 64 ? 1152 : 2048;
    static constexpr int kVectors = THREADS < 64 ? 128 : 512;
};
constexpr float kLowest = -150.f;  // 2^-150 is 0 in fp32: what exponents are kept above, so that 0 * -infinity never comes up

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
    int32_t log2_parts;  // CTAs that share a row
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
__device__ __forceinline__ float number_of(uint32_t order) {  // back again; NaN for NaN's and for 0, which is no number's
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
__device__ __forceinline__ Key key_of(float x, uint32_t place) { return static_cast<Key>(order_of(x)) << 32 | (0xffffffffu - place); }

template <typename T>
__device__ __forceinline__ uint4 all_lowest();  // a vector of -infinities
template <>
__device__ __forceinline__ uint4 all_lowest<float>() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
template <>
__device__ __forceinline__ uint4 all_lowest<__half>() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
template <>
__device__ __forceinline__ uint4 all_lowest<__nv_bfloat16>() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }

// The largest element of a vector, NaN if there is one.
template <typename T>
__device__ __forceinline__ float largest_of(const uint4& v) {
    if constexpr (sizeof(T) == 4) {
        return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else if constexpr (std::is_same<T, __half>::value) {
        const __half2* h = reinterpret_cast<const __half2*>(&v);
        const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return max_nan(__low2float(m), __high2float(m));
    } else {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return max_nan(__low2float(m), __high2float(m));
    }
}

// Raises elements to `span` below the maximum m or a step of the type further down. NaN stays. Where the type has no number that far
// below m (m next to its lowest number, or its steps at m not fine enough for fp32 to tell), below() is less than span.
template <typename T>
struct Floor {
    T low;
    float m;
    __device__ __forceinline__ Floor(float m_, float span) : m(m_) {
        if constexpr (sizeof(T) == 4) low = fmaxf(m - span, -3.4028235e38f);
        else if constexpr (std::is_same<T, __half>::value) low = __float2half_rd(fmaxf(m - span, -65504.f));
        else low = __float2bfloat16_rd(fmaxf(m - span, -3.3895314e38f));
    }
    __device__ __forceinline__ float below() const { return m - VecTraits<T>::to_float(low); }
    __device__ __forceinline__ uint4 raise(const uint4& v) const {
        if constexpr (sizeof(T) == 4) {
            return make_uint4(__float_as_uint(max_nan(__uint_as_float(v.x), low)), __float_as_uint(max_nan(__uint_as_float(v.y), low)),
                              __float_as_uint(max_nan(__uint_as_float(v.z), low)), __float_as_uint(max_nan(__uint_as_float(v.w), low)));
        } else {
            uint4 out = v;
            if constexpr (std::is_same<T, __half>::value) {
                __half2* h = reinterpret_cast<__half2*>(&out);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], __half2half2(low));
            } else {
                __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&out);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __hmax2_nan(h[i], __bfloat162bfloat162(low));
            }
            return out;
        }
    }
};

// A row as up to E - 1 elements in front of the first 16-byte boundary, vectors, and up to E - 1 elements behind the last one.
template <typename T>
struct Row {
    const T* x;
    uint32_t vectors;  // rows have fewer than 2^31 elements
    int32_t head, tail;
    __device__ __forceinline__ Row(const T* row, int64_t n) : x(row) {
        constexpr int E = VecTraits<T>::kElems;
        const int64_t off = static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / static_cast<int64_t>(sizeof(T));
        head = static_cast<int32_t>(off < n ? off : n);
        vectors = static_cast<uint32_t>(n - head) / E;
        tail = static_cast<int32_t>(static_cast<uint32_t>(n - head) % E);
    }
    __device__ __forceinline__ int32_t singles() const { return head + tail; }
    __device__ __forceinline__ int64_t place_of_single(int32_t i) const { return i < head ? i : static_cast<int64_t>(vectors) * VecTraits<T>::kElems + i; }
    __device__ __forceinline__ int64_t place(uint32_t vector) const { return head + static_cast<int64_t>(vector) * VecTraits<T>::kElems; }
};

// How many of keys[0 .. n) are larger than `mine`: four neighbouring lanes share the count (all of a warp's lanes call it).
__device__ __forceinline__ int larger_than(const Key* keys, int n, Key mine) {
    int rank = 0;
#pragma unroll 8
    for (int j = threadIdx.x & 3; j < n; j += 4) rank += keys[j] > mine;
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    return rank + __shfl_xor_sync(0xffffffffu, rank, 2);
}

// The k largest of `n` keys in shared memory, in order. All threads call it.
template <int THREADS>
__device__ __forceinline__ void take_largest(const Key* keys, int n, int k, Key* list) {
    for (int base = 0; base < n; base += THREADS / 4) {
        const int i = base + (threadIdx.x >> 2);
        const Key mine = i < n ? keys[i] : 0;
        const int rank = larger_than(keys, n, mine);
        if (i < n && rank < k && mine != 0) list[rank] = mine;
    }
}

// A bound that k of keys[0 .. n) reach and not many more than k + slack (exactly k, but for equal keys, with slack 0); 0 where there are
// fewer than k. All threads call it, `result` is in shared memory. As long as every key has four lanes they count the keys above it;
// more keys are one warp's, which halves the distance between the least and the largest, some seven steps of n / 32 comparisons a lane:
// with n^2 comparisons for them [4096, 50257] bf16, 20 alternatives, took 170 us instead of 141.
template <int THREADS, typename K>
__device__ __forceinline__ K bound_of(const K* keys, int n, int k, int slack, K* result) {
    const int tid = threadIdx.x, lane = tid & 31;
    if (n < k) {
        if (tid == 0) *result = 0;
    } else if (n <= THREADS / 4) {
        const int i = tid >> 2;
        const K mine = i < n ? keys[i] : 0;
        int rank = 0;
#pragma unroll 8
        for (int j = tid & 3; j < n; j += 4) rank += keys[j] > mine || (keys[j] == mine && j < i);
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if ((tid & 3) == 0 && i < n && rank == k - 1) *result = mine;
    } else if (tid < 32) {
        K low = ~K{0}, high = 0;
        for (int i = lane; i < n; i += 32) {
            low = min(low, keys[i]);
            high = max(high, keys[i]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
            high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
        }
        auto reach = [&](K bound) {
            int count = 0;
            for (int i = lane; i < n; i += 32) count += keys[i] >= bound;
            return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(count)));
        };
        if (reach(high) >= k) low = high;
        int count = n;  // that reach low; fewer than k reach high
        while (count > k + slack && high - low > 1) {
            const K middle = low + (high - low) / 2;
            const int c = reach(middle);
            if (c >= k) {
                low = middle;
                count = c;
            } else {
                high = middle;
            }
        }
        if (lane == 0) *result = low;
    }
    __syncthreads();
    return *result;
}

// Threads of an SM that there are registers for: many rows want many (1536 leave each 40), as far as the kernel keeps to them; few rows
// (512 threads) and short ones have no use for more.
template <typename T, bool TOP, int THREADS>
constexpr int kResident = THREADS < 64 || (TOP && THREADS == 512) ? 1024 : TOP && sizeof(T) == 4 ? 1280 : 1536;

// CTAs of a cluster share a row (clusters of 1 to 8, along x): the first one joins them.
template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, kResident<T, TOP, THREADS> / THREADS) logprobs_kernel(const __grid_constant__ LogprobParams<T> p) {
    constexpr int E = VecTraits<T>::kElems, kSlack = 8, kGroups = THREADS < 256 ? THREADS : THREADS / 4, kList = Lists<THREADS>::kKeys, kVectors = Lists<THREADS>::kVectors;
    __shared__ float scratch[3][32];
    __shared__ float joined[4];  // maximum, S, T of this CTA
    __shared__ Key list[TOP ? kList : 1], group[TOP ? THREADS : 1], best[TOP ? MHLO_CUDA_TOP_LOGPROBS_MAX : 1], bound_shared;
    __shared__ uint32_t found_at[TOP ? kVectors : 1], found_order[TOP ? kVectors : 1], order_shared;
    __shared__ int listed, keys_listed;
    grid_dependency_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = 1 << p.log2_parts;
    const uint32_t part = blockIdx.x & (parts - 1);
    const int64_t row = blockIdx.x >> p.log2_parts;
    const Row<T> r(p.x + row * p.row_stride, p.vocab);
    const uint32_t v0 = static_cast<uint32_t>(static_cast<uint64_t>(r.vectors) * part >> p.log2_parts);
    const uint32_t v1 = static_cast<uint32_t>(static_cast<uint64_t>(r.vectors) * (part + 1) >> p.log2_parts);
    const uint4* const vectors = reinterpret_cast<const uint4*>(r.x + r.head);
    const int tid = threadIdx.x;
    const float c = p.scale * 1.4426950408889634f, span = -kLowest / c;

    // this thread's part of the batch of vectors that begins at `base`, with their maxima; returns the largest element
    auto load = [&](uint4* raw, float* largest, uint32_t base, bool has_single, float* single) {
        const bool whole = base + THREADS * kBatch <= v1;  // every batch of a row but its last
        if (whole) {
            const uint4* const at = vectors + base + tid;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) raw[i] = ld_stream16(at + i * THREADS);
        } else {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const uint32_t v = base + tid + i * THREADS;
                raw[i] = v < v1 ? ld_stream16(vectors + v) : all_lowest<T>();
            }
        }
        *single = has_single ? VecTraits<T>::to_float(r.x[r.place_of_single(tid)]) : -INFINITY;
        float most = *single;
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            largest[i] = -INFINITY;
            if (!whole && base + i * THREADS >= v1) continue;
            largest[i] = largest_of<T>(raw[i]);
            most = max_nan(most, largest[i]);
        }
        return most;
    };
    Key bound = 0;
    if (TOP && tid == 0) listed = 0;
    // The bound from the keys of `groups` groups of neighbouring threads (0: none): what k of them reach.
    auto raise_bound = [&](Key mine, int groups, int slack) {
        const int width = THREADS / groups;
        for (int o = 1; o < width; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        if (tid % width == 0) group[tid / width] = mine;
        __syncthreads();
        bound = max(bound, bound_of<THREADS>(group, groups, p.top_k, slack, &bound_shared));
    };
    // An order that k of the list's maxima reach (0: there are fewer): another bound from below.
    auto bound_of_list = [&](int n) { return bound_of<THREADS>(found_order, n, p.top_k, kSlack, &order_shared); };
    auto put = [&](Key key) {
        if (key < bound) return;
        const int at = atomicAdd(&keys_listed, 1);
        if (at < kList) list[at] = key;
    };
    // Elements so far below the maximum that their exponential is 0 are kept above -infinity, so that 0 * -infinity never comes up:
    // 16-bit types two at a time before they are widened, where the type has such a number.
    Floor<T> floor(0.f, 0.f);
    bool by_two = false;
    float m = -INFINITY, s = 0.f, t = 0.f;
    bool first = true;
    int batches = 0;
    for (uint32_t base = v0; first || base < v1; base += THREADS * kBatch) {
        uint4 raw[kBatch];
        float single, largest[kBatch];
        const bool has_single = first && part == 0 && tid < r.singles();
        const float most = load(raw, largest, base, has_single, &single);
        if (most > m) {
            const float delta = fmaxf((m - most) * c, kLowest), f = ex2(delta);
            t = f * fmaf(s, delta, t);
            s *= f;
            m = most;
            floor = Floor<T>(m, span);
            by_two = floor.below() * c >= 100.f;  // 2^-100 of 2^31 elements are still nothing beside the maximum's 1
        }
        if (m == -INFINITY) {  // nothing but -infinities so far, or a NaN
            if (most != most) s = most;
        } else {
            const bool whole = base + THREADS * kBatch <= v1;
            const float2 minus = make_float2(-m, -m), by = make_float2(c, c);
            float2 s2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);
            auto add_vectors = [&](auto two) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    if (!whole && base + i * THREADS >= v1) break;
                    float2 f[E / 2];
                    VecTraits<T>::unpack2(decltype(two)::value ? floor.raise(raw[i]) : raw[i], f);
#pragma unroll
                    for (int e = 0; e < E / 2; ++e) {
                        float2 d = __fmul2_rn(__fadd2_rn(f[e], minus), by);
                        if (!decltype(two)::value) d = make_float2(max_nan(d.x, kLowest), max_nan(d.y, kLowest));
                        const float2 w = make_float2(ex2(d.x), ex2(d.y));
                        s2 = __fadd2_rn(s2, w);
                        t2 = __ffma2_rn(w, d, t2);
                    }
                }
            };
            if (by_two) add_vectors(std::true_type{});
            else add_vectors(std::false_type{});
            if (has_single) {
                const float d = max_nan((single - m) * c, kLowest), w = ex2(d);
                s2.x += w;
                t2.x = fmaf(w, d, t2.x);
            }
            s += s2.x + s2.y;
            t += t2.x + t2.y;
        }

        if constexpr (TOP) {
            if (first) {  // a maximum counts as the last element of its vector: the bound may be less than it could be, never more
                uint32_t place = has_single ? static_cast<uint32_t>(r.place_of_single(tid)) : 0xffffffffu;
#pragma unroll
                for (int i = kBatch - 1; i >= 0; --i) {
                    const uint32_t v = base + tid + i * THREADS;
                    if (v < v1 && (largest[i] == most || largest[i] != largest[i])) place = static_cast<uint32_t>(r.place(v) + E - 1);
                }
                raise_bound(place == 0xffffffffu ? 0 : key_of(most, place), kGroups, kSlack);
            }
            const float least = number_of(static_cast<uint32_t>(bound >> 32));
            if (!(most < least)) {
                uint32_t hits = 0;  // one addition for all of a thread's vectors
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const uint32_t v = base + tid + i * THREADS;
                    // of a vector whose maximum equals the bound's number only places up to the bound's count
                    if (!(largest[i] < least) && v < v1 && (largest[i] != least || static_cast<uint32_t>(r.place(v)) <= ~static_cast<uint32_t>(bound))) hits |= 1u << i;
                }
                if (hits != 0) {
                    int at = atomicAdd(&listed, __popc(hits));
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        if ((hits >> i & 1) == 0) continue;
                        if (at < kVectors) {
                            found_at[at] = base + tid + i * THREADS;
                            found_order[at] = order_of(largest[i]);
                        }
                        ++at;
                    }
                }
            }
        }
        if constexpr (TOP) {  // each time the row has doubled the list, if it has grown, bounds it anew
            ++batches;
            if ((batches & (batches - 1)) == 0 && batches > 1 && base + THREADS * kBatch < v1) {
                __syncthreads();
                const int n = min(listed, kVectors);
                __syncthreads();
                if (n > kVectors / 4) {
                    const uint32_t least = bound_of_list(n);
                    if (least > static_cast<uint32_t>(bound >> 32)) bound = static_cast<Key>(least) << 32;
                }
            }
        }
        first = false;
    }

    int kept = 0;  // keys on the list
    if constexpr (TOP) {
        if (tid == 0) keys_listed = 0;
        __syncthreads();
        const int n = listed;
        if (n <= kVectors) {
            const uint32_t least = bound_of_list(n);
            for (int i = tid; i < n; i += THREADS) {
                if (found_order[i] < least) continue;
                float f[E];
                const uint32_t v = found_at[i];
                VecTraits<T>::unpack(vectors[v], f);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (order_of(f[e]) >= least) put(key_of(f[e], static_cast<uint32_t>(r.place(v) + e)));
            }
            if (part == 0 && tid < r.singles()) {
                const int64_t at = r.place_of_single(tid);
                put(key_of(VecTraits<T>::to_float(r.x[at]), static_cast<uint32_t>(at)));
            }
        }
        __syncthreads();
        kept = keys_listed;
        if (n > kVectors || kept > kList) {
            __syncthreads();
            kept = 0;
            if (tid == 0) keys_listed = 0;
            __syncthreads();
            // a vector a thread, then the elements beside them as if they were vectors of one
            for (uint32_t base = v0; base < v1 + (part == 0 ? THREADS : 0); base += THREADS) {
                const bool singles = base >= v1;  // the last time round
                const uint32_t v = singles ? 0 : base + tid;
                uint4 raw = all_lowest<T>();
                int n = 0;  // elements of this thread
                uint32_t place = 0;
                if (!singles && v < v1) {
                    raw = vectors[v];
                    place = static_cast<uint32_t>(r.place(v));
                    n = E;
                } else if (singles && tid < r.singles()) {
                    place = static_cast<uint32_t>(r.place_of_single(tid));
                    *reinterpret_cast<T*>(&raw) = r.x[place];
                    n = 1;
                }
                auto add = [&]() {
                    float f[E];
                    VecTraits<T>::unpack(raw, f);
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (e < n) put(key_of(f[e], place + e));
                };
                add();
                __syncthreads();
                while (keys_listed > kList) {  // once: then at most k + 1 threads have anything to add (the bound may lie inside a vector)
                    __syncthreads();
                    if (kept > p.top_k) {  // earlier keys, cut to the k largest
                        take_largest<THREADS>(list, kept, p.top_k, best);
                        __syncthreads();
                        if (tid < p.top_k) list[tid] = best[tid];
                        kept = p.top_k;
                    }
                    if (tid == 0) keys_listed = kept;
                    raise_bound(n == 0 ? 0 : key_of(largest_of<T>(raw), place + n - 1), THREADS, 0);
                    add();
                    __syncthreads();
                }
                kept = keys_listed;
                __syncthreads();  // everybody has read it
            }
        }
    }
    const float top = cta_reduce<MaxOp>(m, scratch[0]), from = top == -INFINITY ? 0.f : top;
    const float delta = fmaxf((m - from) * c, kLowest), f = ex2(delta);
    const float all_t = cta_reduce<SumOp>(f * fmaf(s, delta, t), scratch[1]);
    const float all_s = cta_reduce<SumOp>(f * s, scratch[2]);
    if (tid == 0) {
        joined[0] = top;
        joined[1] = all_s;
        joined[2] = all_t;
    }
    if constexpr (TOP) {
        if (tid < MHLO_CUDA_TOP_LOGPROBS_MAX) best[tid] = 0;
        __syncthreads();
        take_largest<THREADS>(list, kept, p.top_k, best);
    }
    if (parts > 1) {
        cluster.sync();
        if (part == 0) {
            if (TOP) {  // the parts' alternatives
                for (int i = tid; i < parts * p.top_k; i += THREADS) list[i] = cluster.map_shared_rank(best, i / p.top_k)[i % p.top_k];
            }
            if (tid == 0) {
                float most = joined[0];
                for (int i = 1; i < parts; ++i) most = fmaxf(most, cluster.map_shared_rank(joined, i)[0]);
                float sum = 0.f, weighted = 0.f;
                for (int i = 0; i < parts; ++i) {
                    const float* other = cluster.map_shared_rank(joined, i);
                    const float move = fmaxf((other[0] - (most == -INFINITY ? 0.f : most)) * c, kLowest), g = ex2(move);
                    weighted += g * fmaf(other[1], move, other[2]);
                    sum += g * other[1];
                }
                scratch[0][0] = most;
                scratch[0][1] = sum;
                scratch[0][2] = weighted;
            }
        }
        cluster.sync();  // no CTA leaves while its shared memory is read
        if (part != 0) return;
        if (tid == 0) {
            joined[0] = scratch[0][0];
            joined[1] = scratch[0][1];
            joined[2] = scratch[0][2];
        }
        if constexpr (TOP) {
            if (tid < MHLO_CUDA_TOP_LOGPROBS_MAX) best[tid] = 0;
            __syncthreads();
            take_largest<THREADS>(list, parts * p.top_k, p.top_k, best);
        }
    }
    __syncthreads();
    const float most = joined[0], sum = most == -INFINITY ? NAN : joined[1], log_s = logf(sum);
    if (tid == 0) {
        if (p.lse) p.lse[row] = most * p.scale + log_s;
        if (p.entropy) p.entropy[row] = log_s - 0.6931471805599453f * (joined[2] / sum);
        if (p.targets) {
            const int64_t id = target_of(p.targets, p.wide_targets, row);
            p.logprobs[row] = id < 0 ? 0.f : id >= p.vocab ? NAN : (VecTraits<T>::to_float(r.x[id]) - most) * p.scale - log_s;
        }
    }
    if (TOP && tid < p.top_k) {
        const uint32_t id = 0xffffffffu - static_cast<uint32_t>(best[tid]);
        p.top_ids[row * p.top_k + tid] = static_cast<int32_t>(id);
        p.top_logprobs[row * p.top_k + tid] = id < p.vocab ? (VecTraits<T>::to_float(r.x[id]) - most) * p.scale - log_s : NAN;
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

// dx = scale (picked - p (all + e (log p + entropy))): one pass, 16 bytes in and out a step. The target is picked as its vector comes
// by; alternatives are few, and their elements are computed once more by a thread each behind the row (their logits are read before
// anything is written: dx may be x).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) logprobs_grad_kernel(const __grid_constant__ GradParams<T> p) {
    constexpr int E = VecTraits<T>::kElems;
    __shared__ float weight[MHLO_CUDA_TOP_LOGPROBS_MAX];
    __shared__ int32_t ids[MHLO_CUDA_TOP_LOGPROBS_MAX];
    const int64_t row = blockIdx.x;
    const Row<T> r(p.x + row * p.row_stride, p.vocab);
    T* const dx = p.dx + row * p.dx_row_stride;
    const int tid = threadIdx.x;
    int64_t target = -1;
    float g = 0.f;
    if (p.g) {
        target = target_of(p.targets, p.wide_targets, row);
        g = target < 0 ? 0.f : target >= p.vocab ? NAN : p.g[row];
    }
    float all = g, own = 0.f;
    int32_t own_id = -1;
    if (p.top_k > 0) {
        if (tid < p.top_k) {
            own_id = p.top_ids[row * p.top_k + tid];
            ids[tid] = own_id;
            weight[tid] = own_id < 0 ? 0.f : own_id >= p.vocab ? NAN : p.t[row * p.top_k + tid];
            if (own_id >= 0 && own_id < p.vocab) own = VecTraits<T>::to_float(r.x[own_id]);
            else own_id = -1;
        }
        __syncthreads();
        for (int k = 0; k < p.top_k; ++k) all += weight[k];
    }
    const float lse = p.lse[row], e = p.e ? p.e[row] : 0.f, h = p.e ? p.entropy[row] : 0.f;
    const float constant = fmaf(e, h, all), minus_scale = -p.scale;
    auto unpicked = [&](float x) {  // scale (-p (all + e (log p + h)))
        const float logp = fmaf(x, p.scale, -lse), low = max_nan(logp, -200.f);
        return ex2(logp * 1.4426950408889634f) * fmaf(e, low, constant) * minus_scale;
    };
    const float picked = g * p.scale;
    const bool together = ((reinterpret_cast<uintptr_t>(r.x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;  // both rows' vectors on the grid
    const uint4* const vectors = reinterpret_cast<const uint4*>(r.x + r.head);
    for (uint32_t base = 0; base < r.vectors; base += THREADS * kBatch) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const uint32_t v = base + tid + i * THREADS;
            if (v < r.vectors) raw[i] = __ldcs(vectors + v);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const uint32_t v = base + tid + i * THREADS;
            if (v >= r.vectors) break;
            float f[E];
            VecTraits<T>::unpack(raw[i], f);
            const int64_t at = target - r.place(v);
#pragma unroll
            for (int k = 0; k < E; ++k) f[k] = unpicked(f[k]);
            if (at >= 0 && at < E) {
#pragma unroll
                for (int k = 0; k < E; ++k) f[k] += at == k ? picked : 0.f;
            }
            T* const y = dx + r.place(v);
            if (together) {
                st_stream16(y, VecTraits<T>::pack(f));
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k) y[k] = VecTraits<T>::from_float(f[k]);
            }
        }
    }
    if (tid < r.singles()) {
        const int64_t i = r.place_of_single(tid);
        dx[i] = VecTraits<T>::from_float(unpicked(VecTraits<T>::to_float(r.x[i])) + (i == target ? picked : 0.f));
    }
    if (p.top_k > 0) {
        __syncthreads();
        if (own_id >= 0) {
            float sum = own_id == target ? g : 0.f;
            for (int k = 0; k < p.top_k; ++k) sum += ids[k] == own_id ? weight[k] : 0.f;
            dx[own_id] = VecTraits<T>::from_float(fmaf(sum, p.scale, unpicked(own)));
        }
    }
}

int check_rows(const char* what, int32_t dtype, const void* x, int64_t row_stride, int64_t rows, int64_t vocab, float scale, const void* targets,
               int32_t target_dtype, int32_t top_k) {
    if (dtype != MHLO_DT_F16 && dtype != MHLO_DT_BF16 && dtype != MHLO_DT_F32) return fail(MHLO_CUDA_UNSUPPORTED, "%s: dtype %d", what, dtype);
    if (rows < 0 || rows > 0x7fffffff || vocab < 1 || vocab > 0x7fffffff || row_stride < vocab)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld rows of %lld logits, %lld apart", what, static_cast<long long>(rows), static_cast<long long>(vocab), static_cast<long long>(row_stride));
    if (!(scale > 0.f) || scale > 1e38f) return fail(MHLO_CUDA_UNSUPPORTED, "%s: the scale has to be positive and at most 1e38", what);  // times log2(e) it is finite
    if (targets && target_dtype != MHLO_DT_I32 && target_dtype != MHLO_DT_I64) return fail(MHLO_CUDA_UNSUPPORTED, "%s: targets of dtype %d (I32 or I64)", what, target_dtype);
    if (top_k < 0 || top_k > MHLO_CUDA_TOP_LOGPROBS_MAX || top_k > vocab) return fail(MHLO_CUDA_UNSUPPORTED, "%s: %d alternatives of %lld", what, top_k, static_cast<long long>(vocab));
    if (rows > 0 && !x) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null logits", what);
    return MHLO_CUDA_OK;
}

// Rows of up to 512 vectors: 4 batches of a warp.
inline bool short_rows(int64_t vocab, int64_t size) { return vocab * size <= 16 * 512; }

// Threads of a row's CTA. What a warp spends on a row beside its elements (joining the threads, the ragged ends) is a few hundred
// instructions, so with rows enough to fill the machine several times a CTA is small: [4096, 50257] bf16 95 us with 512 threads, 82
// with 256, 79 with 128; short rows get a warp each ([32768, 1000] bf16 52 us with 128 threads, 20 with a warp). The
// alternatives' first bound wants a large batch: 256.
template <typename T, bool TOP>
int launch(LogprobParams<T> p, int64_t rows, cudaStream_t stream) {
    // Few long rows are shared by clusters of CTAs, as long as a thread gets two vectors of its own.
    int parts = 1;
    p.log2_parts = 0;
    while (parts < 8 && rows * parts * 2 <= kNumSMs && p.vocab * static_cast<int64_t>(sizeof(T)) >= int64_t{16} * 512 * 2 * parts * 2) {
        parts *= 2;
        ++p.log2_parts;
    }
    if (rows * parts > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "token_logprobs: too many rows");
    const bool shortest = short_rows(p.vocab, sizeof(T)), small = !TOP && rows >= 8 * kNumSMs, large = rows < 2 * kNumSMs;
    const int threads = shortest ? 32 : small ? 128 : large ? 512 : 256;
    const auto kernel = shortest ? logprobs_kernel<T, TOP, 32> : small ? logprobs_kernel<T, TOP, TOP ? 256 : 128> : large ? logprobs_kernel<T, TOP, 512> : logprobs_kernel<T, TOP, 256>;
    const cudaError_t e = launch_dependent(kernel, dim3(static_cast<unsigned>(rows * parts)), dim3(threads), 0, stream, parts, rows * parts < kNumSMs, p);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of token_logprobs failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("token_logprobs");
    return MHLO_CUDA_OK;
}

template <typename T>
int launch_grad(const GradParams<T>& p, int64_t rows, cudaStream_t stream) {
    if (short_rows(p.vocab, sizeof(T))) logprobs_grad_kernel<T, 32><<<static_cast<unsigned>(rows), 32, 0, stream>>>(p);
    else logprobs_grad_kernel<T, 256><<<static_cast<unsigned>(rows), 256, 0, stream>>>(p);
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
        LogprobParams<T> p{static_cast<const T*>(x_dev), row_stride, vocab, scale, targets_dev, target_dtype == MHLO_DT_I64, logprobs_dev, entropy_dev, lse_dev, top_k, top_logprobs_dev, top_ids_dev, 0};
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        return top_k > 0 ? launch<T, true>(p, rows, st) : launch<T, false>(p, rows, st);
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
        GradParams<T> p{static_cast<const T*>(x_dev), row_stride, vocab, scale, targets_dev, target_dtype == MHLO_DT_I64, lse_dev, entropy_dev, grad_logprobs_dev, grad_entropy_dev,
                        grad_top_dev ? top_k : 0, top_ids_dev, grad_top_dev, static_cast<T*>(dx_dev), dx_row_stride};
        return launch_grad<T>(p, rows, static_cast<cudaStream_t>(stream));
    };
    if (dtype == MHLO_DT_F32) return run(float{});
    if (dtype == MHLO_DT_F16) return run(__half{});
    return run(__nv_bfloat16{});
}

}  // extern "C"
