// Attention over packed sequences: entry points, the plan of a batch, and the kernels of what tcgen05 does not take (fp32, rows off the
// 16-byte grid, head dimensions that are no multiple of 8), forward and backward.
#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "packed_attention.cuh"

namespace mhlo {
namespace {

// ---- the plan ---------------------------------------------------------------------------------------------------------------------
// Tiles that meet more than a kLong-th of what a CTA of a full grid would meet altogether go first, longest first, wherever they are from: late in the
// order they would keep one CTA busy when the others are done. The rest goes run by run. The first CTA places the long tiles, each other one
// those of its run of sequences (first tokens inside run_tokens): it counts the tiles in front of its own, then its own by the 128-token
// blocks they meet, scans, and puts them in place. The order of tiles of one length goes by arrival; no result depends on it. Once for all
// layers of a step: 9 us for 32 sequences of 1024 tokens, 11 for 1000 of 500, 130 for 20 000 of 100 (93 and 2546 with a warp to each sequence in turn
// and its share of the sum an atomic addition of its own).
constexpr int kBuckets = 2048, kPlanThreads = 1024, kLong = 16, kAlone = 4;

__device__ __forceinline__ int32_t bucket_of(int32_t tokens) { return kBuckets - 1 - min((tokens - 1) >> 7, kBuckets - 1); }

// Tiles of a list, `step` tokens each, of a sequence of n tokens.
struct TilesOf {
    int32_t n, step;
    bool ascending, causal;  // ascending: later tiles meet more
    __device__ __forceinline__ int32_t all() const { return (n + step - 1) / step; }
    __device__ __forceinline__ int32_t meets(int32_t at) const { return !causal ? n : ascending ? static_cast<int32_t>(min(static_cast<int64_t>(n), static_cast<int64_t>(at) + step)) : n - at; }
    __device__ __forceinline__ unsigned long long sum() const {  // nearly, of what they meet
        return static_cast<unsigned long long>(all()) * (causal ? (static_cast<unsigned long long>(n) + step + 1) / 2 : n);
    }
    __device__ __forceinline__ int32_t above(int32_t most) const {  // how many meet more
        if (n <= most) return 0;
        return !causal ? all() : ascending ? all() - min(all(), most / step) : (n - most + step - 1) / step;
    }
};

__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(PackedArgs a) {
    __shared__ int32_t counts[2][kBuckets];
    __shared__ int32_t sums[2][32], before[2], all[2];
    __shared__ unsigned long long work[2], held;
    __shared__ int32_t lowest, highest;  // rows of the sequences, in whatever order they come
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, run = static_cast<int>(blockIdx.x) - 1;
    const bool causal = a.causal != 0;
    const int32_t steps[2] = {2 * a.half_tokens, kKeyTile};
    for (int i = tid; i < 2 * kBuckets; i += kPlanThreads) counts[0][i] = 0;
    if (tid < 2) before[tid] = all[tid] = 0, work[tid] = 0;
    if (tid == 0) held = 0, lowest = a.tokens, highest = 0;
    __syncthreads();
    const auto sequence = [&](int32_t b, int32_t* first) {  // its tokens
        const int32_t end = a.starts[b + 1];
        *first = a.starts[b];
        return *first < 0 || end > a.tokens || end < *first ? -1 : end - *first;
    };
    unsigned long long met[2] = {0, 0}, tokens_of = 0;
    int32_t low = a.tokens, high = 0;
    for (int32_t b = tid; b < a.seqs; b += kPlanThreads) {
        int32_t first;
        const int32_t n = sequence(b, &first);
        if (n < 0) kv_report(MHLO_CUDA_KV_ERROR_STARTS);
        if (n <= 0) continue;
        tokens_of += static_cast<unsigned long long>(n);
        low = min(low, first);
        high = max(high, first + n);
#pragma unroll
        for (int list = 0; list < 2; ++list) met[list] += TilesOf{n, steps[list], list == 0, causal}.sum();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tokens_of += __shfl_xor_sync(0xffffffffu, tokens_of, o);
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0 && tokens_of > 0) {
        atomicAdd(&held, tokens_of);
        atomicMin(&lowest, low);
        atomicMax(&highest, high);
    }
#pragma unroll
    for (int list = 0; list < 2; ++list) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) met[list] += __shfl_xor_sync(0xffffffffu, met[list], o);
        if (lane == 0 && met[list] > 0) atomicAdd(&work[list], met[list]);
    }
    __syncthreads();
    PlanHeader* const header = static_cast<PlanHeader*>(a.plan);
    if (held > static_cast<unsigned long long>(a.tokens)) {
        // Starts go back, and sequences that lie over one another have more tokens than there are: their tiles could be more than the lists, and 32 bits, hold.
        // A plan without any. Those of fewer tokens altogether fit: a sequence of n tokens has no more than n / step + 1 tiles of a list.
        if (blockIdx.x == 0 && tid == 0) {
            kv_report(MHLO_CUDA_KV_ERROR_STARTS);
            *header = PlanHeader{kPlanMagic, a.tokens, a.q_heads, a.kv_heads, a.causal, 0, 0, 0, 0, a.seqs, {0, 0}};
        }
        return;
    }
    int32_t most[2];  // that tiles of the runs meet
#pragma unroll
    for (int list = 0; list < 2; ++list) most[list] = static_cast<int32_t>(min(work[list] * a.kv_heads / (kLong * kNumSMs), static_cast<unsigned long long>(1) << 30));
    // tiles in front of this CTA's, and of all
    int32_t mine[2] = {0, 0}, total[2] = {0, 0};
    for (int32_t b = tid; b < a.seqs; b += kPlanThreads) {
        int32_t first;
        const int32_t n = sequence(b, &first);
        if (n <= 0) continue;
#pragma unroll
        for (int list = 0; list < 2; ++list) {
            const TilesOf t{n, steps[list], list == 0, causal};
            const int32_t tiles = t.all(), above = t.above(most[list]);
            total[list] += tiles;
            if (run >= 0) mine[list] += above + (first / a.run_tokens < run ? tiles - above : 0);
        }
    }
#pragma unroll
    for (int list = 0; list < 2; ++list) {
        mine[list] = __reduce_add_sync(0xffffffffu, mine[list]);
        total[list] = __reduce_add_sync(0xffffffffu, total[list]);
        if (lane == 0 && total[list] > 0) {
            atomicAdd(&before[list], mine[list]);
            atomicAdd(&all[list], total[list]);
        }
    }
    __syncthreads();
    for (int place = 0; place < 2; ++place) {
        // A lane looks at a sequence, and puts its tiles in place where they are few; a warp takes the longer ones together, one by one.
        for (int32_t base = warp; base < a.seqs; base += kPlanThreads) {
            const int32_t b = base + 32 * lane;
            int32_t of_lane = 0, tokens = 0;
            if (b < a.seqs) tokens = sequence(b, &of_lane);
            const TilesOf of_rows{tokens, steps[0], true, causal}, of_keys{tokens, steps[1], false, causal};
            const bool mine = tokens > 0 && (run >= 0 ? of_lane / a.run_tokens == run : of_rows.above(most[0]) + of_keys.above(most[1]) > 0);
            const bool alone = mine && of_rows.all() + of_keys.all() <= kAlone;
            auto tiles = [&](int32_t first, int32_t n, int32_t from, int32_t every) {
#pragma unroll
                for (int list = 0; list < 2; ++list) {
                    const TilesOf t{n, steps[list], list == 0, causal};
                    for (int64_t z = static_cast<int64_t>(from) * steps[list]; z < n; z += every * steps[list]) {
                        const int32_t at = static_cast<int32_t>(z), meets = t.meets(at);
                        if ((meets > most[list]) != (run < 0)) continue;
                        const int32_t slot = atomicAdd(&counts[list][bucket_of(meets)], 1);
                        if (place == 0) continue;
                        // starts that another stream changes meanwhile may make more tiles than were counted
                        if (static_cast<uint32_t>(slot) < static_cast<uint32_t>(list == 0 ? a.row_capacity : a.key_capacity)) const_cast<int4*>(list == 0 ? a.row_tiles() : a.key_tiles())[slot] = make_int4(first, n, at, 0);
                    }
                }
            };
            if (alone) tiles(of_lane, tokens, 0, 1);
            for (uint32_t rest = __ballot_sync(0xffffffffu, mine && !alone); rest != 0; rest &= rest - 1) {
                const int from = __ffs(rest) - 1;
                tiles(__shfl_sync(0xffffffffu, of_lane, from), __shfl_sync(0xffffffffu, tokens, from), lane, 32);
            }
        }
        __syncthreads();
        if (place == 1) break;
        // exclusive sums over the buckets
        for (int list = 0; list < 2; ++list) {
            const int32_t x = counts[list][2 * tid], y = counts[list][2 * tid + 1];
            int32_t sum = x + y;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t other = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += other;
            }
            if (lane == 31) sums[list][warp] = sum;
            __syncthreads();
            int32_t at = before[list] + sum - x - y;
            for (int w = 0; w < warp; ++w) at += sums[list][w];
            counts[list][2 * tid] = at;
            counts[list][2 * tid + 1] = at + x;
        }
        __syncthreads();
    }
    if (tid == 0 && blockIdx.x == 0)
        *header = PlanHeader{kPlanMagic, a.tokens, a.q_heads, a.kv_heads, a.causal, min(all[0], a.row_capacity), min(all[1], a.key_capacity), min(lowest, highest), highest, a.seqs, {0, 0}};
}

// ---- the general kernels ------------------------------------------------------------------------------------------------------------
// Tiles of 64 x 64, eight warps of 16 rows by 32 columns, on mma.sync with tf32 operands; what the two warps of a row have summed is joined at the end.
// A number of fp32 goes in as two of 11 bits: x = hi + lo + at most 2^-21 |x|, and a product as hi hi + hi lo + lo hi in fp32, so a sum of products is off by
// 5 * 2^-22 of the sum of their sizes at most, beside what fp32 sums round. (Below 2^-115 lo is less than the smallest normal number, and 11 bits are
// what is left; infinities become NaN.) 16-bit numbers are their hi: one product instead of three, or two where the other side is weights.
// A warp's result of one product (scores) is an operand of the next (times values) in the lanes that it lies in, if that takes keys in the order 0 2 4 6 1 3 5 7.
// Operands lie in shared memory in fp32, rows of DP + 4 floats: the 32 numbers that a warp loads at once are in 32 banks by rows and by columns. The side
// that four warps share is taken apart on its way there.
// mma.sync cuts off what does not fit its fp32 result, so a sum goes through it for 16 terms and is added to the whole with a rounding: 2.7e-7 of the result and 6.7e-7 of
// the gradients are errors like those of fp32 arithmetic (3.8e-7; dq 3.9e-7, dk and dv 7.6e-7). 1.0e-6 and 2.2e-6 if the products add up by themselves, for 4 and 9 us less; 2.2e-7 and
// 5.0e-7 if every 8 terms are added, for 3 and 5 us more.
// Nine sequences of up to 500 tokens, 12 heads of 64 in fp32, take 72 us; 95 on the FMA units, whose 4 x 4 elements a thread wait for what shared memory
// hands to registers (128 bytes a clock and SM, twice the clocks of the multiply-adds). Gradients of five of up to 333, 14 heads on 2: 97 us, and 127.
// Four warps of 64 columns, both sides taken apart where they are used, took 82 and 137.
// The keys' kernel in fp32 holds two sums of 32 numbers beside a step's products and spills 204 bytes at 128 registers (364 at 255 for heads of up to 128).
constexpr int kGT = 256, kGRows = 64, kGKeys = 64, kWN = 4;  // kWN: columns of a warp, by 8

template <int DP>
struct General {
    static constexpr int kPitch = DP + 4, kTile = 64 * kPitch, kSteps = DP / 8;
};

struct GeneralParams {
    PackedArgs a;
    PackedTensor q, k, v, o, grad, dq, dk, dv;
    float* lse;
    float2* stats;  // [kv_heads][tokens][group]: -lse log2(e), delta
    float2* largest;  // of each sequence, see PackedCall
    float *grad_norms, *value_norms;  // null, or where the norms of grad's rows (like stats) and of v's ([kv_heads][tokens]) go
    float scale, scale_log2;
    FastDiv by_group;
    int32_t subs;   // tiles of this kernel to an entry of the plan
    int32_t splits; // shares of the rows that see a tile of keys
    float* shares;
};

struct Parts {
    uint32_t hi, lo;
};
// hi is the nearest of 11 bits, halves away from zero; lo the rest's first 11 bits. A NaN of all ones is lost in hi, but not in lo. (cvt.rna.tf32 for both, and
// both sides taken apart where they are used, took twice the instructions.)
template <bool EXACT>
__device__ __forceinline__ Parts parts(float x) {
    if constexpr (EXACT) return {__float_as_uint(x), 0};
    const uint32_t hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    return {hi, __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u};
}
// Of a tile in shared memory whose lo parts, unless it is EXACT, are a tile behind it.
template <int DP, bool EXACT>
__device__ __forceinline__ Parts parts_at(const float* x) {
    return {__float_as_uint(x[0]), EXACT ? 0 : __float_as_uint(x[General<DP>::kTile])};
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c += a b over 8; A, B: whether the numbers are their hi.
template <bool A, bool B>
__device__ __forceinline__ void multiply(float (&c)[4], const Parts (&a)[4], const Parts (&b)[2]) {
    if constexpr (!A) mma_tf32(c, a[0].lo, a[1].lo, a[2].lo, a[3].lo, b[0].hi, b[1].hi);
    if constexpr (!B) mma_tf32(c, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].lo, b[1].lo);
    mma_tf32(c, a[0].hi, a[1].hi, a[2].hi, a[3].hi, b[0].hi, b[1].hi);
}

// What a thread has of a warp's 16 rows x 32 columns: element e of c[n] is row lane / 4 + 8 (e / 2), column 8 n + 2 (lane % 4) + e % 2.
// c = a b^T: 16 rows of a tile by 32 rows of another, over their elements.
template <int DP, bool EXACT>
__device__ __forceinline__ void rows_by_rows(const float* a, const float* b, float (&c)[kWN][4]) {
    constexpr int P = General<DP>::kPitch;
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
    for (int n = 0; n < kWN; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
    a += g * P + t;
    b += g * P + t;
#pragma unroll 1
    for (int k = 0; k < DP; k += 16) {
        const Parts x[2][4] = {{parts<EXACT>(a[k]), parts<EXACT>(a[8 * P + k]), parts<EXACT>(a[k + 4]), parts<EXACT>(a[8 * P + k + 4])},
                               {parts<EXACT>(a[k + 8]), parts<EXACT>(a[8 * P + k + 8]), parts<EXACT>(a[k + 12]), parts<EXACT>(a[8 * P + k + 12])}};
#pragma unroll
        for (int n = 0; n < kWN; ++n) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const Parts y[2] = {parts_at<DP, EXACT>(b + 8 * n * P + k + 8 * h), parts_at<DP, EXACT>(b + 8 * n * P + k + 8 * h + 4)};
                multiply<EXACT, EXACT>(d, x[h], y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) c[n][e] += d[e];
        }
    }
}
// c += w b: a warp's weights, as rows_by_rows leaves them, by 32 rows of a tile.
template <int DP, bool EXACT>
__device__ __forceinline__ void weights_by_rows(const float (&w)[kWN][4], const float* b, float (&c)[DP / 8][4]) {
    constexpr int P = General<DP>::kPitch;
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    b += 2 * t * P + g;
#pragma unroll
    for (int k = 0; k < kWN; k += 2) {
        Parts x[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) x[h][0] = parts<false>(w[k + h][0]), x[h][1] = parts<false>(w[k + h][2]), x[h][2] = parts<false>(w[k + h][1]), x[h][3] = parts<false>(w[k + h][3]);
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
            float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const Parts y[2] = {parts_at<DP, EXACT>(b + 8 * (k + h) * P + 8 * n), parts_at<DP, EXACT>(b + (8 * (k + h) + 1) * P + 8 * n)};
                multiply<false, EXACT>(d, x[h], y);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) c[n][e] += d[e];
        }
    }
}

// 64 rows into shared memory, their lo parts (SPLIT) a tile behind them; row(r): where row r starts, null: zeros (so are the elements behind head_dim).
template <typename T, int DP, bool SPLIT, typename Row>
__device__ __forceinline__ void stage(float* to, int32_t dim, bool vec, Row row) {
    constexpr int P = General<DP>::kPitch, V = VecTraits<T>::kElems;
    if (vec) {
#pragma unroll 4
        for (int i = threadIdx.x; i < 64 * (DP / V); i += kGT) {
            const int r = i / (DP / V), d = i % (DP / V) * V;
            const T* const at = row(r);
            float x[V];
            if (at != nullptr && d < dim) {
                VecTraits<T>::unpack(*reinterpret_cast<const uint4*>(at + d), x);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                float4 v = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
                if constexpr (SPLIT) {
                    const Parts a = parts<false>(v.x), b = parts<false>(v.y), c = parts<false>(v.z), f = parts<false>(v.w);
                    v = make_float4(__uint_as_float(a.hi), __uint_as_float(b.hi), __uint_as_float(c.hi), __uint_as_float(f.hi));
                    *reinterpret_cast<uint4*>(to + General<DP>::kTile + r * P + d + e) = make_uint4(a.lo, b.lo, c.lo, f.lo);
                }
                *reinterpret_cast<float4*>(to + r * P + d + e) = v;
            }
        }
        return;
    }
    for (int i = threadIdx.x; i < 64 * DP; i += kGT) {
        const int r = i / DP, d = i % DP;
        const T* const at = row(r);
        const float x = at != nullptr && d < dim ? VecTraits<T>::to_float(at[d]) : 0.f;
        const Parts part = parts<!SPLIT>(x);
        to[r * P + d] = __uint_as_float(part.hi);
        if (SPLIT) to[General<DP>::kTile + r * P + d] = __uint_as_float(part.lo);
    }
}

// What the second warp of a row has goes to shared memory (add: comes from there, to the first).
template <int N>
__device__ __forceinline__ void leave_sums(float* to, const float (&c)[N][4]) {
#pragma unroll
    for (int i = 0; i < N * 4; ++i) to[i * (kGT / 2) + threadIdx.x % (kGT / 2)] = c[i / 4][i % 4];
}
template <int N>
__device__ __forceinline__ void add_sums(const float* from, float (&c)[N][4]) {
#pragma unroll
    for (int i = 0; i < N * 4; ++i) c[i / 4][i % 4] += from[i * (kGT / 2) + threadIdx.x % (kGT / 2)];
}

// Row i of the two that a thread has a part of.
template <typename T, int DP>
__device__ __forceinline__ void store_row(T* to, int32_t dim, const float (&c)[DP / 8][4], int i, float factor) {
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 8 * n + 2 * (threadIdx.x & 3) + e;
            if (d < dim) to[d] = VecTraits<T>::from_float(c[n][2 * i + e] * factor);
        }
}

// A run of 64 stacked rows: row r of it is token t0 + (r0 + r) / group.
struct RowRun {
    int32_t first, n, head, t0, r0, end;  // end: the entry's rows
    FastDiv by_group;
    __device__ __forceinline__ int32_t token(const PackedArgs&, int32_t r) const { return t0 + static_cast<int32_t>(by_group.div(r0 + r)); }
    __device__ __forceinline__ bool has(const PackedArgs& a, int32_t r) const { return r0 + r < end && token(a, r) < n; }
    __device__ __forceinline__ int32_t of_group(const PackedArgs& a, int32_t r) const { return r0 + r - static_cast<int32_t>(by_group.div(r0 + r)) * a.group; }
    __device__ __forceinline__ int64_t q_head(const PackedArgs& a, int32_t r) const { return head * a.group + of_group(a, r); }
    __device__ __forceinline__ int64_t stat(const PackedArgs& a, int32_t r) const {
        return (static_cast<int64_t>(head) * a.tokens + first + token(a, r)) * a.group + of_group(a, r);
    }
};

template <typename T>
__device__ __forceinline__ T* row_at(const PackedTensor& t, int64_t token, int64_t head) {
    return static_cast<T*>(t.base) + token * t.token + head * t.head;
}

// Item blockIdx.x of a list of `count` entries: (entry, sub, head), heads next to each other. False: none.
__device__ __forceinline__ bool entry_of(const GeneralParams& p, const int4* list, int32_t count, int4* e, int32_t* sub, int32_t* head) {
    const uint32_t i = blockIdx.x, at = i / static_cast<uint32_t>(p.a.kv_heads);
    *head = i - at * p.a.kv_heads;
    const uint32_t entry = at / static_cast<uint32_t>(p.subs);
    *sub = at - entry * p.subs;
    if (entry >= static_cast<uint32_t>(count)) return false;
    *e = list[entry];
    if (p.a.inside(*e)) return true;
    if (threadIdx.x == 0) kv_report(MHLO_CUDA_KV_ERROR_PLAN);
    return false;
}

// Over the four lanes that share rows.
__device__ __forceinline__ float most_of_row(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float sum_of_row(float x) {
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kGT, DP == 64 ? 2 : 1) packed_general_kernel(const __grid_constant__ GeneralParams p, int32_t vec) {
    using G = General<DP>;
    extern __shared__ __align__(16) float smem[];
    constexpr bool kExact = !std::is_same<T, float>::value;
    float *const q = smem, *const k = q + G::kTile, *const v = k + (kExact ? 1 : 2) * G::kTile;
    const PackedArgs& a = p.a;
    const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
    int4 e;
    int32_t sub, head;
    if (!a.matches(h) || !entry_of(p, a.row_tiles(), h.row_tiles, &e, &sub, &head)) return;
    const RowRun run{e.x, e.y, head, e.z, sub * kGRows, 2 * a.half_tokens * a.group, p.by_group};
    if (!run.has(a, 0)) return;
    const int row0 = threadIdx.x / 32 % 4 * 16, column0 = threadIdx.x / 128 * 32, g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    stage<T, DP, false>(q, a.head_dim, vec, [&](int r) -> const T* { return run.has(a, r) ? row_at<const T>(p.q, run.first + run.token(a, r), run.q_head(a, r)) : nullptr; });
    float acc[G::kSteps][4], most[2], total[2];
    int32_t last[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        most[i] = -INFINITY;
        total[i] = 0.f;
        last[i] = a.causal ? min(run.n - 1, run.token(a, row0 + g + 8 * i)) : run.n - 1;
    }
#pragma unroll
    for (int n = 0; n < G::kSteps; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
    const int32_t seen = a.causal ? min(run.n, run.token(a, kGRows - 1) + 1) : run.n;
    for (int32_t key0 = 0; key0 < seen; key0 += kGKeys) {
        auto key_row = [&](const PackedTensor& x, int r) -> const T* { return key0 + r < run.n ? row_at<const T>(x, run.first + key0 + r, head) : nullptr; };
        __syncthreads();
        stage<T, DP, !kExact>(k, a.head_dim, vec, [&](int r) { return key_row(p.k, r); });
        stage<T, DP, !kExact>(v, a.head_dim, vec, [&](int r) { return key_row(p.v, r); });
        __syncthreads();
        float s[kWN][4];
        rows_by_rows<DP, kExact>(q + row0 * G::kPitch, k + column0 * G::kPitch, s);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float m = -INFINITY;
#pragma unroll
            for (int n = 0; n < kWN; ++n)
#pragma unroll
                for (int e = 2 * i; e < 2 * i + 2; ++e) {
                    s[n][e] = key0 + column0 + 8 * n + 2 * t + (e & 1) <= last[i] ? s[n][e] * p.scale_log2 : -INFINITY;
                    m = fmaxf(m, s[n][e]);
                }
            m = fmaxf(most[i], most_of_row(m));
            const float shift = m == -INFINITY ? 0.f : m, keep = exp2f(most[i] - shift);
            most[i] = m;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < kWN; ++n)
#pragma unroll
                for (int e = 2 * i; e < 2 * i + 2; ++e) sum += s[n][e] = exp2f(s[n][e] - shift);
            total[i] = total[i] * keep + sum;  // of this thread's columns
#pragma unroll
            for (int n = 0; n < G::kSteps; ++n) acc[n][2 * i] *= keep, acc[n][2 * i + 1] *= keep;
        }
        weights_by_rows<DP, kExact>(s, v + column0 * G::kPitch, acc);
    }
    float4* const of_rows = reinterpret_cast<float4*>(smem + G::kTile);
    __syncthreads();
    if (column0 > 0) {
        leave_sums(smem, acc);
        of_rows[threadIdx.x % (kGT / 2)] = make_float4(most[0], total[0], most[1], total[1]);
    }
    __syncthreads();
    if (column0 > 0) return;
    const float4 other = of_rows[threadIdx.x];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float m1 = i == 0 ? other.x : other.z, t1 = i == 0 ? other.y : other.w, m = fmaxf(most[i], m1), shift = m == -INFINITY ? 0.f : m;
        const float keep = exp2f(most[i] - shift), take = exp2f(m1 - shift);
#pragma unroll
        for (int c = 0; c < G::kSteps * 2; ++c) {
            const int n = c / 2, at = 2 * i + c % 2;
            acc[n][at] = acc[n][at] * keep + smem[(n * 4 + at) * (kGT / 2) + threadIdx.x] * take;
        }
        most[i] = m;
        total[i] = sum_of_row(total[i] * keep + t1 * take);
        const int32_t r = row0 + g + 8 * i;
        if (!run.has(a, r)) continue;
        const int64_t token = run.first + run.token(a, r), q_head = run.q_head(a, r);
        store_row<T, DP>(row_at<T>(p.o, token, q_head), a.head_dim, acc, i, total[i] == 0.f ? 0.f : 1.f / total[i]);
        if (t == 0 && p.lse != nullptr) p.lse[token * a.q_heads + q_head] = total[i] == 0.f ? -INFINITY : (most[i] + log2f(total[i])) * 0.6931471805599453f;
    }
}

// What the backward half needs of a row: -lse log2(e) and delta = grad . o; f16 on tcgen05: the norms of grad's rows and of v's, 0 for those that are not finite. LANES of a warp to a row,
// kStatsRows rows at once, and four CTAs to an SM, whose loads run under the others' sums (3 sequences of up to 8192 tokens, 32 heads of 128, bf16: 44 us, 5.6
// TB/s; four rows and two CTAs, which the registers of four rows take, 77; one row 77; f16 with norms, 32 x 1024 tokens of 12 heads of 64: 36 us and 45).
constexpr int kStatsThreads = 256, kStatsRows = 2;
template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(kStatsThreads, 4) packed_stats_kernel(const __grid_constant__ GeneralParams p, FastDiv by_heads, FastDiv by_kv_heads, FastDiv by_group) {
    const PackedArgs& a = p.a;
    constexpr int V = VecTraits<T>::kElems;
    const int lane = threadIdx.x % LANES;
    grid_dependency_wait();
    grid_dependency_release();
    const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
    if (!a.matches(h, false) || h.end <= h.first) return;
    const uint32_t first = (blockIdx.x * kStatsThreads + threadIdx.x) / LANES, step = gridDim.x * (kStatsThreads / LANES);
    auto norm_of = [](float squares) { return squares <= 3.4028235e38f ? sqrtf(squares) : 0.f; };
    auto sum_lanes = [&](float v) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    // this lane's elements of a row
    auto get = [&](const T* row, float* x) {
        if constexpr (VEC) {
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (lane * V < a.head_dim) raw = ld_stream16(row + lane * V);
            VecTraits<T>::unpack(raw, x);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = lane * V + e < a.head_dim ? VecTraits<T>::to_float(row[lane * V + e]) : 0.f;
        }
    };
    const uint32_t from = static_cast<uint32_t>(h.first) * a.q_heads, end = static_cast<uint32_t>(h.end) * a.q_heads;
    // rows of a warp's lanes go past the end together
    for (uint32_t base = from + first - first % (32 / LANES); base < end; base += kStatsRows * step) {
        float o[kStatsRows][V], g[kStatsRows][V], lse[kStatsRows];
        uint32_t token[kStatsRows], head[kStatsRows];
#pragma unroll
        for (int r = 0; r < kStatsRows; ++r) {
            const uint32_t row = min(base + r * step + first % (32 / LANES), end - 1);
            by_heads.divmod(row, &token[r], &head[r]);
            get(row_at<const T>(p.o, token[r], head[r]), o[r]);
            get(row_at<const T>(p.grad, token[r], head[r]), g[r]);
            lse[r] = p.lse[row];
        }
#pragma unroll
        for (int r = 0; r < kStatsRows; ++r) {
            float sum = 0.f, squares = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sum = fmaf(o[r][e], g[r][e], sum);
                squares = fmaf(g[r][e], g[r][e], squares);
            }
            sum = sum_lanes(sum);
            if (p.grad_norms != nullptr) squares = sum_lanes(squares);
            if (lane == 0 && base + r * step + first % (32 / LANES) < end) {
                const uint32_t kv = by_group.div(head[r]);
                const int64_t at = (static_cast<int64_t>(kv) * a.tokens + token[r]) * a.group + head[r] - kv * a.group;
                p.stats[at] = make_float2(-lse[r] * 1.4426950408889634f, sum);
                if (p.grad_norms != nullptr) p.grad_norms[at] = norm_of(squares);
            }
        }
    }
    if (p.grad_norms == nullptr) return;
    const uint32_t v_from = static_cast<uint32_t>(h.first) * a.kv_heads, v_end = static_cast<uint32_t>(h.end) * a.kv_heads;
    for (uint32_t base = v_from + first - first % (32 / LANES); base < v_end; base += kStatsRows * step) {
        float x[kStatsRows][V];
        uint32_t token[kStatsRows], head[kStatsRows];
#pragma unroll
        for (int r = 0; r < kStatsRows; ++r) {
            by_kv_heads.divmod(min(base + r * step + first % (32 / LANES), v_end - 1), &token[r], &head[r]);
            get(row_at<const T>(p.v, token[r], head[r]), x[r]);
        }
#pragma unroll
        for (int r = 0; r < kStatsRows; ++r) {
            float squares = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) squares = fmaf(x[r][e], x[r][e], squares);
            squares = sum_lanes(squares);
            if (lane == 0 && base + r * step + first % (32 / LANES) < v_end) {
                const int64_t at = static_cast<int64_t>(head[r]) * a.tokens + token[r];
                p.value_norms[at] = norm_of(squares);
                p.largest[at] = make_float2(0.f, 0.f);
            }
        }
    }
}

// The largest of those norms in each sequence, by head of keys: a warp to each tile of query rows. (The backward kernels themselves over all rows of the sequence, per item: 18 of
// 167 and 15 of 142 us for 32 x 1024 tokens, 12 heads of 64.)
__global__ void __launch_bounds__(256) packed_largest_kernel(const __grid_constant__ GeneralParams p) {
    const PackedArgs& a = p.a;
    const int lane = threadIdx.x & 31;
    grid_dependency_wait();
    grid_dependency_release();
    const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
    if (!a.matches(h, false)) return;
    const int64_t items = static_cast<int64_t>(h.row_tiles) * a.kv_heads;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); item < items; item += static_cast<int64_t>(gridDim.x) * 8) {
        const int64_t entry = item / a.kv_heads, head = item - entry * a.kv_heads;
        const int4 e = a.row_tiles()[entry];
        if (!a.inside(e)) continue;
        const int32_t tokens = min(e.y - e.z, 2 * a.half_tokens);
        const int64_t at = head * a.tokens + e.x + e.z;
        float g = 0.f, v = 0.f;
#pragma unroll 8
        for (int32_t i = lane; i < tokens * a.group; i += 32) g = fmaxf(g, p.grad_norms[at * a.group + i]);
#pragma unroll 4
        for (int32_t i = lane; i < tokens; i += 32) v = fmaxf(v, p.value_norms[at + i]);
        // bits of numbers that are not negative have the numbers' order
        const uint32_t most_g = __reduce_max_sync(0xffffffffu, __float_as_uint(g)), most_v = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
        if (lane == 0) {
            uint32_t* const to = reinterpret_cast<uint32_t*>(p.largest + head * a.tokens + e.x);
            atomicMax(to, most_g);
            atomicMax(to + 1, most_v);
        }
    }
}

// Sums of the shares of dk and dv, in order; four elements a thread (ANY: one).
template <typename T, bool ANY>
__global__ void __launch_bounds__(256) packed_join_kernel(const __grid_constant__ GeneralParams p, FastDiv by_dim, FastDiv by_heads) {
    constexpr int W = ANY ? 1 : 4;
    const PackedArgs& a = p.a;
    grid_dependency_wait();
    const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
    if (!a.matches(h, false)) return;
    const int64_t all = static_cast<int64_t>(a.tokens) * a.kv_heads * a.head_dim;
    const uint32_t from = static_cast<uint32_t>(h.first) * a.kv_heads * (a.head_dim / W), end = static_cast<uint32_t>(h.end) * a.kv_heads * (a.head_dim / W);
    for (uint32_t i = from + blockIdx.x * 256 + threadIdx.x; i < end; i += gridDim.x * 256) {
        uint32_t row, d, token, head;
        by_dim.divmod(i, &row, &d);
        by_heads.divmod(row, &token, &head);
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const float* const at = p.shares + which * all + static_cast<int64_t>(i) * W;
            float sum[W];
#pragma unroll
            for (int e = 0; e < W; ++e) sum[e] = 0.f;
#pragma unroll 4
            for (int32_t s = 0; s < p.splits; ++s) {
                if constexpr (ANY) {
                    sum[0] += at[2 * s * all];
                } else {
                    const float4 v = *reinterpret_cast<const float4*>(at + 2 * s * all);
                    sum[0] += v.x, sum[1] += v.y, sum[2] += v.z, sum[3] += v.w;
                }
            }
            T* const to = row_at<T>(which == 0 ? p.dk : p.dv, token, head) + d * W;
#pragma unroll
            for (int e = 0; e < W; ++e) to[e] = VecTraits<T>::from_float(sum[e]);
        }
    }
}

// Gradients of keys and values: 64 keys, all rows that see them.
template <typename T, int DP>
__global__ void __launch_bounds__(kGT, DP == 64 ? 2 : 1) packed_general_key_grads_kernel(const __grid_constant__ GeneralParams p, int32_t vec) {
    using G = General<DP>;
    constexpr bool kExact = !std::is_same<T, float>::value;
    extern __shared__ __align__(16) float smem[];
    __shared__ float2 stats[kGRows];
    __shared__ int32_t last[kGRows];  // the last key that a row sees, -1: none
    float *const k = smem, *const v = k + G::kTile, *const q = v + G::kTile, *const grad = q + (kExact ? 1 : 2) * G::kTile;
    const PackedArgs& a = p.a;
    const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
    int4 e;
    int32_t sub, head;
    if (!a.matches(h) || !entry_of(p, a.key_tiles(), h.key_tiles, &e, &sub, &head)) return;
    const int32_t split = sub >> 1, key0 = e.z + (sub & 1) * kGKeys;
    if (key0 >= e.y) return;
    const int tid = threadIdx.x, row0 = tid / 32 % 4 * 16, column0 = tid / 128 * 32, g = (tid & 31) >> 2, t = tid & 3;
    auto key_row = [&](const PackedTensor& x, int r) -> const T* { return key0 + r < e.y ? row_at<const T>(x, e.x + key0 + r, head) : nullptr; };
    stage<T, DP, false>(k, a.head_dim, vec, [&](int r) { return key_row(p.k, r); });
    stage<T, DP, false>(v, a.head_dim, vec, [&](int r) { return key_row(p.v, r); });
    float dk[G::kSteps][4], dv[G::kSteps][4];
#pragma unroll
    for (int n = 0; n < G::kSteps; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) dk[n][c] = dv[n][c] = 0.f;
    const int32_t rows = e.y * a.group, first_row = a.causal ? key0 * a.group : 0;
    const int64_t blocks = (rows - first_row + kGRows - 1) / kGRows;
    const int32_t share0 = first_row + static_cast<int32_t>(blocks * split / p.splits) * kGRows, share1 = first_row + static_cast<int32_t>(blocks * (split + 1) / p.splits) * kGRows;
    for (int32_t r0 = share0; r0 < min(rows, share1); r0 += kGRows) {
        const RowRun run{e.x, e.y, head, 0, r0, rows, p.by_group};
        __syncthreads();
        auto query_row = [&](const PackedTensor& x, int r) -> const T* { return run.has(a, r) ? row_at<const T>(x, run.first + run.token(a, r), run.q_head(a, r)) : nullptr; };
        stage<T, DP, !kExact>(q, a.head_dim, vec, [&](int r) { return query_row(p.q, r); });
        stage<T, DP, !kExact>(grad, a.head_dim, vec, [&](int r) { return query_row(p.grad, r); });
        if (tid < kGRows) {
            const bool has = run.has(a, tid);
            stats[tid] = has ? p.stats[run.stat(a, tid)] : make_float2(0.f, 0.f);
            last[tid] = !has ? -1 : a.causal ? min(run.token(a, tid), e.y - 1) : e.y - 1;
        }
        __syncthreads();
        float s[kWN][4], ds[kWN][4];
        rows_by_rows<DP, kExact>(k + row0 * G::kPitch, q + column0 * G::kPitch, s);
#pragma unroll
        for (int n = 0; n < kWN; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int column = column0 + 8 * n + 2 * t + (c & 1);
                s[n][c] = key0 + row0 + g + 8 * (c >> 1) <= last[column] ? exp2f(fmaf(s[n][c], p.scale_log2, stats[column].x)) : 0.f;
            }
        weights_by_rows<DP, kExact>(s, grad + column0 * G::kPitch, dv);
        rows_by_rows<DP, kExact>(v + row0 * G::kPitch, grad + column0 * G::kPitch, ds);
#pragma unroll
        for (int n = 0; n < kWN; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int column = column0 + 8 * n + 2 * t + (c & 1);
                ds[n][c] = key0 + row0 + g + 8 * (c >> 1) <= last[column] ? s[n][c] * (ds[n][c] - stats[column].y) : 0.f;
            }
        weights_by_rows<DP, kExact>(ds, q + column0 * G::kPitch, dk);
    }
    __syncthreads();
    if (column0 > 0) {
        leave_sums(q, dk);
        leave_sums(grad, dv);
    }
    __syncthreads();
    if (column0 > 0) return;
    add_sums(q, dk);
    add_sums(grad, dv);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int32_t key = key0 + row0 + g + 8 * i;
        if (key >= e.y) continue;
        if (p.splits > 1) {
            float* const to = p.shares + ((static_cast<int64_t>(split) * 2 * a.tokens + e.x + key) * a.kv_heads + head) * a.head_dim;
            store_row<float, DP>(to, a.head_dim, dk, i, p.scale);
            store_row<float, DP>(to + static_cast<int64_t>(a.tokens) * a.kv_heads * a.head_dim, a.head_dim, dv, i, 1.f);
            continue;
        }
        store_row<T, DP>(row_at<T>(p.dk, e.x + key, head), a.head_dim, dk, i, p.scale);
        store_row<T, DP>(row_at<T>(p.dv, e.x + key, head), a.head_dim, dv, i, 1.f);
    }
}

// Gradients of queries: 64 rows, all keys that they see.
template <typename T, int DP>
__global__ void __launch_bounds__(kGT, DP == 64 ? 2 : 1) packed_general_query_grads_kernel(const __grid_constant__ GeneralParams p, int32_t vec) {
    using G = General<DP>;
    constexpr bool kExact = !std::is_same<T, float>::value;
    extern __shared__ __align__(16) float smem[];
    float *const q = smem, *const grad = q + G::kTile, *const k = grad + G::kTile, *const v = k + (kExact ? 1 : 2) * G::kTile;
    const PackedArgs& a = p.a;
    const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
    int4 e;
    int32_t sub, head;
    if (!a.matches(h) || !entry_of(p, a.row_tiles(), h.row_tiles, &e, &sub, &head)) return;
    const RowRun run{e.x, e.y, head, e.z, sub * kGRows, 2 * a.half_tokens * a.group, p.by_group};
    if (!run.has(a, 0)) return;
    const int tid = threadIdx.x, row0 = tid / 32 % 4 * 16, column0 = tid / 128 * 32, g = (tid & 31) >> 2, t = tid & 3;
    auto query_row = [&](const PackedTensor& x, int r) -> const T* { return run.has(a, r) ? row_at<const T>(x, run.first + run.token(a, r), run.q_head(a, r)) : nullptr; };
    stage<T, DP, false>(q, a.head_dim, vec, [&](int r) { return query_row(p.q, r); });
    stage<T, DP, false>(grad, a.head_dim, vec, [&](int r) { return query_row(p.grad, r); });
    float2 stats[2];
    int32_t last[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int32_t r = row0 + g + 8 * i;
        const bool has = run.has(a, r);
        stats[i] = has ? p.stats[run.stat(a, r)] : make_float2(0.f, 0.f);
        last[i] = !has ? -1 : a.causal ? min(run.token(a, r), run.n - 1) : run.n - 1;
    }
    float dq[G::kSteps][4];
#pragma unroll
    for (int n = 0; n < G::kSteps; ++n) dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;
    const int32_t seen = a.causal ? min(run.n, run.token(a, kGRows - 1) + 1) : run.n;
    for (int32_t key0 = 0; key0 < seen; key0 += kGKeys) {
        __syncthreads();
        auto key_row = [&](const PackedTensor& x, int r) -> const T* { return key0 + r < run.n ? row_at<const T>(x, run.first + key0 + r, head) : nullptr; };
        stage<T, DP, !kExact>(k, a.head_dim, vec, [&](int r) { return key_row(p.k, r); });
        stage<T, DP, !kExact>(v, a.head_dim, vec, [&](int r) { return key_row(p.v, r); });
        __syncthreads();
        float s[kWN][4], ds[kWN][4];
        rows_by_rows<DP, kExact>(q + row0 * G::kPitch, k + column0 * G::kPitch, s);
        rows_by_rows<DP, kExact>(grad + row0 * G::kPitch, v + column0 * G::kPitch, ds);
#pragma unroll
        for (int n = 0; n < kWN; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float2 stat = stats[c >> 1];
                ds[n][c] = key0 + column0 + 8 * n + 2 * t + (c & 1) <= last[c >> 1] ? exp2f(fmaf(s[n][c], p.scale_log2, stat.x)) * (ds[n][c] - stat.y) : 0.f;
            }
        weights_by_rows<DP, kExact>(ds, k + column0 * G::kPitch, dq);
    }
    __syncthreads();
    if (column0 > 0) leave_sums(k, dq);
    __syncthreads();
    if (column0 > 0) return;
    add_sums(k, dq);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int32_t r = row0 + g + 8 * i;
        if (run.has(a, r)) store_row<T, DP>(row_at<T>(p.dq, run.first + run.token(a, r), run.q_head(a, r)), a.head_dim, dq, i, p.scale);
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------

template <typename T>
bool vectors(const PackedTensor& t, int32_t dim) {
    constexpr int V = VecTraits<T>::kElems;
    return aligned16(t.base) && t.token % V == 0 && t.head % V == 0 && dim % V == 0;
}

GeneralParams general_params(const PackedCall& c) {
    GeneralParams p;
    p.a = c.a;
    p.q = c.q, p.k = c.k, p.v = c.v, p.o = c.o, p.grad = c.grad, p.dq = c.dq, p.dk = c.dk, p.dv = c.dv;
    p.lse = c.lse;
    p.stats = c.scratch ? c.stats() : nullptr;
    p.largest = nullptr;
    p.grad_norms = p.value_norms = nullptr;
    p.by_group = FastDiv(static_cast<uint32_t>(c.a.group));
    p.splits = 1;
    p.shares = c.scratch ? c.shares() : nullptr;
    p.scale = c.scale;
    p.scale_log2 = c.scale * 1.4426950408889634f;
    p.subs = 0;
    return p;
}

template <typename K>
int launch_general(const char* what, K kernel, GeneralParams p, int32_t subs, int64_t entries, int tiles, int dp, int32_t vec, std::atomic<bool> (&allowed)[64],
                   cudaStream_t stream) {
    const int bytes = tiles * 64 * (dp + 4) * 4;
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), bytes, allowed)) return st;
    p.subs = subs;
    kernel<<<static_cast<unsigned>(entries * subs * p.a.kv_heads), kGT, bytes, stream>>>(p, vec);
    MHLO_CUDA_CHECK_LAUNCH(what);
    return MHLO_CUDA_OK;
}

// Two CTAs to an SM, twice over.
int32_t key_splits_general(const PackedArgs& a) { return key_splits(static_cast<int64_t>(a.key_capacity) * (kKeyTile / kGKeys) * a.kv_heads, 4 * kNumSMs); }

int32_t row_subs(const PackedArgs& a) { return (2 * a.half_tokens * a.group + kGRows - 1) / kGRows; }

template <typename T, int DP>
int forward(const PackedCall& c, cudaStream_t stream) {
    static std::atomic<bool> allowed[64];
    const int32_t vec = vectors<T>(c.q, c.a.head_dim) && vectors<T>(c.k, c.a.head_dim) && vectors<T>(c.v, c.a.head_dim);
    return launch_general("packed_attention", packed_general_kernel<T, DP>, general_params(c), row_subs(c.a), c.a.row_capacity, std::is_same<T, float>::value ? 5 : 3, DP, vec, allowed, stream);
}

template <typename T, int DP>
int backward(const PackedCall& c, cudaStream_t stream) {
    static std::atomic<bool> allowed_keys[64], allowed_queries[64];
    const int32_t vec = vectors<T>(c.q, c.a.head_dim) && vectors<T>(c.k, c.a.head_dim) && vectors<T>(c.v, c.a.head_dim) && vectors<T>(c.grad, c.a.head_dim);
    GeneralParams p = general_params(c);
    p.splits = key_splits_general(c.a);
    if (int st = launch_general("packed_attention_grad", packed_general_key_grads_kernel<T, DP>, p, kKeyTile / kGKeys * p.splits, c.a.key_capacity, std::is_same<T, float>::value ? 6 : 4, DP, vec, allowed_keys, stream))
        return st;
    if (p.splits > 1)
        if (int st = packed_join_shares(c, p.splits, stream)) return st;
    return launch_general("packed_attention_grad", packed_general_query_grads_kernel<T, DP>, general_params(c), row_subs(c.a), c.a.row_capacity, std::is_same<T, float>::value ? 6 : 4, DP, vec, allowed_queries, stream);
}

template <typename T, int LANES, bool VEC>
int stats_of(const PackedCall& c, bool norms, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(c.a.tokens) * c.a.q_heads, of_cta = kStatsRows * (kStatsThreads / LANES);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((rows + of_cta - 1) / of_cta, 8 * kNumSMs));
    GeneralParams p = general_params(c);
    if (norms) p.largest = c.largest(), p.grad_norms = c.grad_norms(), p.value_norms = c.value_norms();
    const auto by = [](int32_t n) { return FastDiv(static_cast<uint32_t>(n)); };
    cudaError_t e = launch_dependent(packed_stats_kernel<T, LANES, VEC>, dim3(grid), dim3(kStatsThreads), 0, stream, 1, grid < kNumSMs, p, by(c.a.q_heads), by(c.a.kv_heads),
                                           by(c.a.group));
    if (e == cudaSuccess && norms) {
        const int64_t items = static_cast<int64_t>(c.a.row_capacity) * c.a.kv_heads;
        e = launch_dependent(packed_largest_kernel, dim3(static_cast<unsigned>(std::min<int64_t>((items + 7) / 8, 8 * kNumSMs))), dim3(256), 0, stream, 1, true, p);
    }
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of packed_attention_grad failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("packed_attention_grad");
    return MHLO_CUDA_OK;
}
template <typename T>
int stats(const PackedCall& c, bool norms, cudaStream_t stream) {
    constexpr int V = VecTraits<T>::kElems, kFew = 64 / V, kMany = 128 / V;
    const bool vec = vectors<T>(c.o, c.a.head_dim) && vectors<T>(c.grad, c.a.head_dim) && vectors<T>(c.v, c.a.head_dim), few = c.a.head_dim <= 64;
    if (vec) return few ? stats_of<T, kFew, true>(c, norms, stream) : stats_of<T, kMany, true>(c, norms, stream);
    return few ? stats_of<T, kFew, false>(c, norms, stream) : stats_of<T, kMany, false>(c, norms, stream);
}

template <typename T>
int join_shares(const PackedCall& c, int32_t splits, cudaStream_t stream) {
    GeneralParams p = general_params(c);
    p.splits = splits;
    const bool any = c.a.head_dim % 4 != 0;
    const int64_t threads = static_cast<int64_t>(c.a.tokens) * c.a.kv_heads * c.a.head_dim / (any ? 1 : 4);
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>((threads + 255) / 256, 8 * kNumSMs)));
    const FastDiv by_dim(static_cast<uint32_t>(c.a.head_dim / (any ? 1 : 4))), by_heads(static_cast<uint32_t>(c.a.kv_heads));
    const cudaError_t e = any ? launch_dependent(packed_join_kernel<T, true>, grid, dim3(256), 0, stream, 1, true, p, by_dim, by_heads)
                              : launch_dependent(packed_join_kernel<T, false>, grid, dim3(256), 0, stream, 1, true, p, by_dim, by_heads);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of packed_attention_grad failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("packed_attention_grad");
    return MHLO_CUDA_OK;
}

template <typename F>
int by_type(const PackedCall& c, F f) {
    switch (c.dtype) {
        case MHLO_DT_F32: return f(float{});
        case MHLO_DT_F16: return f(__half{});
        default: return f(__nv_bfloat16{});
    }
}

// A call's layout may keep it from the tensor cores: the larger of both.
int64_t grad_scratch_bytes(int32_t dtype, const PackedArgs& a, int64_t dim) {
    const int64_t splits = std::max(key_splits_general(a), dtype == MHLO_DT_F32 ? 1 : key_splits_tc(a));
    const int64_t shares = splits > 1 ? splits * 2 * a.tokens * a.kv_heads * dim * 4 : 0;
    return (static_cast<int64_t>(a.tokens) * a.q_heads + 1) / 2 * 2 * static_cast<int64_t>(sizeof(float2)) + packed_norms(dtype, a) * 4 + shares;
}

// What the host can see of a batch.
int packed_args(const char* what, const mhlo_cuda_packed_batch* b, PackedArgs* out) {
    if (!b) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null batch", what);
    if (b->seqs < 0 || b->seqs > (1 << 24) || b->tokens < 0 || b->tokens > (1 << 30))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld sequences, %lld tokens", what, static_cast<long long>(b->seqs), static_cast<long long>(b->tokens));
    if (b->kv_heads < 1 || b->kv_heads > 65535 || b->q_heads < 1 || b->q_heads > 65535 || b->q_heads % b->kv_heads != 0)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld query heads on %lld heads of keys", what, static_cast<long long>(b->q_heads), static_cast<long long>(b->kv_heads));
    if (b->tokens * b->q_heads > (int64_t{1} << 30))  // rows, and a tile behind the last one, are numbered in 32 bits
        return fail(MHLO_CUDA_UNSUPPORTED, "%s: %lld tokens of %lld heads (up to 2^30 rows)", what, static_cast<long long>(b->tokens), static_cast<long long>(b->q_heads));
    out->starts = b->starts;
    out->plan = b->plan;
    out->seqs = static_cast<int32_t>(b->seqs);
    out->tokens = static_cast<int32_t>(b->tokens);
    out->q_heads = static_cast<int32_t>(b->q_heads);
    out->kv_heads = static_cast<int32_t>(b->kv_heads);
    out->group = out->q_heads / out->kv_heads;
    out->head_dim = 0;
    out->causal = b->causal != 0;
    out->half_tokens = std::max(1, kRows / out->group);
    const int64_t most = std::min(b->seqs, b->tokens);  // sequences that have tokens
    out->row_capacity = static_cast<int32_t>(b->tokens / (2 * out->half_tokens) + most);
    out->key_capacity = static_cast<int32_t>(b->tokens / kKeyTile + most);
    // 16-bit keys and values of 128 elements a head: a quarter of L2
    out->run_tokens = std::max<int32_t>(128, (32 << 20) / (512 * out->kv_heads));
    // items of the general kernels, the finest
    const int64_t finest = std::max<int64_t>(static_cast<int64_t>(out->row_capacity) * std::max(2, row_subs(*out)), 2 * static_cast<int64_t>(out->key_capacity) * key_splits_general(*out)) * out->kv_heads;
    if (finest > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "%s: too many tiles", what);
    return MHLO_CUDA_OK;
}

int64_t plan_bytes(const PackedArgs& a) { return static_cast<int64_t>(sizeof(PlanHeader)) + 16 * (static_cast<int64_t>(a.row_capacity) + a.key_capacity); }

int tensor(const char* what, const char* name, const void* base, const int64_t* strides, PackedTensor* out) {
    if (!base) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null %s", what, name);
    if (int st = kv_row_strides(what, name, strides)) return st;
    out->base = const_cast<void*>(base);
    out->token = strides[0];
    out->head = strides[1];
    return MHLO_CUDA_OK;
}
// Results: no two rows in one place.
int result(const char* what, const char* name, const void* base, const int64_t* strides, int64_t tokens, int64_t heads, int64_t dim, PackedTensor* out) {
    if (int st = tensor(what, name, base, strides, out)) return st;
    const bool apart = (tokens <= 1 || out->token >= dim) && (heads <= 1 || out->head >= dim) &&
                       (tokens <= 1 || heads <= 1 || out->token >= (heads - 1) * out->head + dim || out->head >= (tokens - 1) * out->token + dim);
    return apart ? MHLO_CUDA_OK : fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: rows of %s overlap", what, name);
}

int call_args(const char* what, int32_t dtype, const mhlo_cuda_packed_batch* batch, int64_t head_dim, float scale, PackedCall* c) {
    if (dtype != MHLO_DT_F16 && dtype != MHLO_DT_BF16 && dtype != MHLO_DT_F32) return fail(MHLO_CUDA_UNSUPPORTED, "%s: dtype %d", what, dtype);
    if (int st = packed_args(what, batch, &c->a)) return st;
    if (head_dim < 1 || head_dim > 128) return fail(MHLO_CUDA_UNSUPPORTED, "%s: head dimension %lld (1 .. 128)", what, static_cast<long long>(head_dim));
    if (!(scale > 0.f) || scale > 1e38f) return fail(MHLO_CUDA_UNSUPPORTED, "%s: scale %g", what, scale);
    c->a.head_dim = static_cast<int32_t>(head_dim);
    c->dtype = dtype;
    c->scale = scale;
    if (c->a.seqs > 0 && c->a.tokens > 0 && (!c->a.plan || !aligned16(c->a.plan))) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null or unaligned plan", what);
    return MHLO_CUDA_OK;
}

bool on_tensor_cores(const PackedCall& c, std::initializer_list<const PackedTensor*> of_queries, std::initializer_list<const PackedTensor*> of_keys) {
    if (c.dtype == MHLO_DT_F32 || c.a.head_dim % 8 != 0 || c.a.group > kRows) return false;
    for (const PackedTensor* t : of_queries)
        if (!packed_on_grid(*t, c.a.tokens, c.a.q_heads)) return false;
    for (const PackedTensor* t : of_keys)
        if (!packed_on_grid(*t, c.a.tokens, c.a.kv_heads)) return false;
    return true;
}

}  // namespace

int packed_join_shares(const PackedCall& c, int32_t splits, cudaStream_t stream) {
    return by_type(c, [&](auto t) { return join_shares<decltype(t)>(c, splits, stream); });
}

int packed_attention_device_error() {
    // One word at a time: each is of calls of its own, the others are left for the next one.
    int v = take_kv_error();
    if (v == 0) v = packed_attention_tc_device_error();
    return v == 0 ? packed_attention_grad_tc_device_error() : v;
}

}  // namespace mhlo

using namespace mhlo;

extern "C" {

int64_t mhlo_cuda_packed_plan_bytes(const mhlo_cuda_packed_batch* batch) {
    PackedArgs a;
    return packed_args("packed_plan", batch, &a) == MHLO_CUDA_OK ? plan_bytes(a) : 0;
}

int mhlo_cuda_packed_plan(const mhlo_cuda_packed_batch* batch, mhlo_cuda_stream_t stream) {
    PackedArgs a;
    if (int st = packed_args("packed_plan", batch, &a)) return st;
    if (a.seqs == 0 || a.tokens == 0) return MHLO_CUDA_OK;
    if (!a.starts || !a.plan || !aligned16(a.plan)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "packed_plan: null starts, or null or unaligned plan");
    packed_plan_kernel<<<static_cast<unsigned>(1 + (a.tokens + a.run_tokens - 1) / a.run_tokens), kPlanThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    MHLO_CUDA_CHECK_LAUNCH("packed_plan");
    return MHLO_CUDA_OK;
}

int mhlo_cuda_packed_attention(int32_t dtype, const mhlo_cuda_packed_batch* batch, int64_t head_dim, float scale, const void* q_dev, const int64_t q_strides[2],
                               const void* k_dev, const int64_t k_strides[2], const void* v_dev, const int64_t v_strides[2], void* o_dev, const int64_t o_strides[2],
                               float* lse_dev, mhlo_cuda_stream_t stream) {
    static const char* const what = "packed_attention";
    PackedCall c;
    if (int st = call_args(what, dtype, batch, head_dim, scale, &c)) return st;
    if (c.a.seqs == 0 || c.a.tokens == 0) return MHLO_CUDA_OK;
    if (int st = tensor(what, "q", q_dev, q_strides, &c.q)) return st;
    if (int st = tensor(what, "k", k_dev, k_strides, &c.k)) return st;
    if (int st = tensor(what, "v", v_dev, v_strides, &c.v)) return st;
    if (int st = result(what, "o", o_dev, o_strides, c.a.tokens, c.a.q_heads, head_dim, &c.o)) return st;
    c.lse = lse_dev;
    c.scratch = nullptr;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (on_tensor_cores(c, {&c.q, &c.o}, {&c.k, &c.v})) return packed_attention_tc(c, s);
    return by_type(c, [&](auto t) { return c.a.head_dim <= 64 ? forward<decltype(t), 64>(c, s) : forward<decltype(t), 128>(c, s); });
}

int64_t mhlo_cuda_packed_attention_grad_scratch_bytes(int32_t dtype, const mhlo_cuda_packed_batch* batch, int64_t head_dim) {
    PackedArgs a;
    if (head_dim < 1 || head_dim > 128 || packed_args("packed_attention_grad", batch, &a) != MHLO_CUDA_OK) return 0;
    return grad_scratch_bytes(dtype, a, head_dim);
}

int mhlo_cuda_packed_attention_grad(int32_t dtype, const mhlo_cuda_packed_batch* batch, int64_t head_dim, float scale, const void* q_dev, const int64_t q_strides[2],
                                    const void* k_dev, const int64_t k_strides[2], const void* v_dev, const int64_t v_strides[2], const void* o_dev,
                                    const int64_t o_strides[2], const float* lse_dev, const void* grad_dev, const int64_t grad_strides[2], void* dq_dev,
                                    const int64_t dq_strides[2], void* dk_dev, const int64_t dk_strides[2], void* dv_dev, const int64_t dv_strides[2], void* scratch_dev,
                                    int64_t scratch_bytes, mhlo_cuda_stream_t stream) {
    static const char* const what = "packed_attention_grad";
    PackedCall c;
    if (int st = call_args(what, dtype, batch, head_dim, scale, &c)) return st;
    if (c.a.seqs == 0 || c.a.tokens == 0) return MHLO_CUDA_OK;
    if (int st = tensor(what, "q", q_dev, q_strides, &c.q)) return st;
    if (int st = tensor(what, "k", k_dev, k_strides, &c.k)) return st;
    if (int st = tensor(what, "v", v_dev, v_strides, &c.v)) return st;
    if (int st = tensor(what, "o", o_dev, o_strides, &c.o)) return st;
    if (int st = tensor(what, "grad", grad_dev, grad_strides, &c.grad)) return st;
    if (int st = result(what, "dq", dq_dev, dq_strides, c.a.tokens, c.a.q_heads, head_dim, &c.dq)) return st;
    if (int st = result(what, "dk", dk_dev, dk_strides, c.a.tokens, c.a.kv_heads, head_dim, &c.dk)) return st;
    if (int st = result(what, "dv", dv_dev, dv_strides, c.a.tokens, c.a.kv_heads, head_dim, &c.dv)) return st;
    if (!lse_dev) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null lse", what);
    const int64_t need = grad_scratch_bytes(dtype, c.a, head_dim);
    if (!scratch_dev || !aligned16(scratch_dev) || scratch_bytes < need)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld bytes of scratch, %lld needed, on 16 bytes", what, static_cast<long long>(scratch_bytes), static_cast<long long>(need));
    c.lse = const_cast<float*>(lse_dev);
    c.scratch = scratch_dev;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool tensor_cores = on_tensor_cores(c, {&c.q, &c.grad, &c.dq}, {&c.k, &c.v, &c.dk, &c.dv});
    if (int st = by_type(c, [&](auto t) { return stats<decltype(t)>(c, tensor_cores && dtype == MHLO_DT_F16, s); })) return st;
    if (tensor_cores) return packed_attention_grad_tc(c, s);
    return by_type(c, [&](auto t) { return c.a.head_dim <= 64 ? backward<decltype(t), 64>(c, s) : backward<decltype(t), 128>(c, s); });
}

}  // extern "C"
