// What the two kernels of attention over the paged 8-bit cache share: how the work of a call is cut, and how cut pieces are joined.
//
// The work is cut into segments: (sequence, ROWS rows, cache head). The rows of a segment are (token, query head) pairs that read the
// same cache head: row r of a sequence is token r / group, query head head * group + r % group. A segment's keys are walked in tiles
// of KEYS; CTAs share all tiles of the call evenly, so a CTA's piece may begin or end inside a segment. Whole segments are written at
// once, pieces go to scratch as (maximum, sum, output), the output divided by the sum, and join_kernel joins them in the order of the
// CTAs: no atomics, and no order of arrival in the result.
#pragma once

#include <algorithm>
#include <cmath>

#include "kv_cache.cuh"

namespace mhlo {

// CTAs of the two kernels, all of them resident: two to an SM for few rows (while one joins its warps or looks up its next segment, the
// other reads: 32 ragged sequences of up to 4096 tokens 52 us with one of twice the warps, 48 with two), one for many.
constexpr int kFewGrid = 2 * kNumSMs, kLongGrid = kNumSMs;

template <typename T>
struct CachedParams {
    KvArgs kv;
    const T* q;
    T* o;
    float* lse;
    int64_t qs[2], os[2];
    int32_t q_heads, group;
    float scale, key_unit;  // the scale of the scores is scale * key_unit: see set_scale()
    int32_t q_vec;      // rows of q on the 16-byte grid
    int32_t o_vec;      // 1: results four at a time, 2: rows of o on the 16-byte grid
    int32_t whole;      // no segment has more than the least share of a CTA: none is cut
    int32_t few_rows;   // sequences of up to this many rows belong to the kernel of few rows, longer ones to the other
    int32_t* pieces;    // [CTAs][8]: the cut segment that a CTA's share ends with: CTAs it goes over (0: none), first row, rows, sequence's first row, head
    float* partial;     // [CTAs][2][ROWS (head_dim + 2)]: maxima (log2), sums, outputs / sums
};

// Scratch of one of the kernels: pieces, then partial results.
constexpr int64_t cached_scratch(int64_t ctas, int64_t rows, int64_t dim) { return ctas * (8 * 4 + 2 * rows * (dim + 2) * 4); }
template <typename T>
void cached_scratch(CachedParams<T>* p, int64_t ctas, void* scratch) {
    p->pieces = static_cast<int32_t*>(scratch);
    p->partial = reinterpret_cast<float*>(p->pieces + ctas * 8);
}
constexpr int kLongRows = 256;

// A scale in [2^-12, 2^-11) goes with the queries, whose own powers of two (2^-120 .. 2^114, and 2^24 where codes are subnormals of fp16)
// then leave it an ordinary number; the other power of two, as far as it is one itself, goes with the scales of the keys.
template <typename T>
void set_scale(CachedParams<T>* p, float scale) {
    const int exponent = std::min(std::ilogb(scale) + 12, 120);
    p->scale = std::scalbn(scale, -exponent);
    p->key_unit = std::scalbn(1.f, exponent);
}

namespace {

// Where one exponential serves a weight and the row's sum. A row has two references: m, near its largest z, and d, so that m + d is near
// its largest z + log2 vs. A weight is 2^(z - m) times 2^(log2 vs - d + unit): as long as the second factor is above 2^-40 nothing that
// counts in the sum is lost with the weight. Beyond kNearZero, z - m comes first: log2 vs would be lost beside z.
constexpr float kReach = 40.f, kBelow = 40.f, kNearZero = 4096.f;

// The power of two of a sum; 0 for sums that have none.
__device__ __forceinline__ float whole_log2(float l) {
    return l > 1e-37f && l < INFINITY ? static_cast<float>(static_cast<int>(__float_as_uint(l) >> 23) - 127) : 0.f;
}

// A key scale in units of key_unit. It stays finite: products of zero are zero whatever the scale.
__device__ __forceinline__ float key_scale(float ks, float unit) {
    const float x = ks * unit;
    return x > 3.4028235e38f ? 3.4028235e38f : x;
}

template <int V>
__device__ __forceinline__ void load_f32(const float* at, float* x) {
    if constexpr (V == 4) {
        const float4 v = *reinterpret_cast<const float4*>(at);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else if constexpr (V == 2) {
        const float2 v = *reinterpret_cast<const float2*>(at);
        x[0] = v.x, x[1] = v.y;
    } else {
        x[0] = *at;
    }
}

struct Segment {
    KvSequence s;
    int32_t b, head, row0, rows;  // sequence, cache head, first row and rows
    int32_t t0, t1, tiles;        // this piece's tiles, and all that the segment counts as
    int64_t begin;                // its first tile among all tiles of the call
    bool cut;
    __device__ __forceinline__ int32_t seen_by(int32_t r, int32_t group) const {  // keys that row r of the segment sees
        return s.length == 0 ? 0 : s.length - s.count + (row0 + r) / group + 1;
    }
    template <typename T>
    __device__ __forceinline__ int64_t token(const CachedParams<T>& p, int32_t r) const { return s.first + (row0 + r) / p.group; }
    template <typename T>
    __device__ __forceinline__ int64_t q_head(const CachedParams<T>& p, int32_t r) const { return head * p.group + (row0 + r) % p.group; }
};

// ROWS, KEYS: of a segment and a tile. LEAST: a CTA's share, in tiles, where there is little to do. LONG: takes the sequences of many rows.
template <int ROWS, int KEYS, int LEAST, bool LONG>
struct Work {
    static constexpr int kGrid = LONG ? kLongGrid : kFewGrid;
    struct Share {  // of one sequence
        KvSequence s;
        int32_t row_tiles, tiles;  // tiles: 1 where there are no keys: somebody has to write the zeros
        __device__ __forceinline__ int32_t counted(bool pad) const { return pad ? (tiles + LEAST - 1) / LEAST * LEAST : tiles; }
    };
    struct Scratch {  // in shared memory
        int64_t sums[64], totals[2], found[2];
    };
    int64_t at, end, per, inside;  // tiles of the call; inside: from the sequence's first
    int32_t b;
    bool pad;
    Share w;

    template <typename T>
    __device__ __forceinline__ static Share share_of(const CachedParams<T>& p, int32_t b) {
        Share w;
        w.s = kv_sequence(p.kv, b);
        const int64_t rows = static_cast<int64_t>(w.s.count) * p.group;
        w.row_tiles = (rows > p.few_rows) != LONG ? 0 : static_cast<int32_t>((rows + ROWS - 1) / ROWS);
        w.tiles = max(1, (w.s.length + KEYS - 1) / KEYS);
        return w;
    }
    __device__ __forceinline__ static int64_t warp_sum(int64_t v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }

    // The share of this CTA; false: none. All THREADS threads of the CTA call it. Where there is little to do segments count in whole
    // shares, so that no CTA gets the ends of two.
    template <int THREADS, typename T>
    __device__ __forceinline__ bool start(const CachedParams<T>& p, Scratch& scratch) {
        constexpr int W = THREADS / 32;
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        int64_t all = 0, all_padded = 0;
        for (int32_t i = tid; i < p.kv.seqs; i += THREADS) {
            const Share x = share_of(p, i);
            const int64_t segments = static_cast<int64_t>(x.row_tiles) * p.kv.heads;
            all += segments * x.tiles;
            all_padded += segments * x.counted(true);
        }
        all = warp_sum(all);
        all_padded = warp_sum(all_padded);
        if (lane == 0) {
            scratch.sums[warp] = all;
            scratch.sums[32 + warp] = all_padded;
        }
        __syncthreads();
        if (tid == 0) {
            int64_t x = 0, y = 0;
            for (int i = 0; i < W; ++i) {
                x += scratch.sums[i];
                y += scratch.sums[32 + i];
            }
            scratch.totals[0] = x;
            scratch.totals[1] = y;
            scratch.found[0] = -1;
        }
        __syncthreads();
        pad = p.whole || scratch.totals[1] <= static_cast<int64_t>(kGrid) * LEAST;
        const int64_t total = scratch.totals[pad ? 1 : 0];
        per = pad ? (total / LEAST + kGrid - 1) / kGrid * LEAST : (total + kGrid - 1) / kGrid;
        at = blockIdx.x * per;
        end = min(total, at + per);
        if (tid == 0 && !p.whole) p.pieces[blockIdx.x * 8] = 0;
        if (at >= end) return false;
        // the sequence that holds tile `at`, and where in it
        int64_t before = 0;
        for (int32_t base = 0; base < p.kv.seqs; base += THREADS) {
            int64_t mine = 0;
            if (base + tid < p.kv.seqs) {
                const Share x = share_of(p, base + tid);
                mine = static_cast<int64_t>(x.row_tiles) * p.kv.heads * x.counted(pad);
            }
            int64_t sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t other = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += other;
            }
            if (lane == 31) scratch.sums[warp] = sum;
            __syncthreads();
            int64_t chunk = 0, lower = 0;
            for (int i = 0; i < W; ++i) {
                lower += i < warp ? scratch.sums[i] : 0;
                chunk += scratch.sums[i];
            }
            const int64_t first = before + lower + sum - mine;
            if (mine > 0 && at >= first && at < first + mine) {
                scratch.found[0] = base + tid;
                scratch.found[1] = at - first;
            }
            before += chunk;
            __syncthreads();
            if (before > at) break;
        }
        b = static_cast<int32_t>(scratch.found[0]);
        inside = scratch.found[1];
        if (b < 0) return false;  // cannot be: lengths that change under the kernel
        w = share_of(p, b);
        return true;
    }

    // The next piece of this CTA's share.
    template <typename T>
    __device__ __forceinline__ bool next(const CachedParams<T>& p, Segment* s) {
        while (at < end) {
            const int32_t tiles = w.counted(pad);
            if (inside >= static_cast<int64_t>(w.row_tiles) * p.kv.heads * tiles) {  // on to the next sequence
                if (++b >= p.kv.seqs) return false;
                w = share_of(p, b);
                inside = 0;
                continue;
            }
            // 64-bit divisions are routines of a hundred instructions, and every warp of the tensor-core kernel walks by itself
            const bool small = inside < 0x80000000ll;
            const int32_t segment = small ? static_cast<int32_t>(static_cast<uint32_t>(inside) / static_cast<uint32_t>(tiles)) : static_cast<int32_t>(inside / tiles);
            const int32_t row_tile = segment / p.kv.heads;
            s->s = w.s;
            s->b = b;
            s->head = segment - row_tile * p.kv.heads;
            s->row0 = row_tile * ROWS;
            s->rows = min(ROWS, w.s.count * p.group - s->row0);
            s->t0 = static_cast<int32_t>(inside - static_cast<int64_t>(segment) * tiles);
            s->t1 = static_cast<int32_t>(min(static_cast<int64_t>(tiles), s->t0 + (end - at)));
            s->tiles = tiles;
            s->begin = at - s->t0;
            s->cut = s->t0 != 0 || s->t1 != tiles;
            at += s->t1 - s->t0;
            inside += s->t1 - s->t0;
            return true;
        }
        return false;
    }

    // Where a cut piece goes: a CTA may end one segment that others began, and begin one that others go on with.
    template <typename T>
    __device__ __forceinline__ float* partial(const CachedParams<T>& p, const Segment& s, int dim) const {
        return p.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (s.t0 == 0 ? 1 : 0)) * (ROWS * (dim + 2));
    }
    // One thread, for a cut piece: the CTA that began a segment leaves what joining it needs.
    template <typename T>
    __device__ __forceinline__ void leave_piece(const CachedParams<T>& p, const Segment& s) const {
        if (s.t0 != 0) return;
        int32_t* const piece = p.pieces + blockIdx.x * 8;
        piece[1] = s.row0;
        piece[2] = s.rows;
        piece[3] = s.s.first;
        piece[4] = s.head;
        piece[0] = static_cast<int32_t>((s.begin + s.tiles - 1) / per - blockIdx.x) + 1;
    }
};

// Joins row r of the segment that a CTA began and others went on with: sum_i o_i l_i 2^(m_i - m) / sum_i l_i 2^(m_i - m). A warp: the maxima
// and sums of up to 32 pieces are read at once, a lane each.
template <typename T, int D>
__device__ __forceinline__ void join_row(const CachedParams<T>& p, const int32_t* pieces, const float* partial, int32_t of_segment, int32_t cta, int32_t r) {
    constexpr int kEach = D / 32, V = D % 128 == 0 ? 4 : D == 64 ? 2 : 1;  // elements of a lane, and how many of them side by side
    const int lane = threadIdx.x & 31;
    const int32_t* const piece = pieces + cta * 8;
    const int32_t count = piece[0], row0 = piece[1], rows = piece[2], seq_first = piece[3], head = piece[4];
    if (count == 0 || r >= rows) return;
    auto part = [&](int32_t i) { return partial + ((static_cast<int64_t>(cta) + i) * 2 + (i == 0 ? 1 : 0)) * (of_segment * (D + 2)); };
    float most = -INFINITY, total = 0.f, sum[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum[e] = 0.f;
    for (int32_t base = 0; base < count; base += 32) {
        const bool there = base + lane < count;
        const float m = there ? part(base + lane)[r] : -INFINITY, l = there ? part(base + lane)[of_segment + r] : 0.f;
        const float top = fmaxf(most, warp_reduce<MaxOp>(m)), shift = top == -INFINITY ? 0.f : top;
        const float keep = ex2(most - shift), weight = l * ex2(m - shift);
        most = top;
        total = total * keep + warp_reduce<SumOp>(weight);
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] *= keep;
        const int32_t n = min(32, count - base);
#pragma unroll 4
        for (int32_t i = 0; i < n; ++i) {
            const float w = __shfl_sync(0xffffffffu, weight, i);
            const float* const o = part(base + i) + 2 * of_segment + r * D + lane * V;
            float x[kEach];
#pragma unroll
            for (int e = 0; e < kEach; e += V) load_f32<V>(o + 32 * e, x + e);
#pragma unroll
            for (int e = 0; e < kEach; ++e) sum[e] = fmaf(x[e], w, sum[e]);
        }
    }
    const int32_t row = row0 + r;
    const int64_t token = seq_first + row / p.group, q_head = head * p.group + row % p.group;
    T* const y = p.o + token * p.os[0] + q_head * p.os[1] + lane * V;
#pragma unroll
    for (int e = 0; e < kEach; ++e) y[32 * (e / V * V) + e % V] = VecTraits<T>::from_float(total == 0.f ? 0.f : sum[e] / total);
    if (p.lse != nullptr && lane == 0) p.lse[token * p.q_heads + q_head] = total == 0.f ? -INFINITY : (most + log2f(total)) * 0.6931471805599453f;
}

// One launch after both kernels, a CTA for kJoinRows rows of a CTA's note: y below long_rows / kJoinRows is of the kernel of many rows, y
// behind that of the other. Most have nothing to do; CTAs that look through all notes and share the rows that there are took 395 us for
// chunks of 512 tokens on four sequences of 8192 when these took 386.
constexpr int kJoinRows = 8;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinRows) join_kernel(const __grid_constant__ CachedParams<T> p, int32_t few_rows, const int32_t* long_pieces,
                                                              const float* long_partial, int32_t long_rows) {
    grid_dependency_wait();
    const bool is_long = static_cast<int32_t>(blockIdx.y) * kJoinRows < long_rows;
    if (is_long && blockIdx.x >= kLongGrid) return;
    const int32_t r = blockIdx.y * kJoinRows - (is_long ? 0 : long_rows) + (threadIdx.x >> 5);
    join_row<T, D>(p, is_long ? long_pieces : p.pieces, is_long ? long_partial : p.partial, is_long ? long_rows : few_rows, blockIdx.x, r);
}

}  // namespace

// The kernel of many rows (16-bit types, head dimension 64 or 128; cached_attention_tc.cu), with p's scratch set. Joining is the caller's.
template <typename T>
int cached_attention_long(const CachedParams<T>& p, cudaStream_t stream);
int cached_attention_long_device_error();

}  // namespace mhlo
