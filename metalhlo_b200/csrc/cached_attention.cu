// Attention of new tokens over the paged 8-bit key/value cache: o = softmax(scale q k^T) v with k = ks c, v = vs c. This is the kernel of
// few rows; sequences with more go to cached_attention_tc.cu where that takes their type.
//
// Inside a CTA every warp takes tiles by itself and keeps a running maximum, sum and output of the rows; the warps are joined
// through shared memory at the end of a segment. Nothing but the segment's end synchronises the warps.
//
// The products are transposed, S^T = C q^T and O^T = C^T P^T (16 x 8 x 16 steps): keys and elements of values take the long side of
// the instruction, rows the short one. A decoding step has as many rows as query heads share a cache head, mostly 4 to 8, and would
// fill 16 to a half or less: half the products, exponentials and output registers.
//
// A row's references for its sum and its output are of keys that it sees (m and d below): a block that it does not see, or whose keys have
// nothing of its weight, costs it no digits, however large the block's values are.
//
// What bounds it: the codes have to come from memory once, 64 sequences of 8192 keys with 8 heads of 128 (4 query heads each, bf16)
// 175 us in a graph for 1.07 GB, 6.1 TB/s. With fewer or ragged sequences the ends of segments show: 32 of up to 4096 keys 48 us for 179 MB,
// of which reading alone would take 28. ncu, 32 of 8192 keys: 44 % of issue slots, 20 % of the tensor pipe, 168 registers.
#include <algorithm>
#include <type_traits>

#include "cached_attention.cuh"

namespace mhlo {
namespace {

constexpr int kTileKeys = 32;
constexpr int kLeastTiles = 12;  // a CTA's share where there is little to do: two tiles of a warp

template <int D>
struct Layout {
    static constexpr int kWarps = D == 256 ? 3 : 6;  // two CTAs to an SM
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kStages = D == 64 ? 4 : 2;
    static constexpr int kTileBytes = kTileKeys * D;  // of keys, and of values
    static constexpr int kRing = kWarps * kStages * 2 * kTileBytes;
    // A row of codes is stored as parts of 128, 64 or 32 bytes, each [32 keys][W].
    static constexpr int kParts = D == 256 ? 2 : D == 96 ? 2 : 1;
    __host__ __device__ static constexpr int width(int part) { return D == 96 ? (part == 0 ? 64 : 32) : D == 64 ? 64 : 128; }
    __host__ __device__ static constexpr int first(int part) { return part == 0 ? 0 : D == 96 ? 64 : 128; }
    static constexpr int kSteps = D / 16;
};

// ---- the kernel's parts ----------------------------------------------------------------------------------------------------

__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {  // the transpose of an 8 x 8 matrix of 16-bit elements, two a lane
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Codes as fp16. A code with its sign bit turned round is code + 128 in 0 .. 255: as the low byte of an fp16 number with nothing else
// that is the subnormal (code + 128) 2^-24, which the tensor cores take as it is. The 128 comes off again from the sums: those of q
// are known beforehand, those of the weights are one more column of the product. With 16-bit inputs that saves the subtraction of
// every code (a quarter of all instructions). A sum that carries 128 times the weights loses digits with every step of 16 keys (the
// tensor cores cut off, all in one direction), so it comes off every kCorrect tiles: 2 steps each, 2^-22 of at most 255 weights a step, make
// 2^-11 of a code's step at most, however many keys there are. Without, averages of 131072 keys were off by 0.015 of a code's step, 5 % of
// what is left of them; now by 5e-6 (head dimension 128, 12 rows). In fp32 the sums would lose too much, so there a code is put behind 0x64
// (1024 + x) and 1152 is taken off, which is exact.
constexpr uint32_t kSignBits = 0x80808080u;
constexpr int kCorrect = 4;
template <bool EXACT>
__device__ __forceinline__ uint32_t two_codes(uint32_t codes, uint32_t order) {
    if (!EXACT) return __byte_perm(codes, 0, order);
    const uint32_t x = __byte_perm(codes, 0x64646464u, order), bias = 0x64806480u;  // 1152, 1152
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
}
constexpr float kCodeUnit = 16777216.f;    // 2^24: what the sums of 16-bit inputs are short of
constexpr uint32_t kBiasPair = 0x00800080u;  // 128 2^-24, twice
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void cp_async16(uint32_t smem, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(smem), "l"(src) : "memory");
}

// Where 16-byte chunk `chunk` of row `row` of a part lies. Keys are read 16 bytes a lane, four lanes a row; values by eight groups of
// lanes, each W / 8 bytes of rows 2 c + e (c = 0 .. 3). The exclusive ors make both free of bank conflicts for 128-byte and 64-byte
// parts; 32-byte parts lie in order.
template <int W, bool VALUES>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
    if (W == 128) return row * 128 + ((chunk ^ (VALUES ? row & 6 : (row & 1) << 2)) << 4);
    if (W == 64) {
        const int slot = (row & 1) * 4 + chunk;
        return (row >> 1) * 128 + ((VALUES ? slot ^ (row & 6) : slot) << 4);
    }
    return row * 32 + (chunk << 4);
}

// Starts the copies of 16 keys and values (half a tile, contiguous in a page): `from` their offset in the codes. The lane's part of
// every address is the same for each pass of the loop but for the exclusive or, so it costs no more than that.
template <int D>
__device__ __forceinline__ void load_half(const int8_t* k, const int8_t* v, uint32_t keys, int half) {
    using L = Layout<D>;
    const int lane = threadIdx.x & 31;
    constexpr int kChunks = D / 16;  // of a row
#pragma unroll
    for (int i = 0; i < 16 * kChunks / 32; ++i) {
        const int index = i * 32 + lane, row = half * 16 + index / kChunks, chunk = index % kChunks;
        const int part = L::kParts == 1 ? 0 : chunk * 16 >= L::first(1);
        const int c = part == 0 ? chunk : chunk - L::first(1) / 16;
        uint32_t ko, vo;
        if (part == 0) {
            ko = chunk_at<L::width(0), false>(row, c);
            vo = chunk_at<L::width(0), true>(row, c);
        } else {
            ko = kTileKeys * L::width(0) + chunk_at<L::width(1), false>(row, c);
            vo = kTileKeys * L::width(0) + chunk_at<L::width(1), true>(row, c);
        }
        cp_async16(keys + ko, k + i * 512);
        cp_async16(keys + L::kTileBytes + vo, v + i * 512);
    }
}

// Fragment order of a row's elements. A step of 16 products uses, from lane c of four, four neighbouring elements: in a 64-byte
// stretch those at 16 c + 4 s (s = 0 .. 3), in a 32-byte part those at 8 c + 4 s (s = 0, 1). Any order will do as long as q and k agree.
template <int D>
__device__ __forceinline__ int step_element(int step, int c) {
    if (D == 96 && step >= 4) return 64 + 8 * c + 4 * (step - 4);
    return 64 * (step >> 2) + 16 * c + 4 * (step & 3);
}

// Weights 2^(z - m + log2 vs - d), m + d a row's largest z + log2 vs so far, go into fp16 times a power of two, so that those far below the
// largest keep some bits above the smallest step, 2^-24. In fp32 the unit is 2^14; with 16-bit inputs 2^6, and what a row sees may exceed
// m + d by 2^8 before everything is scaled anew: with exact maxima some row of 16 found a new one in almost every tile, 10 % of all
// instructions. m and d are whole numbers, so that what is scaled by their differences is not rounded.
template <typename T>
constexpr float kUnitLog2Of = sizeof(T) == 4 ? 14.f : 6.f;
template <typename T>
constexpr float kHeadroomOf = sizeof(T) == 4 ? 1.9f : 8.f;
constexpr float kNone = -3e38f;  // m + d of a row that has seen nothing: below every sum, but less -infinity it is not NaN
// 2^whole; 0 and infinity out of fp32's ordinary exponents. The sum leaves whole + 127 in the low bits.
__device__ __forceinline__ float pow2_of(float whole) { return __int_as_float(__float_as_int(fminf(fmaxf(whole, -127.f), 128.f) + 12583039.f) << 23); }

// NT: groups of 8 rows.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(Layout<D>::kThreads, 2) cached_attention_kernel(const __grid_constant__ CachedParams<T> p) {
    using L = Layout<D>;
    constexpr int kRows = 8 * NT;
    constexpr bool kTwoParts = sizeof(T) == 4;  // fp32: q and the weights as sums of two fp16 numbers
    constexpr float kUnitLog2 = kUnitLog2Of<T>, kHeadroom = kHeadroomOf<T>;
    constexpr int W = L::kWarps;
    extern __shared__ __align__(128) uint8_t smem[];
    uint2* const q_frag = reinterpret_cast<uint2*>(smem + L::kRing);  // [1 or 2 parts][steps][NT][32]
    __shared__ float row_factor[kRows];                               // scale log2(e) 2^exponent of the row's q
    __shared__ float row_bias[kRows];                                 // -128 2^-24 times the sum of the row's q as fp16
    __shared__ __align__(8) float sm[W][kRows], sd[W][kRows];  // references of a warp's rows
    __shared__ float sl[W][kRows], sf[W][kRows], top_m[kRows], top_l[kRows];
    __shared__ int32_t used[W];
    __shared__ float2 top_unit[kRows];  // a power of two as two
    // Of a tile's halves: scales of the keys (-infinity: not there) and log2 of those of the values (a half that is not there has the
    // other's); those of the values, or with 16-bit inputs 1 / (weight unit * scale).
    __shared__ float4 meta[W][L::kStages];
    __shared__ float2 meta_v[W][L::kStages];
    __shared__ typename Work<kRows, kTileKeys, kLeastTiles, false>::Scratch scratch;

    const KvArgs& a = p.kv;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;

    Work<kRows, kTileKeys, kLeastTiles, false> work;
    const bool any = work.template start<L::kThreads>(p, scratch);
    grid_dependency_release();
    Segment seg;
    while (any && work.next(p, &seg)) {
        const int32_t b = seg.b, head = seg.head, t0 = seg.t0, rows = seg.rows;
        auto seen_by = [&](int r) { return seg.seen_by(r, p.group); };
        const int32_t limit = seen_by(rows - 1), least = seen_by(0);
        const int32_t last = min(seg.t1, (limit + kTileKeys - 1) / kTileKeys);  // tiles t0 .. last - 1 have keys to read

        // -- q as fragments in shared memory, rows brought to the same size by powers of two
        const float to_log2 = p.scale * 1.4426950408889634f;
        for (int r = warp; r < kRows; r += W) {
            float most = 0.f, x[D / 32];
            const T* q = p.q + seg.token(p, r) * p.qs[0] + seg.q_head(p, r) * p.qs[1];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                x[i] = r < rows ? VecTraits<T>::to_float(q[lane + 32 * i]) : 0.f;
                most = fmaxf(most, fabsf(x[i]));
            }
            int shift = 0;
            if (!std::is_same<T, __half>::value) {
                most = warp_reduce<MaxOp>(most);
                if (most > 0.f && most < INFINITY) shift = max(-120, ilogbf(most) - 13);
            }
            const float unit = scalbnf(1.f, -shift);
            float sum = 0.f;
            if (!kTwoParts) {
#pragma unroll
                for (int i = 0; i < D / 32; ++i) sum += __half2float(__float2half_rn(x[i] * unit));
                sum = warp_reduce<SumOp>(sum);
            }
            if (lane == 0) {
                row_factor[r] = scalbnf(to_log2, shift) * (kTwoParts ? 1.f : kCodeUnit);
                row_bias[r] = sum * (-128.f / kCodeUnit);
                sf[0][r] = unit;
            }
        }
        __syncthreads();
        for (int i = tid; i < L::kSteps * NT * 32; i += L::kThreads) {
            const int l = i & 31, j = (i >> 5) % NT, step = (i >> 5) / NT, r = 8 * j + (l >> 2);
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (r < rows) {
                const T* q = p.q + seg.token(p, r) * p.qs[0] + seg.q_head(p, r) * p.qs[1] + step_element<D>(step, l & 3);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = VecTraits<T>::to_float(q[e]) * sf[0][r];
            }
            q_frag[i] = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
            if (kTwoParts) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] -= __half2float(__float2half_rn(x[e]));
                q_frag[L::kSteps * NT * 32 + i] = make_uint2(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]));
            }
        }
        __syncthreads();

        // -- this warp's tiles: t0 + warp, t0 + warp + W, ...
        // Lane (g, c) has rows 8 j + 2 c + i of keys g and g + 8 of a half, and of elements W / 8 g .. of each part of the values.
        // A row's references: m (z - m in the sum l) and d (z - m + log2 vs - d in weights and o). What follows from them: both (m + d), and
        // near, the least log2 vs for which one exponential serves l and o. With 16-bit inputs l is in units of 2^(m + d), as far as
        // kReach allows (sum_unit()), so it gets what o gets, and m and d lie in shared memory: ordinary tiles need only what follows from
        // them, and registers are short. fp32: conv is 2^-d times the unit of the weights.
        float o[D / 16][NT][4], m[NT][2], d[NT][2], both[NT][2], l[NT][2], conv[kTwoParts ? NT : 1][2], near = -kReach, conv_most = 0.f, o_bias[NT][4], factor[NT][2], bias[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) o[t][j][e] = 0.f;
                o_bias[j][e] = 0.f;
                if (e < 2) {
                    m[j][e] = d[j][e] = -INFINITY;
                    both[j][e] = kNone;
                    l[j][e] = 0.f;
                    if (kTwoParts) conv[kTwoParts ? j : 0][e] = 0.f;
                    factor[j][e] = row_factor[8 * j + 2 * c + e];
                    bias[j][e] = row_bias[8 * j + 2 * c + e];
                }
            }
        auto sum_unit = [](float x) { return kTwoParts || x == -INFINITY ? 0.f : fminf(fmaxf(x, -kReach), kReach); };
        auto measure = [&]() {
            near = -kReach;
            conv_most = 0.f;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float x = d[j][r];
                    both[j][r] = x == -INFINITY ? kNone : m[j][r] + x;
                    if (kTwoParts) {
                        conv[kTwoParts ? j : 0][r] = x == -INFINITY ? 0.f : pow2_of(kUnitLog2 - x);
                        conv_most = fmaxf(conv_most, conv[kTwoParts ? j : 0][r]);
                    }
                    if (x != -INFINITY) near = fabsf(x) <= kReach && fabsf(m[j][r]) <= kNearZero ? fmaxf(near, x - kBelow) : INFINITY;
                }
        };
        auto load_references = [&]() {
            if (kTwoParts) return;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const float2 x = *reinterpret_cast<const float2*>(&sm[warp][8 * j + 2 * c]), y = *reinterpret_cast<const float2*>(&sd[warp][8 * j + 2 * c]);
                m[j][0] = x.x, m[j][1] = x.y, d[j][0] = y.x, d[j][1] = y.y;
            }
        };
        auto store_references = [&]() {
            __syncwarp();
            if (g == 0) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    *reinterpret_cast<float2*>(&sm[warp][8 * j + 2 * c]) = make_float2(m[j][0], m[j][1]);
                    *reinterpret_cast<float2*>(&sd[warp][8 * j + 2 * c]) = make_float2(d[j][0], d[j][1]);
                }
            }
            __syncwarp();
        };
        if (!kTwoParts) store_references();
        constexpr bool kKeepQ = NT == 1 && !kTwoParts && D <= 128;  // in registers
        uint2 q_kept[kKeepQ ? L::kSteps : 1];
        if (kKeepQ) {
#pragma unroll
            for (int i = 0; i < L::kSteps; ++i) q_kept[i] = q_frag[i * 32 + lane];
        }
        const int32_t mine = last > t0 + warp ? (last - t0 - warp + W - 1) / W : 0;
        const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * L::kStages * 2 * L::kTileBytes;
        // Pages and scales of 16 tiles at a time, a half tile per lane.
        const int8_t *const k_lane = a.k_codes + lane * 16, *const v_lane = a.v_codes + lane * 16;
        int64_t base = -1;
        float ks = 0.f, vs = 0.f, vs_log2 = 0.f;
        auto issue = [&](int32_t i) {
            if (i < mine) {
                if ((i & 15) == 0) {
                    const int32_t tile = t0 + warp + (i + (lane >> 1)) * W, key = tile * kTileKeys + (lane & 1) * 16;
                    base = -1;
                    if (tile < last && key < limit) {
                        const int32_t page = kv_page(a, b, key >> a.page_shift);
                        if (page >= 0) {
                            const int64_t block = static_cast<int64_t>(page) * a.heads + head;
                            base = ((block << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * D;
                            ks = a.k_scales[block];
                            vs = a.v_scales[block];
                        }
                    }
                }
                const int from = (i & 15) * 2, stage = i % L::kStages;
                const int64_t base0 = __shfl_sync(0xffffffffu, base, from), base1 = __shfl_sync(0xffffffffu, base, from + 1);
                if (base0 >= 0) load_half<D>(k_lane + base0, v_lane + base0, ring + stage * 2 * L::kTileBytes, 0);
                if (base1 >= 0) load_half<D>(k_lane + base1, v_lane + base1, ring + stage * 2 * L::kTileBytes, 1);
                asm volatile("cp.async.commit_group;" ::: "memory");
                if ((i & 15) == 0) {  // only now: the copies do not wait for the scales
                    ks = key_scale(ks, p.key_unit);
                    vs_log2 = log2f(vs);
                    if (!kTwoParts) vs = __fdividef(exp2f(-kUnitLog2), vs);
                }
                const float k1 = __shfl_down_sync(0xffffffffu, ks, 1), v1 = __shfl_down_sync(0xffffffffu, vs, 1), log1 = __shfl_down_sync(0xffffffffu, vs_log2, 1);
                if (lane == from) {
                    meta[warp][stage] = make_float4(base0 < 0 ? -INFINITY : ks, base1 < 0 ? -INFINITY : k1, base0 < 0 ? log1 : vs_log2, base1 < 0 ? vs_log2 : log1);
                    meta_v[warp][stage] = make_float2(base0 < 0 ? 0.f : vs, base1 < 0 ? 0.f : v1);
                }
            } else {
                asm volatile("cp.async.commit_group;" ::: "memory");
            }
        };
        for (int i = 0; i < L::kStages - 1; ++i) issue(i);
        for (int32_t i = 0; i < mine; ++i) {
            issue(i + L::kStages - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 1) : "memory");
            __syncwarp();
            const int stage = i % L::kStages;
            const uint8_t* const keys = smem + warp * L::kStages * 2 * L::kTileBytes + stage * 2 * L::kTileBytes;
            const uint8_t* const values = keys + L::kTileBytes;
            const float4 scales = meta[warp][stage];
            const float out_again[2] = {meta_v[warp][stage].x, meta_v[warp][stage].y};
            const bool half_there[2] = {scales.x != -INFINITY, scales.y != -INFINITY};

            // S^T = C q^T, 16 keys a step
            float s[2][NT][4];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[half][j][e] = kTwoParts ? 0.f : bias[j][e & 1];
#pragma unroll
            for (int part = 0; part < L::kParts; ++part) {
                const int width = L::width(part), step0 = L::first(part) / 16;
                const uint8_t* const base_part = keys + kTileKeys * L::first(part);
#pragma unroll
                for (int chunk = 0; chunk < (width + 63) / 64; ++chunk) {
                    uint32_t codes[4][4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const int row = n * 8 + g;
                        if (width == 32) {
                            const uint2 x = *reinterpret_cast<const uint2*>(base_part + row * 32 + c * 8);
                            codes[n][0] = x.x ^ kSignBits;
                            codes[n][1] = x.y ^ kSignBits;
                        } else {
                            const uint32_t where = width == 128 ? chunk_at<128, false>(row, chunk * 4 + c) : chunk_at<64, false>(row, c);
                            const uint4 x = *reinterpret_cast<const uint4*>(base_part + where);
                            codes[n][0] = x.x ^ kSignBits;
                            codes[n][1] = x.y ^ kSignBits;
                            codes[n][2] = x.z ^ kSignBits;
                            codes[n][3] = x.w ^ kSignBits;
                        }
                    }
#pragma unroll
                    for (int i4 = 0; i4 < (width == 32 ? 2 : 4); ++i4) {
                        const int step = step0 + chunk * 4 + i4;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t a0 = two_codes<kTwoParts>(codes[2 * half][i4], 0x4140), a1 = two_codes<kTwoParts>(codes[2 * half + 1][i4], 0x4140);
                            const uint32_t a2 = two_codes<kTwoParts>(codes[2 * half][i4], 0x4342), a3 = two_codes<kTwoParts>(codes[2 * half + 1][i4], 0x4342);
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                const uint2 qb = kKeepQ ? q_kept[kKeepQ ? step : 0] : q_frag[(step * NT + j) * 32 + lane];
                                mma_f16(s[half][j], a0, a1, a2, a3, qb);
                                if (kTwoParts) mma_f16(s[half][j], a0, a1, a2, a3, q_frag[((L::kSteps + step) * NT + j) * 32 + lane]);
                            }
                        }
                    }
                }
            }
            // Scores in units of log2(e) are s f. Tiles that every row sees whole keep them so; others are brought to f = 1 and masked.
            const int32_t key0 = (t0 + warp + i * W) * kTileKeys;
            const float values_log2[2] = {scales.z, scales.w};
            const bool edge = key0 + kTileKeys > least || !half_there[0] || !half_there[1];
            float f[2][NT][2];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    f[0][j][r] = factor[j][r] * scales.x;
                    f[1][j][r] = factor[j][r] * scales.y;
                }
            if (edge) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int32_t seen[2] = {seen_by(8 * j + 2 * c), seen_by(8 * j + 2 * c + 1)};
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool hidden = !half_there[half] || key0 + half * 16 + (e >> 1) * 8 + g >= seen[e & 1];
                            s[half][j][e] = hidden ? -INFINITY : s[half][j][e] * f[half][j][e & 1];
                        }
                        f[half][j][0] = f[half][j][1] = 1.f;
                    }
                }
            }
            // plain: the scales of both halves are near enough to the references, so the value scale goes into the exponent, and the sum takes
            // it out again once per half. Else the sum has exponentials of its own. References move only when what a row sees leaves
            // the headroom of the weights: every lane looks at its own scores, and lanes talk once a tile and more only when they have to.
            // A half that a row does not see is at -infinity, whatever its scales.
            auto largest = [&](int j, int r, int half) { return fmaxf(s[half][j][r], s[half][j][2 + r]); };
            float top[NT][2];
            bool plain = !kTwoParts, move = false;
            if (plain) {
                move = !(values_log2[0] >= near && values_log2[1] >= near && values_log2[0] <= kReach && values_log2[1] <= kReach);
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        top[j][r] = fmaxf(fmaf(largest(j, r, 0), f[0][j][r], values_log2[0]), fmaf(largest(j, r, 1), f[1][j][r], values_log2[1]));
                        move = move || top[j][r] > both[j][r] + kHeadroom;
                    }
                move = __any_sync(0xffffffffu, move);
            }
            if (!plain || move) {
                load_references();
                float keep[NT][2];
                auto over_keys = [&](float (&x)[NT][2]) {  // of all rows side by side
#pragma unroll
                    for (int lanes = 4; lanes < 32; lanes <<= 1)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int r = 0; r < 2; ++r) x[j][r] = fmaxf(x[j][r], __shfl_xor_sync(0xffffffffu, x[j][r], lanes));
                };
                const float least = fminf(values_log2[0], values_log2[1]);
                if (plain) {  // may one maximum do?
                    bool odd = !(least >= near && fabsf(values_log2[0]) <= kReach && fabsf(values_log2[1]) <= kReach && fabsf(values_log2[0] - values_log2[1]) <= 30.f);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const bool valueless = d[j][r] == -INFINITY && m[j][r] != -INFINITY;  // value scales of 0 so far: m may be anywhere
                            odd = odd || valueless || (fabsf(top[j][r]) > kNearZero && top[j][r] != -INFINITY);
                        }
                    plain = !__any_sync(0xffffffffu, odd);
                }
                if (plain) {  // then m is as near to the largest z as the value scales are to one another
                    over_keys(top);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const bool grow = top[j][r] > both[j][r] + kHeadroom;
                            const float to = floorf(top[j][r]), was = m[j][r];
                            keep[j][r] = grow ? ex2(both[j][r] - to) : 1.f;
                            l[j][r] *= !grow ? 1.f : was == -INFINITY ? 0.f : ex2(was + sum_unit(d[j][r]) - to);
                            m[j][r] = grow ? fmaxf(was, to - floorf(least)) : was;
                            d[j][r] = grow ? to - m[j][r] : d[j][r];
                        }
                } else {
                    move = false;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float z0 = fmaf(largest(j, r, 0), f[0][j][r], -m[j][r]), z1 = fmaf(largest(j, r, 1), f[1][j][r], -m[j][r]);
                            move = move || fmaxf(z0 + values_log2[0], z1 + values_log2[1]) > d[j][r] + kHeadroom || fmaxf(z0, z1) > kHeadroom;
                        }
                    move = __any_sync(0xffffffffu, move);
                    if (move) {
                        // With value scales within a factor of 2 the largest z bounds the largest z - m + log2 vs closely enough.
                        float mine[NT][2];
                        bool odd = !(fabsf(values_log2[0] - values_log2[1]) <= 1.f);
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                mine[j][r] = fmaxf(largest(j, r, 0) * f[0][j][r], largest(j, r, 1) * f[1][j][r]);
                                odd = odd || (fabsf(mine[j][r]) > kNearZero && mine[j][r] != -INFINITY);
                            }
                        odd = __any_sync(0xffffffffu, odd);
                        over_keys(mine);
                        float before[NT][2];
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const bool grow = mine[j][r] > m[j][r] + kHeadroom;
                                before[j][r] = m[j][r];
                                m[j][r] = grow ? floorf(mine[j][r]) : m[j][r];
                                mine[j][r] = (mine[j][r] - m[j][r]) + fmaxf(values_log2[0], values_log2[1]);
                            }
                        if (odd) {
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int r = 0; r < 2; ++r)
                                    mine[j][r] = fmaxf(fmaf(largest(j, r, 0), f[0][j][r], -m[j][r]) + values_log2[0], fmaf(largest(j, r, 1), f[1][j][r], -m[j][r]) + values_log2[1]);
                            over_keys(mine);
                        }
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const bool first = before[j][r] == -INFINITY;
                                const float down = first ? 0.f : before[j][r] - m[j][r], unit = sum_unit(d[j][r]), now = d[j][r] + down, to = floorf(mine[j][r]);
                                const bool grow = mine[j][r] > now + kHeadroom;
                                keep[j][r] = !grow ? 1.f : now == -INFINITY ? 0.f : ex2(now - to);
                                d[j][r] = grow ? to : now;
                                l[j][r] *= first ? 0.f : ex2(down + (unit - sum_unit(d[j][r])));
                            }
                    }
                }
                if (move) {
                    if (i > 0) {  // there is an output already
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
#pragma unroll
                                for (int t = 0; t < D / 16; ++t) o[t][j][e] *= keep[j][e & 1];
                                o_bias[j][e] *= keep[j][e & 1];
                            }
                    }
                    measure();
                    if (!kTwoParts) store_references();
                }
            }
            if (plain) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float in_exponent = values_log2[half] + kUnitLog2;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float sum[2] = {0.f, 0.f}, off[2];
#pragma unroll
                        for (int r = 0; r < 2; ++r) off[r] = in_exponent - both[j][r];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float& x = s[half][j][e];
                            x = ex2(fmaf(x, f[half][j][e & 1], off[e & 1]));
                            sum[e & 1] += x;
                        }
                        l[j][0] = fmaf(sum[0], out_again[half], l[j][0]);
                        l[j][1] = fmaf(sum[1], out_again[half], l[j][1]);
                    }
                }
            } else if (kTwoParts && !__any_sync(0xffffffffu, !(out_again[0] * conv_most <= 1e22f && out_again[1] * conv_most <= 1e22f))) {
                // fp32: a weight is its exponential times conv and the value scale, which rounds once.
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const float ratio[2] = {out_again[half] * conv[kTwoParts ? j : 0][0], out_again[half] * conv[kTwoParts ? j : 0][1]};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float own = ex2(fmaf(s[half][j][e], f[half][j][e & 1], m[j][e & 1] == -INFINITY ? 0.f : -m[j][e & 1]));
                            l[j][e & 1] += own;
                            s[half][j][e] = own * ratio[e & 1];  // hidden: 0 times a number
                        }
                    }
            } else {
                // Two exponentials. In fp32 the value scale's whole power of two goes into that of the weights.
                load_references();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float rest = 1.f, whole = values_log2[half];
                    if (kTwoParts) {
                        const int exponent = ilogbf(out_again[half]);
                        whole = out_again[half] == 0.f ? -INFINITY : static_cast<float>(exponent);
                        rest = out_again[half] == 0.f ? 0.f : scalbnf(out_again[half], -exponent);
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float minus[2], unit[2], off[2];
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            minus[r] = m[j][r] == -INFINITY ? 0.f : -m[j][r];
                            unit[r] = sum_unit(d[j][r]);
                            off[r] = whole + (kUnitLog2 - (d[j][r] == -INFINITY ? 0.f : d[j][r]));
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool hidden = edge && s[half][j][e] == -INFINITY;
                            const float z = fmaf(s[half][j][e], f[half][j][e & 1], minus[e & 1]);
                            l[j][e & 1] += ex2(z - unit[e & 1]);
                            s[half][j][e] = hidden ? 0.f : rest * ex2(z + off[e & 1]);  // whatever the scale of a block that the row does not see
                        }
                    }
                }
            }
            // P^T as fragments: keys 2 c, 2 c + 1 and 8 + 2 c, 9 + 2 c of row g
            uint2 pa[2][NT], pb[2][NT];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float* const x = s[half][j];
                    pa[half][j] = make_uint2(turned(pack_half2(x[0], x[1])), turned(pack_half2(x[2], x[3])));
                    if (kTwoParts) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] -= __half2float(__float2half_rn(x[e]));
                        pb[half][j] = make_uint2(turned(pack_half2(x[0], x[1])), turned(pack_half2(x[2], x[3])));
                    } else {
                        mma_f16(o_bias[j], kBiasPair, kBiasPair, kBiasPair, kBiasPair, pa[half][j]);
                    }
                }
            // O^T += C^T P^T: group g of lanes holds W / 8 neighbouring elements of a part, two per product
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int part = 0; part < L::kParts; ++part) {
                    const int width = L::width(part), words = width / 32, tile0 = L::first(part) / 16;
                    const uint8_t* const base_part = values + kTileKeys * L::first(part);
                    uint32_t rows4[4][4];  // rows 2 c, 2 c + 1, 8 + 2 c, 9 + 2 c
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = half * 16 + (r >> 1) * 8 + 2 * c + (r & 1);
                        if (width == 128) {
                            const uint4 x = *reinterpret_cast<const uint4*>(base_part + chunk_at<128, true>(row, g));
                            rows4[r][0] = x.x ^ kSignBits;
                            rows4[r][1] = x.y ^ kSignBits;
                            rows4[r][2] = x.z ^ kSignBits;
                            rows4[r][3] = x.w ^ kSignBits;
                        } else if (width == 64) {
                            const uint2 x = *reinterpret_cast<const uint2*>(base_part + chunk_at<64, true>(row, g >> 1) + (g & 1) * 8);
                            rows4[r][0] = x.x ^ kSignBits;
                            rows4[r][1] = x.y ^ kSignBits;
                        } else {
                            rows4[r][0] = *reinterpret_cast<const uint32_t*>(base_part + row * 32 + g * 4) ^ kSignBits;
                        }
                    }
#pragma unroll
                    for (int word = 0; word < words; ++word)
#pragma unroll
                        for (int pair = 0; pair < 2; ++pair) {  // bytes 2 pair, 2 pair + 1
                            const uint32_t even = __byte_perm(rows4[0][word], rows4[1][word], pair ? 0x7362 : 0x5140);
                            const uint32_t odd = __byte_perm(rows4[2][word], rows4[3][word], pair ? 0x7362 : 0x5140);
                            const uint32_t a0 = two_codes<kTwoParts>(even, 0x4140), a1 = two_codes<kTwoParts>(even, 0x4342);
                            const uint32_t a2 = two_codes<kTwoParts>(odd, 0x4140), a3 = two_codes<kTwoParts>(odd, 0x4342);
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                float* const acc = o[tile0 + word * 2 + pair][j];
                                mma_f16(acc, a0, a1, a2, a3, pa[half][j]);
                                if (kTwoParts) mma_f16(acc, a0, a1, a2, a3, pb[half][j]);
                            }
                        }
                }
            if (!kTwoParts && (i & (kCorrect - 1)) == kCorrect - 1) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
#pragma unroll
                        for (int t = 0; t < D / 16; ++t) o[t][j][e] -= o_bias[j][e];
                        o_bias[j][e] = 0.f;
                    }
            }
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // every warp is done with the rings: they hold the warps' outputs now

        // -- join the warps
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[j][r] += __shfl_xor_sync(0xffffffffu, l[j][r], x);
                if (g == 0) {
                    // the sum's power of two goes to its reference, which may have stayed behind: sums of other warps are weighed by that
                    float &m_out = sm[warp][8 * j + 2 * c + r], &d_out = sd[warp][8 * j + 2 * c + r];
                    if (kTwoParts) m_out = m[j][r], d_out = d[j][r];
                    const float up = whole_log2(l[j][r]), unit = sum_unit(d_out);
                    sl[warp][8 * j + 2 * c + r] = l[j][r] * ex2(-up);
                    m_out += unit + up;
                    d_out -= unit + up;
                }
            }
        if (lane == 0) used[warp] = mine > 0;
        float4* const joined = reinterpret_cast<float4*>(smem);  // [warp][row][D / 4], chunks turned against bank conflicts
        auto joined_at = [](int w_, int row, int d4) {
            const int pair = (row >> 1) & 3;
            return (w_ * kRows + row) * (D / 4) + (d4 ^ (D == 64 ? (pair & 1) | (pair >> 1) << 2 : pair));
        };
        if (mine > 0) {
#pragma unroll
            for (int part = 0; part < L::kParts; ++part) {
                const int each = L::width(part) / 8, tile0 = L::first(part) / 16;  // elements L::first + each g ..
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int k = 0; k < each; k += 4) {
                            const float off = o_bias[j][r];
                            const float(*x)[NT][4] = &o[tile0 + k / 2];
                            joined[joined_at(warp, 8 * j + 2 * c + r, (L::first(part) + g * each + k) >> 2)] =
                                make_float4(x[0][j][r] - off, x[0][j][2 + r] - off, x[1][j][r] - off, x[1][j][2 + r] - off);
                        }
            }
        }
        __syncthreads();
        if (tid < kRows) {
            float ms[W], ds[W], ls[W], most = -INFINITY, unit = -INFINITY, sum = 0.f;  // unit: the largest m + d, less most
#pragma unroll
            for (int i = 0; i < W; ++i) ms[i] = sm[i][tid], ds[i] = sd[i][tid], ls[i] = sl[i][tid];
#pragma unroll
            for (int i = 0; i < W; ++i) most = fmaxf(most, ms[i]);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                sum += ms[i] == -INFINITY ? ls[i] : ls[i] * ex2(ms[i] - most);
                ds[i] = ds[i] == -INFINITY ? -INFINITY : ds[i] + (ms[i] - most);
                unit = fmaxf(unit, ds[i]);
            }
#pragma unroll
            for (int i = 0; i < W; ++i) sf[i][tid] = ds[i] == -INFINITY ? 0.f : pow2_of(ds[i] - unit);
            const float whole = unit == -INFINITY ? 0.f : unit - kUnitLog2 + (kTwoParts ? 0.f : 24.f), first = floorf(0.5f * whole);
            top_unit[tid] = make_float2(pow2_of(first), pow2_of(whole - first));
            top_m[tid] = most;
            top_l[tid] = sum;
        }
        __syncthreads();
        float* const out = work.partial(p, seg, D);
        for (int i = tid; i < kRows * (D / 4); i += L::kThreads) {
            const int r = i / (D / 4), d4 = i % (D / 4);
            if (r >= rows) break;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < W; ++k) {
                if (!used[k]) continue;
                const float4 x = joined[joined_at(k, r, d4)];
                const float f = sf[k][r];
                sum.x += x.x * f;
                sum.y += x.y * f;
                sum.z += x.z * f;
                sum.w += x.w * f;
            }
            const float total_l = top_l[r], inv = total_l == 0.f ? 0.f : 1.f / total_l;
            const float2 unit = top_unit[r];
            const float4 x = total_l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                            : make_float4(sum.x * inv * unit.x * unit.y, sum.y * inv * unit.x * unit.y, sum.z * inv * unit.x * unit.y, sum.w * inv * unit.x * unit.y);
            if (seg.cut) {
                reinterpret_cast<float4*>(out + 2 * kRows)[i] = x;
                continue;
            }
            T* const y = p.o + seg.token(p, r) * p.os[0] + seg.q_head(p, r) * p.os[1] + d4 * 4;
            if constexpr (sizeof(T) == 4) {
                if (p.o_vec) *reinterpret_cast<float4*>(y) = x;
                else y[0] = x.x, y[1] = x.y, y[2] = x.z, y[3] = x.w;
            } else {
                const float xs[8] = {x.x, x.y, x.z, x.w, 0.f, 0.f, 0.f, 0.f};
                const uint4 packed = VecTraits<T>::pack(xs);
                if (p.o_vec) *reinterpret_cast<uint2*>(y) = make_uint2(packed.x, packed.y);
                else
                    for (int e = 0; e < 4; ++e) y[e] = VecTraits<T>::from_float(xs[e]);
            }
        }
        if (tid < rows) {
            if (seg.cut) {
                out[tid] = top_m[tid];
                out[kRows + tid] = top_l[tid];
            } else if (p.lse != nullptr) {
                p.lse[seg.token(p, tid) * p.q_heads + seg.q_head(p, tid)] = top_l[tid] == 0.f ? -INFINITY : (top_m[tid] + log2f(top_l[tid])) * 0.6931471805599453f;
            }
        }
        if (seg.cut && tid == 0) work.leave_piece(p, seg);
        __syncthreads();
    }
    // Where the kernel of many rows went before, this one began as that one's CTAs ended (their rows are not these); what joins the
    // pieces of both waits for this kernel alone, so this kernel ends after that one.
    grid_dependency_wait();
}

constexpr bool long_takes(int64_t head_dim) { return head_dim == 64 || head_dim == 128; }
// Sequences of up to this many rows are this kernel's, where the other takes the type. It walks the keys once for each 16 rows, the other
// once for 256. Calls through this kernel with the other's launch in front, which has nothing to do and takes 7 us, and through the other
// alone, us, bf16: 64 sequences of 1000 keys, 8 cache heads of 128: 32 rows 105 and 148, 48 rows 143 and 149, 64 rows 165 (less the 7) and
// 150; 8 of 6000 keys: 48 rows 80 and 84, 64 rows 90 (less the 7) and 85; 2 of 8000: 48 rows 46 and 40; head dimension 64, 64 of 1000: 48
// rows 98 and 113, 64 rows 117 and 114; 8 of 6000: 48 rows 55 and 67, 64 rows 65 and 66; 2 of 8000: 48 rows 36 and 33.
constexpr int kFewRows = 48;
// Whether a sequence of the call may have more rows: the host knows only how many there are in all.
bool may_be_long(const int32_t* starts, int64_t tokens, int64_t group, int64_t head_dim) {
    return starts != nullptr && long_takes(head_dim) && tokens * group > kFewRows;
}

template <typename T, int D, int NT>
int launch_rows(const CachedParams<T>& p, bool behind, cudaStream_t stream) {
    using L = Layout<D>;
    constexpr int smem = L::kRing + L::kSteps * NT * 32 * 8 * (sizeof(T) == 4 ? 2 : 1);
    auto kernel = cached_attention_kernel<T, D, NT>;
    static std::atomic<bool> smem_set[64];
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, smem_set)) return st;
    // Behind the kernel of many rows it may begin before that one ends. In front of it is then only what that one waited for; behind
    // anything else it has to wait, whatever the environment says of overlap: it reads before grid_dependency_wait().
    if (behind) {
        const cudaError_t e = launch_dependent(kernel, dim3(kFewGrid), dim3(L::kThreads), smem, stream, 1, true, p);
        if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of cached_attention failed: %s", cudaGetErrorString(e));
    } else {
        kernel<<<kFewGrid, L::kThreads, smem, stream>>>(p);
    }
    MHLO_CUDA_CHECK_LAUNCH("cached_attention");
    return MHLO_CUDA_OK;
}

template <typename T, int D>
int launch_dim(CachedParams<T> p, void* scratch, cudaStream_t stream) {
    // Which kernels: sequences of many rows go to the one, where there may be any, the rest to the other. One sequence by itself that may
    // have many rows goes to the one whatever it has.
    const bool may_long = sizeof(T) == 2 && may_be_long(p.kv.starts, p.kv.tokens, p.group, D);
    const bool few = !may_long || p.kv.seqs > 1;
    CachedParams<T> many = p;
    many.few_rows = p.few_rows = !may_long ? 0x7fffffff : few ? kFewRows : 0;
    // Groups of 8 rows as long as the sequences have no more on average: 16 sequences of 4000 keys, 8 cache heads of 128, 8 rows 38 us in
    // groups of 8 and 47 in groups of 16; 12 rows 50 and 47.
    const int groups = static_cast<int64_t>(p.kv.tokens) * p.group <= 8 * static_cast<int64_t>(p.kv.seqs) ? 1 : 2;
    cached_scratch(&p, kFewGrid, scratch);
    cached_scratch(&many, kLongGrid, scratch != nullptr ? static_cast<uint8_t*>(scratch) + cached_scratch(kFewGrid, 16, D) : nullptr);
    if constexpr (sizeof(T) == 2 && long_takes(D)) {
        if (may_long) {
            if (int st = cached_attention_long(many, stream)) return st;
        }
    }
    if (few) {
        if (int st = groups == 1 ? launch_rows<T, D, 1>(p, may_long, stream) : launch_rows<T, D, 2>(p, may_long, stream)) return st;
    }
    if (p.whole) return MHLO_CUDA_OK;
    const int rows = few ? 8 * groups : 0, long_rows = may_long ? kLongRows : 0;
    const cudaError_t e = launch_dependent(join_kernel<T, D>, dim3(few ? kFewGrid : kLongGrid, (rows + long_rows) / kJoinRows), dim3(32 * kJoinRows), 0, stream,
                                           1, true, p, rows, static_cast<const int32_t*>(many.pieces), static_cast<const float*>(many.partial), long_rows);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of cached_attention failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("cached_attention (joining)");
    return MHLO_CUDA_OK;
}

template <typename T>
int launch(const KvArgs& kv, const void* q, const int64_t* qs, int64_t q_heads, float scale, void* o, const int64_t* os, float* lse, void* scratch, cudaStream_t stream) {
    CachedParams<T> p;
    p.kv = kv;
    p.q = static_cast<const T*>(q);
    p.o = static_cast<T*>(o);
    p.lse = lse;
    for (int i = 0; i < 2; ++i) p.qs[i] = qs[i], p.os[i] = os[i];
    p.q_heads = static_cast<int32_t>(q_heads);
    p.group = static_cast<int32_t>(q_heads / kv.heads);
    set_scale(&p, scale);
    p.whole = scratch == nullptr;
    constexpr int64_t E = VecTraits<T>::kElems;
    p.q_vec = aligned16(q) && qs[0] % E == 0 && qs[1] % E == 0;
    p.o_vec = aligned16(o) && os[0] % E == 0 && os[1] % E == 0 ? 2 : reinterpret_cast<uintptr_t>(o) % (4 * sizeof(T)) == 0 && os[0] % 4 == 0 && os[1] % 4 == 0;
    switch (kv.head_dim) {
        case 64: return launch_dim<T, 64>(p, scratch, stream);
        case 96: return launch_dim<T, 96>(p, scratch, stream);
        case 128: return launch_dim<T, 128>(p, scratch, stream);
        default: return launch_dim<T, 256>(p, scratch, stream);
    }
}

}  // namespace

int cached_attention_device_error() {
    const int few = take_kv_error(), many = cached_attention_long_device_error();  // one call's: reported, and cleared, as one
    return few < 0 || many < 0 ? -1 : few != 0 ? few : many;
}

}  // namespace mhlo

using namespace mhlo;

extern "C" {

int64_t mhlo_cuda_cached_attention_scratch_bytes(const mhlo_cuda_kv_cache* cache, const mhlo_cuda_kv_batch* batch, int64_t q_heads) {
    if (!cache || !batch || q_heads < 1) return 0;
    if (cache->head_dim < 1 || batch->pages_per_seq * cache->page_tokens <= kLeastTiles * kTileKeys) return 0;  // no segment is worth cutting
    const int64_t group = q_heads / std::max<int64_t>(1, cache->heads);
    int64_t bytes = cached_scratch(kFewGrid, 16, cache->head_dim);
    if (may_be_long(batch->token_starts, batch->tokens, group, cache->head_dim))
        bytes += cached_scratch(kLongGrid, kLongRows, cache->head_dim);
    return bytes;
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
    if (!(scale > 0.f) || scale > 1e38f) return fail(MHLO_CUDA_UNSUPPORTED, "%s: the scale has to be positive and at most 1e38", what);
    if (batch->tokens * q_heads > 0x7fffffff)
        return fail(MHLO_CUDA_UNSUPPORTED, "%s: %lld tokens of %lld heads (2^31 - 1 rows at most)", what, static_cast<long long>(batch->tokens), static_cast<long long>(q_heads));
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
    if (dtype == MHLO_DT_F32) return launch<float>(kv, q_dev, q_strides, q_heads, scale, o_dev, o_strides, lse_dev, need > 0 ? scratch_dev : nullptr, st);
    if (dtype == MHLO_DT_F16) return launch<__half>(kv, q_dev, q_strides, q_heads, scale, o_dev, o_strides, lse_dev, need > 0 ? scratch_dev : nullptr, st);
    return launch<__nv_bfloat16>(kv, q_dev, q_strides, q_heads, scale, o_dev, o_strides, lse_dev, need > 0 ? scratch_dev : nullptr, st);
}

}  // extern "C"
