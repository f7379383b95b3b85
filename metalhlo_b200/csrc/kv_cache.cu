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

// Both kernels work in units of 16 elements of a row. A unit of a rotated row holds whole pairs: 8 neighbouring elements of the first
// half and their partners, or 16 neighbours where pairs are interleaved. A thread has the same unit of every row it takes, rows a
// fixed number apart, and all of them in registers at once (kKeep): no division and no second read.
//
// What bounds it: 16-bit elements come in two bytes each and take about seven instructions, rotation and quantisation two elements at
// a time, and a CTA that owns a block waits for its rows once before the scale and once for the codes of before. Five prompts of 6369
// tokens in all, 32 + 8 + 8 heads of 128, bf16: 30.5 us in a graph for 143 MB; one token of 64 sequences 4.0 us, which is a launch and three
// dependent reads.
template <typename T>
struct AppendParams {
    KvArgs kv;
    const T* x[2];       // keys, values
    int64_t xs[2][2];    // their {token, head} strides
    const T* q;
    T* q_out;
    int64_t qs[2], os[2];
    const float* rope;
    int64_t rope_positions;
    int32_t rotary_dim, interleaved, q_heads;
    int32_t vec[4];      // k, v, q, q_out: rows on the 16-byte grid
    FastDiv units, heads;  // units of a row of a head, query heads
    int32_t rows;          // of queries to a CTA
    float one;             // 1, which the compiler must not know
    int64_t blocks;      // CTAs that append, a block of keys or values each; the CTAs behind them rotate queries
};

template <typename T>
__device__ __forceinline__ void store8(T* y, bool vec, const float2* f) {
    if (vec) {
        constexpr int E = VecTraits<T>::kElems;
#pragma unroll
        for (int i = 0; i < 8; i += E) *reinterpret_cast<uint4*>(y + i) = VecTraits<T>::pack2(f + i / 2);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[2 * i] = VecTraits<T>::from_float(f[i].x);
            y[2 * i + 1] = VecTraits<T>::from_float(f[i].y);
        }
    }
}

// Two products and two sums at once, each rounded by itself. Written as a product and a sum the assembler makes one rounding of them
// (mul.rn.f32x2 and add.rn.f32x2 as well); a sum as x * 1 + y with a 1 that it does not know cannot be taken together with anything.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b, float one) { return __ffma2_rn(a, make_float2(one, one), b); }

// Where a unit's two groups of eight elements lie.
struct Unit {
    int32_t low, high, index;
    bool rotated;
};
__device__ __forceinline__ Unit unit_at(int32_t unit, int32_t rotary_dim, int32_t interleaved) {
    Unit u{unit * 16, unit * 16 + 8, unit, unit * 16 < rotary_dim};
    if (u.rotated && !interleaved) {
        u.low = unit * 8;
        u.high = (rotary_dim >> 1) + unit * 8;
    }
    return u;
}

// Rotates a unit by the cosines and sines of its position: products and sums rounded one by one (-(b s) is b (-s) to the last bit).
__device__ __forceinline__ void turn(float2* f, const float* row, int32_t unit, int32_t rotary_dim, int32_t interleaved, float one) {
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        *reinterpret_cast<float4*>(cs + i) = __ldg(reinterpret_cast<const float4*>(row + unit * 8 + i));
        *reinterpret_cast<float4*>(sn + i) = __ldg(reinterpret_cast<const float4*>(row + (rotary_dim >> 1) + unit * 8 + i));
    }
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            f[i] = add2(mul2(f[i], make_float2(cs[i], cs[i])), mul2(make_float2(f[i].y, f[i].x), make_float2(-sn[i], sn[i])), one);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 c = make_float2(cs[2 * i], cs[2 * i + 1]), n = make_float2(sn[2 * i], sn[2 * i + 1]), m = make_float2(-n.x, -n.y);
            const float2 a = f[i], b = f[4 + i];
            f[i] = add2(mul2(a, c), mul2(b, m), one);
            f[4 + i] = add2(mul2(b, c), mul2(a, n), one);
        }
    }
}
template <typename T>
__device__ __forceinline__ const float* rope_row(const AppendParams<T>& p, int32_t position) {
    if (position >= p.rope_positions) {
        kv_report(MHLO_CUDA_KV_ERROR_POSITION);
        position = static_cast<int32_t>(p.rope_positions - 1);
    }
    return p.rope + static_cast<int64_t>(position) * p.rotary_dim;
}

constexpr int kKeep = 4;  // units of a thread

// A unit as it lies in memory: half the registers of its numbers with 16-bit types.
template <typename T>
struct RawUnit {
    static constexpr int kVectors = 16 / VecTraits<T>::kElems;
    uint4 v[kVectors];
    __device__ __forceinline__ void load(const T* x, const Unit& u, bool vec) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const T* const at = x + (i < kVectors / 2 ? u.low + i * VecTraits<T>::kElems : u.high + (i - kVectors / 2) * VecTraits<T>::kElems);
            if (vec) {
                v[i] = __ldcs(reinterpret_cast<const uint4*>(at));  // not the read-only path: q may be rotated in place
            } else {
                float f[VecTraits<T>::kElems];
#pragma unroll
                for (int e = 0; e < VecTraits<T>::kElems; ++e) f[e] = VecTraits<T>::to_float(at[e]);
                v[i] = VecTraits<T>::pack(f);
            }
        }
    }
    __device__ __forceinline__ void numbers(float2* f) const {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) VecTraits<T>::unpack2(v[i], f + i * VecTraits<T>::kElems / 2);
    }
};

// Queries: a CTA takes p.rows rows. Their elements are on the way before the rows' sequences are looked up: three dependent reads of
// a few bytes each, which otherwise stood in front of every CTA's loads.
constexpr int kMostRows = 32;
template <typename T>
constexpr int kUnitsOfRows = sizeof(T) == 2 ? 4 : 2;

template <typename T>
__device__ __forceinline__ void rotate_rows(const AppendParams<T>& p, int32_t first_row) {
    const KvArgs& a = p.kv;
    __shared__ int32_t position[kMostRows];  // -1: the row is of no sequence
    const int32_t d = static_cast<int32_t>(p.units.d), rows = min(p.rows, a.tokens - first_row), all = rows * p.q_heads;
    const int32_t mine = static_cast<int32_t>(p.units.div(threadIdx.x)), step = static_cast<int32_t>(p.units.div(blockDim.x));
    const Unit u = unit_at(threadIdx.x - mine * d, p.rotary_dim, p.interleaved);
    constexpr int kMine = kUnitsOfRows<T>;
    for (int32_t start = 0; start < all; start += kMine * step) {
        RawUnit<T> raw[kMine];
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int32_t i = start + mine + k * step, row = static_cast<int32_t>(p.heads.div(i));
            if (mine < step && i < all) raw[k].load(p.q + static_cast<int64_t>(first_row + row) * p.qs[0] + (i - row * p.q_heads) * p.qs[1], u, p.vec[2]);
        }
        if (start == 0) {
            for (int32_t i = threadIdx.x >> 5; i < rows; i += blockDim.x >> 5) {  // a warp per row
                const int32_t r = first_row + i;
                int32_t b = r;
                if (a.starts != nullptr) b = kv_search(a.seqs, r, [&](int32_t j) { return static_cast<int64_t>(a.starts[j]); });
                const KvSequence s = kv_sequence(a, b);
                if ((threadIdx.x & 31) == 0) position[i] = s.length == 0 || r < s.first || r >= s.first + s.count ? -1 : s.position(r);
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int32_t i = start + mine + k * step, row = static_cast<int32_t>(p.heads.div(i));
            if (mine >= step || i >= all || position[row] < 0) continue;
            float2 f[8];
            raw[k].numbers(f);
            if (u.rotated) turn(f, rope_row(p, position[row]), u.index, p.rotary_dim, p.interleaved, p.one);
            T* const y = p.q_out + static_cast<int64_t>(first_row + row) * p.os[0] + (i - row * p.q_heads) * p.os[1];
            store8(y + u.low, p.vec[3], f);
            store8(y + u.high, p.vec[3], f + 4);
        }
    }
}

// round(x step) of four numbers as bytes: adding 1.5 * 2^23 leaves the integer, rounded to nearest even, in the low bits. |x step| is at
// most 127 and a rounding, step being the inverse of the largest magnitude / 127.
__device__ __forceinline__ uint32_t codes_of(float2 x, float2 y, float step, float one) {
    const float2 by = make_float2(step, step), magic = make_float2(12582912.f, 12582912.f);
    const float2 a = add2(mul2(x, by), magic, one), b = add2(mul2(y, by), magic, one);
    const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}

// A thread keeps the elements of its units as they are and rotates them twice, for the maximum and for the codes: with 16-bit types that
// leaves registers for three CTAs of 256 threads (80 each; prompts of 6369 tokens, 32 + 8 + 8 heads of 128: 37 us with the rotated numbers kept,
// 122 registers; 33 as they are with 122; 31 with 80). fp32 elements are 64 registers by themselves: 80 in all spilled 1 KB a thread,
// and two CTAs of 122 take 36.4 us for five chunks of 880 tokens instead of 42.6, 13.7 instead of 23.7 without queries. The largest pages
// of the widest heads have 512 threads to a CTA.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? (sizeof(T) == 2 ? 3 : 2) : 1) append_kernel(const __grid_constant__ AppendParams<T> p) {
    const KvArgs& a = p.kv;
    if (blockIdx.x >= p.blocks) return rotate_rows(p, static_cast<int32_t>(blockIdx.x - p.blocks) * p.rows);
    // Block `slot` of the sequences' touched blocks. A sequence has n / P + 2 slots at least, as many as n tokens can touch:
    // slot of its first block = floor(first row / P) + 2 b.
    const int32_t which = static_cast<int32_t>(blockIdx.x & 1), head = static_cast<int32_t>((blockIdx.x >> 1) % a.heads);
    const int64_t slot = (blockIdx.x >> 1) / a.heads;
    int32_t b, nth = 0;
    if (a.starts == nullptr) {
        b = static_cast<int32_t>(slot);
    } else {
        auto first = [&](int32_t i) { return static_cast<int64_t>(a.starts[i] >> a.page_shift) + 2 * i; };
        b = kv_search(a.seqs, slot, first);
        nth = static_cast<int32_t>(slot - first(b));
    }
    const KvSequence s = kv_sequence(a, b);
    // a sequence of n tokens touches n / P + 2 blocks at most; more slots come only from starts that are out of order
    if (s.length == 0 || s.count == 0 || nth < 0 || nth > (s.count >> a.page_shift) + 1) return;
    const int32_t page_index = ((s.length - s.count) >> a.page_shift) + nth, page_tokens = 1 << a.page_shift, dim = a.head_dim;
    const int32_t from = max(s.length - s.count, page_index << a.page_shift), to = min(s.length, (page_index + 1) << a.page_shift);
    if (from >= to) return;
    const int32_t slot0 = from & (page_tokens - 1), n = to - from, row0 = from - (s.length - s.count) + s.first;
    const int32_t d = static_cast<int32_t>(p.units.d), mine = static_cast<int32_t>(p.units.div(threadIdx.x)), step_rows = static_cast<int32_t>(p.units.div(blockDim.x));
    const int32_t rotary = which == 0 ? p.rotary_dim : 0;
    const Unit u = unit_at(threadIdx.x - mine * d, rotary, p.interleaved);
    const T* const x = p.x[which] + row0 * p.xs[which][0] + head * p.xs[which][1];
    auto token = [&](int k) { return mine < step_rows ? mine + k * step_rows : n; };  // of the block's new ones; n: none

    RawUnit<T> raw[kKeep];
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
        const int32_t t = token(k);
        if (t < n) raw[k].load(x + t * p.xs[which][0], u, p.vec[which]);
    }
    auto numbers = [&](int k, float2* f) {  // rotated
        raw[k].numbers(f);
        if (u.rotated) turn(f, rope_row(p, from + token(k)), u.index, rotary, p.interleaved, p.one);
    };
    // only now the page: the elements are on the way meanwhile
    const int32_t page = kv_page(a, b, page_index);
    if (page < 0) return;
    const int64_t block = static_cast<int64_t>(page) * a.heads + head;
    int8_t* const codes = (which == 0 ? a.k_codes : a.v_codes) + block * page_tokens * dim;
    float* const scales = (which == 0 ? a.k_scales : a.v_scales) + block;
    const float before = slot0 == 0 ? 0.f : *scales;
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
        const int32_t t = token(k);
        if (t >= n) continue;
        float2 f[8];
        numbers(k, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max_nan(most, max_nan(fabsf(f[e].x), fabsf(f[e].y)));
    }
    // as bits, magnitudes are ordered like the numbers, infinity and NaN above all
    uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(most) & 0x7fffffffu);
    __shared__ uint32_t largest[16];
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) m = max(m, largest[w]);
    float scale = __fmul_rn(__uint_as_float(m), 1.f / 127.f);
    if (scale < 1.17549435e-38f) scale = 0.f;
    scale = before > scale || before != before ? before : scale;
    if (m >= 0x7f800000u) scale = __uint_as_float(0x7fffffffu);
    if (threadIdx.x == 0) *scales = scale;
    if (scale > before) {  // earlier tokens of the block
        const float ratio = __fdiv_rn(before, scale);
        for (int32_t i = threadIdx.x * 16; i < slot0 * dim; i += blockDim.x * 16) {
            uint4 v = *reinterpret_cast<const uint4*>(codes + i);
            uint32_t* const w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float c[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] = static_cast<float>(static_cast<int8_t>(w[k] >> (8 * e)));
                w[k] = codes_of(make_float2(c[0], c[1]), make_float2(c[2], c[3]), ratio, p.one);
            }
            *reinterpret_cast<uint4*>(codes + i) = v;
        }
    }
    const float step = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;  // NaN scales: codes 0
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
        const int32_t t = token(k);
        if (t >= n) continue;
        uint32_t w[4] = {0, 0, 0, 0};
        if (step > 0.f) {
            float2 f[8];
            numbers(k, f);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = codes_of(f[2 * e], f[2 * e + 1], step, p.one);
        }
        int8_t* const y = codes + (slot0 + t) * dim;
        *reinterpret_cast<uint2*>(y + u.low) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(y + u.high) = make_uint2(w[2], w[3]);
    }
}

template <typename T>
__global__ void __launch_bounds__(128) read_kernel(const __grid_constant__ KvArgs a, T* k_out, T* v_out, int64_t s_seq, int64_t s_token, int64_t s_head,
                                                   int64_t max_tokens, int64_t pieces, FastDiv units, int32_t vec) {
    const int32_t page_tokens = 1 << a.page_shift, dim = a.head_dim;
    const int32_t which = static_cast<int32_t>(blockIdx.x & 1), head = static_cast<int32_t>((blockIdx.x >> 1) % a.heads);
    T* out = which == 0 ? k_out : v_out;
    if (out == nullptr) return;
    const int64_t piece = (blockIdx.x >> 1) / a.heads;
    const int32_t b = static_cast<int32_t>(piece / pieces), i0 = static_cast<int32_t>(piece % pieces);
    int32_t length = a.lengths[b];
    if (length < 0 || length > static_cast<int64_t>(a.pages_per_seq) << a.page_shift) {
        kv_report(MHLO_CUDA_KV_ERROR_LENGTH);
        length = 0;
    }
    const int64_t first = static_cast<int64_t>(i0) << a.page_shift;
    const int32_t page = first < length ? kv_page(a, b, i0) : -1;
    const int64_t block = static_cast<int64_t>(page) * a.heads + head;
    const float scale = page < 0 ? 0.f : (which == 0 ? a.k_scales : a.v_scales)[block];
    const int8_t* const codes = (which == 0 ? a.k_codes : a.v_codes) + block * page_tokens * dim;
    const int32_t tokens = static_cast<int32_t>(min(static_cast<int64_t>(page_tokens), max_tokens - first));
    const int32_t there = page < 0 ? 0 : static_cast<int32_t>(min(static_cast<int64_t>(tokens), length - first));
    out += b * s_seq + head * s_head + first * s_token;
#pragma unroll 4
    for (int32_t i = threadIdx.x; i < tokens * static_cast<int32_t>(units.d); i += 128) {
        const int32_t t = static_cast<int32_t>(units.div(i)), unit = i - t * static_cast<int32_t>(units.d);
        float2 f[8];
        if (t < there) {
            const uint4 v = ld_stream16(codes + i * 16);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                f[e] = make_float2(__fmul_rn(static_cast<float>(static_cast<int8_t>(w[e >> 1] >> (16 * (e & 1)))), scale),
                                   __fmul_rn(static_cast<float>(static_cast<int8_t>(w[e >> 1] >> (16 * (e & 1) + 8))), scale));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = make_float2(0.f, 0.f);
        }
        T* const y = out + t * s_token + unit * 16;
        store8(y, vec, f);
        store8(y + 8, vec, f + 4);
    }
}

// Rows of a tensor on the 16-byte grid.
template <typename T>
int32_t on_grid(const void* x, int64_t s0, int64_t s1) {
    constexpr int64_t E = VecTraits<T>::kElems;
    return aligned16(x) && s0 % E == 0 && s1 % E == 0;
}

template <typename T>
int append(const KvArgs& kv, const void* k, const int64_t* ks, const void* v, const int64_t* vs, const void* q, const int64_t* qs, void* q_out,
           const int64_t* os, int64_t q_heads, const float* rope, int64_t rope_positions, int64_t rotary_dim, int32_t interleaved, cudaStream_t stream) {
    AppendParams<T> p;
    p.kv = kv;
    p.x[0] = static_cast<const T*>(k);
    p.x[1] = static_cast<const T*>(v);
    p.q = static_cast<const T*>(q);
    p.q_out = static_cast<T*>(q_out);
    for (int i = 0; i < 2; ++i) {
        p.xs[0][i] = ks[i];
        p.xs[1][i] = vs[i];
        p.qs[i] = q ? qs[i] : 0;
        p.os[i] = q ? os[i] : 0;
    }
    p.vec[0] = on_grid<T>(k, ks[0], ks[1]);
    p.vec[1] = on_grid<T>(v, vs[0], vs[1]);
    p.vec[2] = q && on_grid<T>(q, qs[0], qs[1]);
    p.vec[3] = q && on_grid<T>(q_out, os[0], os[1]);
    p.rope = rope;
    p.rope_positions = rope_positions;
    p.rotary_dim = static_cast<int32_t>(rope ? rotary_dim : 0);
    p.interleaved = interleaved != 0;
    p.one = 1.f;
    p.q_heads = static_cast<int32_t>(q_heads);
    p.units = FastDiv(static_cast<uint32_t>(kv.head_dim / 16));
    p.blocks = 2 * kv.heads * (kv.starts ? (static_cast<int64_t>(kv.tokens) >> kv.page_shift) + 2 * static_cast<int64_t>(kv.seqs) : kv.seqs);
    // A whole block in the registers of a CTA: kKeep of a thread's units, 512 threads at most (pages of 128 tokens of 256 elements).
    // Single tokens need few threads for their keys and values, as many as there are query heads for those.
    const int d = kv.head_dim / 16;
    const int64_t wanted = kv.starts ? (int64_t{1} << kv.page_shift) / kKeep * d : q ? std::min<int64_t>(128, (q_heads + kKeep - 1) / kKeep * d) : 32;
    const int threads = static_cast<int>((std::max<int64_t>(32, std::max<int64_t>(wanted, d)) + 31) / 32 * 32);
    p.heads = FastDiv(static_cast<uint32_t>(std::max<int64_t>(1, q_heads)));
    // Rows of queries to a CTA: as many as its threads hold, unless that would leave SMs idle (64 rows of 32 x 128: 6.2 us three at a
    // time, 4.4 one by one).
    const int64_t fit = kUnitsOfRows<T> * (threads / d) / std::max<int64_t>(1, q_heads), spread = (kv.tokens + 4 * kNumSMs - 1) / (4 * kNumSMs);
    p.rows = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>(kMostRows, std::min(fit, spread))));
    const int64_t grid = p.blocks + (q ? (kv.tokens + p.rows - 1) / p.rows : 0);
    if (grid > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "kv_cache_append: too many blocks");
    if (threads <= 256) append_kernel<T, 256><<<static_cast<unsigned>(grid), threads, 0, stream>>>(p);
    else append_kernel<T, 512><<<static_cast<unsigned>(grid), threads, 0, stream>>>(p);
    MHLO_CUDA_CHECK_LAUNCH("kv_cache_append");
    return MHLO_CUDA_OK;
}

template <typename T>
int read(const KvArgs& kv, int64_t max_tokens, void* k_out, void* v_out, const int64_t* strides, cudaStream_t stream) {
    const int64_t pieces = (max_tokens + (int64_t{1} << kv.page_shift) - 1) >> kv.page_shift, grid = 2 * pieces * kv.heads * kv.seqs;
    if (grid > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "kv_cache_read: too many blocks");
    const int32_t vec = on_grid<T>(k_out, strides[0], strides[1]) && on_grid<T>(v_out, strides[2], 0);
    read_kernel<T><<<static_cast<unsigned>(grid), 128, 0, stream>>>(kv, static_cast<T*>(k_out), static_cast<T*>(v_out), strides[0], strides[1], strides[2],
                                                                    max_tokens, pieces, FastDiv(static_cast<uint32_t>(kv.head_dim / 16)), vec);
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
