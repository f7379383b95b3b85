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
// half and their partners, or 16 neighbours where pairs are interleaved.
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
    int64_t blocks;      // CTAs that append, a block of keys or values each; the CTAs behind them rotate queries
};

template <typename T>
__device__ __forceinline__ void load8(const T* x, bool vec, float* f) {
    if (vec) {
        constexpr int E = VecTraits<T>::kElems;
#pragma unroll
        for (int i = 0; i < 8; i += E) VecTraits<T>::unpack(__ldcs(reinterpret_cast<const uint4*>(x + i)), f + i);  // not the read-only path: q may be rotated in place
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = VecTraits<T>::to_float(x[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* y, bool vec, const float* f) {
    if (vec) {
        constexpr int E = VecTraits<T>::kElems;
#pragma unroll
        for (int i = 0; i < 8; i += E) *reinterpret_cast<uint4*>(y + i) = VecTraits<T>::pack(f + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = VecTraits<T>::from_float(f[i]);
    }
}

// Where a unit's two groups of eight elements lie.
struct Unit {
    int32_t low, high;
    bool rotated;
};
__device__ __forceinline__ Unit unit_at(int32_t unit, int32_t rotary_dim, int32_t interleaved) {
    Unit u{unit * 16, unit * 16 + 8, unit * 16 < rotary_dim};
    if (u.rotated && !interleaved) {
        u.low = unit * 8;
        u.high = (rotary_dim >> 1) + unit * 8;
    }
    return u;
}

// The cosines and sines of a unit's eight pairs.
__device__ __forceinline__ void load_turn(const float* row, int32_t unit, int32_t rotary_dim, float* cs, float* sn) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        *reinterpret_cast<float4*>(cs + i) = __ldg(reinterpret_cast<const float4*>(row + unit * 8 + i));
        *reinterpret_cast<float4*>(sn + i) = __ldg(reinterpret_cast<const float4*>(row + (rotary_dim >> 1) + unit * 8 + i));
    }
}
__device__ __forceinline__ void turn(float* f, const float* cs, const float* sn, int32_t interleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int lo = interleaved ? 2 * i : i, hi = interleaved ? 2 * i + 1 : i + 8;
        const float a = f[lo], b = f[hi];
        f[lo] = __fsub_rn(__fmul_rn(a, cs[i]), __fmul_rn(b, sn[i]));
        f[hi] = __fadd_rn(__fmul_rn(b, cs[i]), __fmul_rn(a, sn[i]));
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

constexpr int kKeep = 4;  // units a thread keeps in registers between the maximum and the codes

// Queries: a CTA takes p.rows rows, kKeep units a thread. Their elements are on the way before the rows' sequences are looked up: three
// dependent reads of a few bytes each, which otherwise stood in front of every CTA's loads ([4400, 32, 128] bf16: 41 us).
constexpr int kMostRows = 32;

template <typename T>
__device__ __forceinline__ void rotate_rows(const AppendParams<T>& p, int32_t first_row) {
    const KvArgs& a = p.kv;
    __shared__ int32_t position[kMostRows];  // -1: the row is of no sequence
    const int32_t rows = min(p.rows, a.tokens - first_row), threads = blockDim.x, d = static_cast<int32_t>(p.units.d), all = rows * p.q_heads * d;
    for (int32_t start = 0; start < all; start += kKeep * threads) {
        float f[kKeep][16];
        int32_t row[kKeep], head[kKeep], unit[kKeep];
#pragma unroll
        for (int k = 0; k < kKeep; ++k) {
            const int32_t i = start + threadIdx.x + k * threads, column = static_cast<int32_t>(p.units.div(i));
            unit[k] = i - column * d;
            row[k] = i < all ? static_cast<int32_t>(p.heads.div(column)) : -1;
            head[k] = column - row[k] * p.q_heads;
            if (row[k] < 0) continue;
            const Unit u = unit_at(unit[k], p.rotary_dim, p.interleaved);
            const T* const x = p.q + static_cast<int64_t>(first_row + row[k]) * p.qs[0] + head[k] * p.qs[1];
            load8(x + u.low, p.vec[2], f[k]);
            load8(x + u.high, p.vec[2], f[k] + 8);
        }
        if (start == 0) {
            for (int32_t i = threadIdx.x >> 5; i < rows; i += threads >> 5) {  // a warp per row
                const int32_t r = first_row + i;
                int32_t b = r;
                if (a.starts != nullptr) b = kv_search(a.seqs, r, [&](int32_t j) { return static_cast<int64_t>(a.starts[j]); });
                const KvSequence s = kv_sequence(a, b);
                if ((threadIdx.x & 31) == 0) position[i] = s.length == 0 || r < s.first || r >= s.first + s.count ? -1 : s.position(r);
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < kKeep; ++k) {
            if (row[k] < 0 || position[row[k]] < 0) continue;
            const Unit u = unit_at(unit[k], p.rotary_dim, p.interleaved);
            if (u.rotated) {
                float cs[8], sn[8];
                load_turn(rope_row(p, position[row[k]]), unit[k], p.rotary_dim, cs, sn);
                if (p.interleaved) turn(f[k], cs, sn, 1);
                else turn(f[k], cs, sn, 0);
            }
            T* const y = p.q_out + static_cast<int64_t>(first_row + row[k]) * p.os[0] + head[k] * p.os[1];
            store8(y + u.low, p.vec[3], f[k]);
            store8(y + u.high, p.vec[3], f[k] + 8);
        }
    }
}

__device__ __forceinline__ uint32_t code_of(float x, float step) {
    return static_cast<uint32_t>(min(127, max(-127, __float2int_rn(__fmul_rn(x, step))))) & 255u;
}

template <typename T>
__global__ void __launch_bounds__(512) append_kernel(const __grid_constant__ AppendParams<T> p) {
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
    if (s.length == 0 || s.count == 0 || nth < 0) return;
    const int32_t page_index = ((s.length - s.count) >> a.page_shift) + nth, page_tokens = 1 << a.page_shift, dim = a.head_dim;
    const int32_t from = max(s.length - s.count, page_index << a.page_shift), to = min(s.length, (page_index + 1) << a.page_shift);
    if (from >= to) return;
    const int32_t slot0 = from & (page_tokens - 1), row0 = from - (s.length - s.count) + s.first;
    const int32_t threads = blockDim.x, all = (to - from) * static_cast<int32_t>(p.units.d);
    const int64_t pitch = p.xs[which][0];
    const T* const x = p.x[which] + row0 * pitch + head * p.xs[which][1];
    const int32_t rotary = which == 0 ? p.rotary_dim : 0;

    auto load_unit = [&](int32_t i, float* f) {
        const int32_t t = static_cast<int32_t>(p.units.div(i)), unit = i - t * static_cast<int32_t>(p.units.d);
        const Unit u = unit_at(unit, rotary, p.interleaved);
        load8(x + t * pitch + u.low, p.vec[which], f);
        load8(x + t * pitch + u.high, p.vec[which], f + 8);
        if (u.rotated) {
            float cs[8], sn[8];
            load_turn(rope_row(p, from + t), unit, rotary, cs, sn);
            if (p.interleaved) turn(f, cs, sn, 1);
            else turn(f, cs, sn, 0);
        }
    };
    uint32_t m = 0;  // magnitudes as bits: ordered like the numbers, infinity and NaN above all
    auto largest_of = [&](const float* f) {
#pragma unroll
        for (int e = 0; e < 16; ++e) m = max(m, __float_as_uint(f[e]) & 0x7fffffffu);
    };
    float kept[kKeep][16];
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
        const int32_t i = threadIdx.x + k * threads;
        if (i < all) {
            load_unit(i, kept[k]);
            largest_of(kept[k]);
        }
    }
    for (int32_t i = threadIdx.x + kKeep * threads; i < all; i += threads) {  // blocks of more than 512 threads' units
        float f[16];
        load_unit(i, f);
        largest_of(f);
    }
    // only now the page: the elements are on the way meanwhile
    const int32_t page = kv_page(a, b, page_index);
    if (page < 0) return;
    const int64_t block = static_cast<int64_t>(page) * a.heads + head;
    int8_t* const codes = (which == 0 ? a.k_codes : a.v_codes) + block * page_tokens * dim;
    float* const scales = (which == 0 ? a.k_scales : a.v_scales) + block;
    const float before = slot0 == 0 ? 0.f : *scales;
    m = __reduce_max_sync(0xffffffffu, m);
    __shared__ uint32_t largest[16];
    if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < threads >> 5; ++w) m = max(m, largest[w]);
    float scale = __fmul_rn(__uint_as_float(m), 1.f / 127.f);
    if (scale < 1.17549435e-38f) scale = 0.f;
    scale = before > scale || before != before ? before : scale;
    if (m >= 0x7f800000u) scale = __uint_as_float(0x7fffffffu);
    if (threadIdx.x == 0) *scales = scale;
    if (scale > before) {  // earlier tokens of the block
        const float ratio = __fdiv_rn(before, scale);
        for (int32_t i = threadIdx.x * 16; i < slot0 * dim; i += threads * 16) {
            uint4 v = *reinterpret_cast<const uint4*>(codes + i);
            uint32_t* const w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t out = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    out |= (static_cast<uint32_t>(__float2int_rn(__fmul_rn(static_cast<float>(static_cast<int8_t>(w[k] >> (8 * e))), ratio))) & 255u) << (8 * e);
                w[k] = out;
            }
            *reinterpret_cast<uint4*>(codes + i) = v;
        }
    }
    const float step = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;  // NaN scales: codes 0
    auto store_unit = [&](int32_t i, const float* f) {
        const int32_t t = static_cast<int32_t>(p.units.div(i)), unit = i - t * static_cast<int32_t>(p.units.d);
        const Unit u = unit_at(unit, rotary, p.interleaved);
        int8_t* const y = codes + (slot0 + t) * dim;
        uint32_t w[4] = {0, 0, 0, 0};
        if (step > 0.f) {
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e >> 2] |= code_of(f[e], step) << (8 * (e & 3));
        }
        *reinterpret_cast<uint2*>(y + u.low) = make_uint2(w[0], w[1]);
        *reinterpret_cast<uint2*>(y + u.high) = make_uint2(w[2], w[3]);
    };
#pragma unroll
    for (int k = 0; k < kKeep; ++k) {
        const int32_t i = threadIdx.x + k * threads;
        if (i < all) store_unit(i, kept[k]);
    }
    for (int32_t i = threadIdx.x + kKeep * threads; i < all; i += threads) {
        float f[16];
        load_unit(i, f);
        store_unit(i, f);
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
        float f[16];
        if (t < there) {
            const uint4 v = ld_stream16(codes + i * 16);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] = __fmul_rn(static_cast<float>(static_cast<int8_t>(w[e >> 2] >> (8 * (e & 3)))), scale);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) f[e] = 0.f;
        }
        T* const y = out + t * s_token + unit * 16;
        store8(y, vec, f);
        store8(y + 8, vec, f + 8);
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
    p.q_heads = static_cast<int32_t>(q_heads);
    p.units = FastDiv(static_cast<uint32_t>(kv.head_dim / 16));
    p.blocks = 2 * kv.heads * (kv.starts ? (static_cast<int64_t>(kv.tokens) >> kv.page_shift) + 2 * static_cast<int64_t>(kv.seqs) : kv.seqs);
    // a whole block in the registers of a CTA, kKeep units a thread; single tokens need a warp or two
    const int units = (kv.starts ? 1 << kv.page_shift : 4) * (kv.head_dim / 16);
    const int threads = std::min(512, std::max(64, (units / kKeep + 31) / 32 * 32));
    p.heads = FastDiv(static_cast<uint32_t>(std::max<int64_t>(1, q_heads)));
    const int64_t row_units = std::max<int64_t>(1, q_heads * (kv.head_dim / 16));
    p.rows = static_cast<int32_t>(std::min<int64_t>(kMostRows, std::max<int64_t>(1, kKeep * threads / row_units)));
    const int64_t grid = p.blocks + (q ? (kv.tokens + p.rows - 1) / p.rows : 0);
    if (grid > 0x7fffffff || q_heads * kMostRows * (kv.head_dim / 16) > 0x7fffffff) return fail(MHLO_CUDA_UNSUPPORTED, "kv_cache_append: too many blocks");
    append_kernel<T><<<static_cast<unsigned>(grid), threads, 0, stream>>>(p);
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
