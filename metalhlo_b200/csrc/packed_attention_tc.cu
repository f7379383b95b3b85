// Attention over packed sequences on tcgen05: o = softmax(scale q k^T) v for bf16 / f16, head dimensions up to 128, grouped heads,
// causal or not, with the logarithms of the sums of exponentials. Scores do not leave the SM.
//
// A CTA takes items (tile of stacked query rows, head of keys) in the order of the batch's plan. A tile is two halves of 128 rows:
//   warp 0             producer: rows of q, then blocks of 128 keys and values through rings of two stages
//   warp 1             MMA issuer: S_h = Q_h K^T (both in shared memory), O_h += P_h V (P in tensor memory); one half's products run
//                      under the other's exponentials
//   warps 2-5, 6-9     softmax of half 0 / 1, a thread per row
// The maximum in the exponent moves only when scores exceed it by 2^8; O is rescaled in tensor memory only then.
// Weights are rounded once, to the type of the values, as their product has operands of one type (half a step: 2^-8 of a weight at most in bf16, 2^-11 in f16); sums of
// weights are those of the weights before that, in fp32. Sums of the rounded ones would leave the same error: it is that of each weight, not of their sum.
//
// Bound by the exponential unit beside the tensor pipe: a block of 128 x 128 needs 1024 clocks of either at D = 128 (of the tensor pipe 512 at 64). Causal,
// 32 query heads of 128 on 8, bf16: 24 sequences of up to 2048 tokens 417 us (958 TFLOP/s of what the mask leaves, the diagonal blocks' other half not
// counted), one of 16 384 1.73 ms (1270), at 1965 MHz (called on end, at 1.56 GHz and 1000 W, 499 us and 1.99 ms); either unit is busy for half of the time (50 and 52 %). A chain of a
// half, scores to weights to the next scores, is what both wait for; two run side by side, as many as tensor memory holds.
#include <algorithm>

#include "packed_tc.cuh"

namespace mhlo {
namespace {

constexpr int kStages = 2, kThreads = 32 * (2 + 4 * kHalves);
constexpr float kGrowth = 8.f;
// f16 weights go to their product times 2^7: growth to 2^8 of the reference leaves room for that below 2^16. Weights down to 2^-21 of the reference keep all their bits
// then, smaller ones are off by 2^-32 of it (unscaled, 16 000 keys 16 nats below another lost 6 % of what they add up to, scaled 0.1 %).
template <bool BF16>
constexpr float kUnit = BF16 ? 0.f : 7.f;
constexpr float kCarry = 32768.f;  // a row's sum of a block below this bounds every weight below the largest f16
constexpr int kWaitError = 60;     // + where a bounded wait ran out

struct ForwardParams {
    PackedArgs a;
    void* o;
    float* lse;
    int64_t os_token, os_head;
    float scale_log2;
    int32_t k_steps;    // head_dim / 16, rounded up
    int32_t one_half;   // items are half tiles: few rows, more CTAs
    int32_t wide;       // results 32 bytes at a time
    FastDiv by_group;
};

template <int D>
struct ForwardSmem {
    static constexpr int kTile = 128 * D * 2;
    static constexpr int kQ = 0, kK = kQ + kHalves * kTile, kV = kK + kStages * kTile, kEnd = kV + kStages * kTile, kTotal = kEnd + 1024;
};

// Two packed weights by alpha: through fp32, as alpha may be less than the smallest f16 number where their product is not.
template <bool BF16>
__device__ __forceinline__ uint32_t scale16x2(uint32_t v, float alpha) {
    float2 f;
    if constexpr (BF16) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
    else f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    return pack16<BF16>(f.x * alpha, f.y * alpha);
}

// 2^d of a whole number d <= 0 (-infinity: 0).
__device__ __forceinline__ float power_of_two(float d) { return d < -126.f ? 0.f : __uint_as_float(static_cast<uint32_t>(static_cast<int>(d) + 127) << 23); }

// Scores of 64 keys behind number `last` become -infinity.
__device__ __forceinline__ void hide(uint32_t* sr, int32_t last) {
    const uint64_t seen = last < 0 ? 0 : last >= 63 ? ~0ull : (2ull << last) - 1;
    const uint32_t lo = static_cast<uint32_t>(seen), hi = static_cast<uint32_t>(seen >> 32);
#pragma unroll
    for (int c = 0; c < 32; ++c) {
        if (!(lo >> c & 1)) sr[c] = 0xff800000u;
        if (!(hi >> c & 1)) sr[c + 32] = 0xff800000u;
    }
}

// A reference is a rounded product. Taken off the unrounded one, in one instruction, it leaves a difference that is common to all of a row's weights: nothing up to 2^22, beyond 2^27 more
// than f16 has room for, and all weights of a row could vanish. So the products are rounded like the reference first, where that costs nothing (head dimensions up to 64: 32 x 1024
// tokens, 12 heads, f16 108 and 109 us, 24 x 2048, 32 heads on 8, bf16 385 and 364; a branch for far rows 116 and 421) or where a reference is far (at 128, the slow way of a block:
// 414 and 417 us).
constexpr float kFar = 4194304.f;

// Weights of 64 scores, packed, and their sum: 2^(s * scale_log2 - m), m: the reference less the unit. ROUNDED: the products are rounded like the reference.
template <bool BF16, bool ROUNDED>
__device__ __forceinline__ void weights(const uint32_t* sr, float scale_log2, float m, uint32_t* packed, float2* sums) {
    const float2 c2 = make_float2(scale_log2, scale_log2), m2 = make_float2(-m, -m);
#pragma unroll
    for (int c = 0; c < 64; c += 2) {
        const float2 s = make_float2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
        const float2 x = ROUNDED ? __fadd2_rn(make_float2(__fmul_rn(s.x, scale_log2), __fmul_rn(s.y, scale_log2)), m2) : __ffma2_rn(s, c2, m2);
        const float2 e = make_float2(ex2(x.x), ex2(x.y));
        sums[(c >> 1) & 1] = __fadd2_rn(sums[(c >> 1) & 1], e);
        packed[c / 2] = pack16<BF16>(e.x, e.y);
    }
}

__device__ __forceinline__ float largest(const uint32_t* sr) {
    float a = -INFINITY, b = -INFINITY;
#pragma unroll
    for (int c = 0; c < 64; c += 4) {
        a = fmax3(a, __uint_as_float(sr[c]), __uint_as_float(sr[c + 1]));
        b = fmax3(b, __uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3]));
    }
    return fmaxf(a, b);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) packed_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                       const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ForwardParams p) {
    using L = ForwardSmem<D>;
    constexpr int kPanels = D / 64;
    // Tensor memory: scores 2 x 128 columns, O 2 x D. At D = 64 there is room for the weights beside the scores, so the scores of a
    // half's next block go out as soon as it has read those of this one; at 128 the weights lie over the scores.
    constexpr bool kBeside = D == 64;
    constexpr uint32_t kTmemCols = 512, kSCol = 0, kOCol = kHalves * 128, kPCol = kBeside ? kOCol + kHalves * D : kSCol, kPStride = kBeside ? 64 : 128;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t bars[7 * kHalves + 4 * kStages + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ ItemRing ring;
    uint64_t* const q_full = bars;                 // per half: the tile's rows of q are in shared memory
    uint64_t* const q_empty = q_full + kHalves;    // per half: their last product is done
    uint64_t* const s_full = q_empty + kHalves;    // per half: scores of a block are in tensor memory
    uint64_t* const s_free = s_full + kHalves;     // per half (kBeside): they have been read
    uint64_t* const p_full = s_free + kHalves;     // per half: the block's weights are, and O is rescaled if need be
    uint64_t* const pv_done = p_full + kHalves;    // per half: the products with values so far have completed
    uint64_t* const k_full = pv_done + kHalves;
    uint64_t* const k_empty = k_full + kStages;
    uint64_t* const v_full = k_empty + kStages;
    uint64_t* const v_empty = v_full + kStages;
    uint64_t* const own = v_empty + kStages;       // tiles that the producer waits for itself

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = p.a.half_tokens * p.a.group;  // of a half tile that hold a token
    if (tid == 0) {
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
        for (int h = 0; h < kHalves; ++h) {
            mbar_init(&q_full[h], 1);
            mbar_init(&q_empty[h], 1);
            mbar_init(&s_full[h], 1);
            mbar_init(&s_free[h], 4);
            mbar_init(&p_full[h], 4);
            mbar_init(&pv_done[h], 1);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        mbar_init(own, 1);
        ring.init(9);
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    // rows that no box brings hold numbers from the start
    for (int i = rows * 8 + tid; i < 128 * 8; i += kThreads) {
#pragma unroll
        for (int pn = 0; pn < kHalves * kPanels; ++pn) *reinterpret_cast<uint4*>(smem + L::kQ + pn * kPanelBytes + i * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    grid_dependency_wait();
    grid_dependency_release();
    bool ok = true;
    int4 entry;
    int32_t part;
    ItemSink sink(ring);
    auto next = [&](RowTile* t) {
        const bool more = sink.next(&entry, &part, &ok);
        if (more) *t = row_tile(p.a, p.one_half != 0, entry, part);
        else if (!ok) kv_report(kWaitError + 13);
        return more;
    };
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
        if (ok && !mbar_wait(bar, parity)) {
            kv_report(kWaitError + where);
            ok = false;
        }
        return ok;
    };

    if (warp == 0) {
        // ---- producer
        int stage = 0;
        uint32_t phase = 0, own_phase = 0, q_of[kHalves] = {0, 0};
        ItemSource source(ring, p.a, false, p.a.kv_heads * (p.one_half ? 2 : 1));
        auto take = [&]() { return source.next(&entry, &part, &ok, [&](const int4& e, int32_t i) { return row_tile(p.a, p.one_half != 0, e, i).nblk > 0; }); };
        bool more = take();
        while (more && ok) {
            const RowTile t = row_tile(p.a, p.one_half != 0, entry, part);
            more = take();
            for (int h = 0; h < kHalves; ++h) {
                if (t.nb[h] == 0) continue;
                if (!wait(&q_empty[h], (q_of[h]++ & 1) ^ 1, 0)) break;
                load_tile<kPanels>(smem + L::kQ + h * L::kTile, &map_q, &q_full[h], own, &own_phase, rows, rows, false, 0, t.head, t.first + t.t0 + h * p.a.half_tokens);
            }
            for (int j = 0; j < t.nblk && ok; ++j) {
                if (!wait(&k_empty[stage], phase ^ 1, 1)) break;
                load_tile<kPanels>(smem + L::kK + stage * L::kTile, &map_k, &k_full[stage], own, &own_phase, kKeyTile, kKeyTile, false, t.head, t.first + j * kKeyTile, 0);
                if (!wait(&v_empty[stage], phase ^ 1, 2)) break;
                if (!load_tile<kPanels>(smem + L::kV + stage * L::kTile, &map_v, &v_full[stage], own, &own_phase, kKeyTile, t.n - j * kKeyTile, true, t.head, t.first + j * kKeyTile, 0)) {
                    kv_report(kWaitError + 3);
                    ok = false;
                }
                if (++stage == kStages) stage = 0, phase ^= 1;
            }
        }
        if (!ok) {
            kv_report(kWaitError + 14);
            source.drain();
        }
    } else if (warp == 1) {
        // ---- MMA issuer
        const uint32_t idesc_s = instruction(BF16, false, kKeyTile), idesc_o = instruction(BF16, true, static_cast<uint32_t>(p.k_steps * 16));
        const uint32_t q_addr = smem_u32(smem + L::kQ), k_addr = smem_u32(smem + L::kK), v_addr = smem_u32(smem + L::kV);
        auto commit_to = [&](uint64_t* bar) {
            if (elect_one()) umma_commit(bar);
            __syncwarp();
        };
        auto issue_s = [&](int h, int stage) {
            tc_fence_after();
            if (elect_one()) {  // one thread issues all of a product's instructions: an election for each costs as much as the instruction
                const uint64_t da = make_smem_desc(q_addr + h * L::kTile, 16, 1024), db = make_smem_desc(k_addr + stage * L::kTile, 16, 1024);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    if (kk >= p.k_steps) break;
                    const uint32_t at = ((kk / 4) * kPanelBytes + (kk % 4) * 32) >> 4;
                    umma_f16(tmem + kSCol + h * 128, da + at, db + at, idesc_s, kk != 0 ? 1u : 0u);
                }
                umma_commit(&s_full[h]);
            }
            __syncwarp();
        };
        auto issue_pv = [&](int h, int stage, bool more) {
            tc_fence_after();
            if (elect_one()) {
                const uint64_t db = make_smem_desc(v_addr + stage * L::kTile, kPanelBytes, 1024);
#pragma unroll
                for (int kk = 0; kk < kKeyTile / 16; ++kk)
                    umma_ts(tmem + kOCol + h * D, tmem + kPCol + h * kPStride + kk * 8, db + (kk * 16 * 128 >> 4), idesc_o, more || kk != 0 ? 1u : 0u);
                umma_commit(&pv_done[h]);
            }
            __syncwarp();
        };
        RowTile cur, nxt;
        bool has = next(&cur);
        uint32_t block = 0;                              // blocks of keys so far
        uint32_t s_of[kHalves] = {0, 0}, p_of[kHalves] = {0, 0}, q_of[kHalves] = {0, 0};
        // The scores of block j of tile t, half h (whose turn it is), with the waits for what they read.
        auto scores = [&](const RowTile& t, int j, int h, uint32_t at) {
            const int stage = at % kStages;
            if (h == 0 && !wait(&k_full[stage], at / kStages & 1, 4)) return;
            if (j < t.nb[h]) {
                if (j == 0 && !wait(&q_full[h], q_of[h]++ & 1, 5)) return;
                // one arrival on s_free for each block of scores: those before have been read
                if (kBeside && s_of[h] > 0 && !wait(&s_free[h], (s_of[h] - 1) & 1, 6)) return;
                ++s_of[h];
                issue_s(h, stage);
                if (j + 1 == t.nb[h]) commit_to(&q_empty[h]);
            }
            if (h == kHalves - 1) commit_to(&k_empty[stage]);
        };
        auto values = [&](const RowTile& t, int j, int h, uint32_t at) {
            const int stage = at % kStages;
            if (h == 0 && !wait(&v_full[stage], at / kStages & 1, 7)) return;
            if (j < t.nb[h]) {
                if (!wait(&p_full[h], p_of[h]++ & 1, 8)) return;
                issue_pv(h, stage, j > 0);
            }
            if (h == kHalves - 1) commit_to(&v_empty[stage]);
        };
        if (has)
            for (int h = 0; h < kHalves && ok; ++h) scores(cur, 0, h, block);
        // Order on the pipe, which runs one thread's products in turn. Weights over the scores: PV_0(j), S_0(next), PV_1(j), S_1(next), so
        // that scores replace weights that have been read. Beside them: S_0(next), S_1(next), PV_0(j), PV_1(j).
        while (has && ok) {
            const bool more_tiles = next(&nxt);
            for (int j = 0; j < cur.nblk && ok; ++j, ++block) {
                const bool last = j + 1 == cur.nblk;
                const RowTile& next = last ? nxt : cur;
                const int nj = last ? 0 : j + 1;
                const bool more = !last || more_tiles;
                if (kBeside) {
                    for (int h = 0; h < kHalves && ok && more; ++h) scores(next, nj, h, block + 1);
                    for (int h = 0; h < kHalves && ok; ++h) values(cur, j, h, block);
                } else {
                    for (int h = 0; h < kHalves && ok; ++h) {
                        values(cur, j, h, block);
                        if (ok && more) scores(next, nj, h, block + 1);
                    }
                }
            }
            cur = nxt;
            has = more_tiles;
        }
    } else {
        // ---- softmax
        const int h = (warp - 2) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_taddr = tmem + lane_base + kSCol + h * 128, o_taddr = tmem + lane_base + kOCol + h * D, p_taddr = tmem + lane_base + kPCol + h * kPStride;
        uint32_t row_token, row_head;
        p.by_group.divmod(r, &row_token, &row_head);
        RowTile t;
        uint32_t it = 0;  // blocks of this half so far
        while (ok && next(&t)) {
            const int32_t i = t.t0 + h * p.a.half_tokens + row_token;  // the row's token
            const int32_t last = p.a.causal ? min(t.n - 1, i) : t.n - 1;
            const bool mine = r < rows && i < t.n;
            const int nb = t.nb[h];
            // what the warp's first and last row see: tokens ascend with the rows
            const int32_t least = __shfl_sync(0xffffffffu, last, 0), most = __shfl_sync(0xffffffffu, last, 31);
            float m_ref = -INFINITY, l = 0.f;  // m_ref: with the unit taken off
            for (int j = 0; j < nb; ++j, ++it) {
                if (!wait(&s_full[h], it & 1, 9)) break;
                tc_fence_after();
                const int32_t key0 = j * kKeyTile;
                float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                if constexpr (kBeside) {
                    bool pv_waited = it == 0;  // for the product of the block before this one, which reads its weights and adds to O
#pragma unroll 1
                    for (int ci = 0; ci < 2; ++ci) {
                        uint32_t sr[64], packed[32];
                        load64(s_taddr + ci * 64, sr);
                        if (ci == 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&s_free[h]);
                        }
                        // one decision a warp: loads and stores of tensor memory are warp-wide
                        if (key0 + ci * 64 + 63 > least) hide(sr, last - key0 - ci * 64);
                        const float mx = __fmul_rn(largest(sr), p.scale_log2);  // rounded for itself, as the weights of far rows are
                        const bool grow = mx - m_ref > kGrowth + kUnit<BF16>;
                        if (__any_sync(0xffffffffu, grow)) {
                            float alpha = 1.f;
                            if (grow) {
                                // by whole steps: weights that are rounded already follow by a power of two, which rounds them no further
                                const float top = mx - kUnit<BF16>, rise = ceilf(top - m_ref);
                                const bool whole = fabsf(top) <= kFar && rise <= kFar;  // else m_ref + rise may round to less than top; the first reference is top
                                alpha = whole ? power_of_two(-rise) : ex2(m_ref - top);
                                m_ref = whole ? m_ref + rise : top;
                                l *= alpha;
                            }
                            sums[0].x *= alpha, sums[0].y *= alpha, sums[1].x *= alpha, sums[1].y *= alpha;
                            if (j > 0 || ci > 0) {
                                if (!pv_waited) {
                                    if (!wait(&pv_done[h], (it - 1) & 1, 10)) break;
                                    tc_fence_after();
                                    pv_waited = true;
                                }
                                // O of the blocks before, then the weights of this block's first half
#pragma unroll 1
                                for (int c0 = j > 0 ? 0 : D; c0 < D + (ci > 0 ? 32 : 0); c0 += 32) {
                                    const uint32_t at = c0 < D ? o_taddr + c0 : p_taddr;
                                    uint32_t x[32];
                                    if (c0 >= D) tmem_st_wait();
                                    tmem_ld32(at, x);
                                    tmem_ld_wait();
#pragma unroll
                                    for (int c = 0; c < 32; ++c) x[c] = c0 < D ? __float_as_uint(__uint_as_float(x[c]) * alpha) : scale16x2<BF16>(x[c], alpha);
                                    tmem_st32(at, x);
                                }
                            }
                        }
                        weights<BF16, true>(sr, p.scale_log2, m_ref == -INFINITY ? 0.f : m_ref, packed, sums);
                        if (!pv_waited) {
                            if (!wait(&pv_done[h], (it - 1) & 1, 11)) break;
                            tc_fence_after();
                            pv_waited = true;
                        }
                        tmem_st32(p_taddr + ci * 32, packed);
                    }
                    if (!ok) break;
                    l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                } else {
                    // Against the maximum of earlier blocks, in a tile's first block that of its first 64 keys: nothing is written until the
                    // warp's sums have shown that no weight is too large for 16 bits. Otherwise the block's own maximum is found first.
                    uint32_t packed[2][32];
                    bool done = false;
                    float m_try = m_ref;
#pragma unroll
                    for (int ci = 0; ci < 2; ++ci) {
                        if (key0 + ci * 64 > most) {  // no row of the warp sees any of these
#pragma unroll
                            for (int c = 0; c < 32; ++c) packed[ci][c] = 0;
                            continue;
                        }
                        uint32_t sr[64];
                        load64(s_taddr + ci * 64, sr);
                        if (key0 + ci * 64 + 63 > least) hide(sr, last - key0 - ci * 64);
                        if (ci == 0 && j == 0) m_try = __fmul_rn(largest(sr), p.scale_log2) - kUnit<BF16>;
                        weights<BF16, false>(sr, p.scale_log2, m_try == -INFINITY ? 0.f : m_try, packed[ci], sums);
                    }
                    const float sum = (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                    done = !__any_sync(0xffffffffu, mine && !(sum < kCarry && fabsf(m_try) <= kFar));  // rows that are another sequence's have no say
                    if (done) {
                        l += sum;
                        m_ref = m_try;
#pragma unroll
                        for (int ci = 0; ci < 2; ++ci) tmem_st32(p_taddr + ci * 32, packed[ci]);
                    }
                    if (!done) {
                        float mx = -INFINITY;
#pragma unroll 1
                        for (int ci = 0; ci < 2; ++ci) {
                            uint32_t sr[64];
                            if (key0 + ci * 64 > most) break;
                            load64(s_taddr + ci * 64, sr);
                            if (key0 + ci * 64 + 63 > least) hide(sr, last - key0 - ci * 64);
                            mx = fmaxf(mx, largest(sr));
                        }
                        mx = __fmul_rn(mx, p.scale_log2);
                        const bool grow = mx - m_ref > kGrowth + kUnit<BF16>;
                        float alpha = 1.f;
                        if (grow) {
                            const float next = mx - kUnit<BF16>;
                            alpha = m_ref == -INFINITY ? 0.f : ex2(m_ref - next);
                            m_ref = next;
                            l *= alpha;
                        }
                        // the products so far completed before these scores did
                        if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
                            for (int c0 = 0; c0 < D; c0 += 32) {
                                uint32_t x[32];
                                tmem_ld32(o_taddr + c0, x);
                                tmem_ld_wait();
#pragma unroll
                                for (int c = 0; c < 32; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * alpha);
                                tmem_st32(o_taddr + c0, x);
                            }
                        }
                        sums[0] = sums[1] = make_float2(0.f, 0.f);
#pragma unroll 1
                        for (int ci = 0; ci < 2; ++ci) {  // the weights lie over scores that have been read
                            uint32_t sr[64];
                            load64(s_taddr + ci * 64, sr);
                            if (key0 + ci * 64 + 63 > least) hide(sr, last - key0 - ci * 64);
                            weights<BF16, true>(sr, p.scale_log2, m_ref == -INFINITY ? 0.f : m_ref, packed[0], sums);
                            tmem_st32(p_taddr + ci * 32, packed[0]);
                        }
                        l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[h]);
            }
            if (!ok || nb == 0) continue;
            // ---- results. The next tile's first product with values waits for weights that these warps write after this.
            if (!wait(&pv_done[h], (it - 1) & 1, 12)) break;
            tc_fence_after();
            const int64_t token = t.first + i, head = t.head * p.a.group + row_head;
            const float inv = l == 0.f ? 0.f : 1.f / l;
            uint8_t* const to = static_cast<uint8_t*>(p.o) + (token * p.os_token + head * p.os_head) * 2;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                if (c0 >= p.a.head_dim) break;
                uint32_t x[32];
                tmem_ld32(o_taddr + c0, x);
                tmem_ld_wait();
                if (mine) store_result<BF16>(to, x, inv, c0, p.a.head_dim, p.wide != 0);
            }
            if (mine && p.lse != nullptr) p.lse[token * p.a.q_heads + head] = l == 0.f ? -INFINITY : (m_ref + log2f(l)) * kLn2;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <int D, bool BF16>
int launch(const PackedCall& c, cudaStream_t stream) {
    using L = ForwardSmem<D>;
    const PackedArgs& a = c.a;
    CUtensorMap mq, mk, mv;
    if (int st = query_map(&mq, c.q, a)) return st;
    if (int st = key_map(&mk, c.k, a)) return st;
    if (int st = key_map(&mv, c.v, a)) return st;
    ForwardParams p;
    p.a = a;
    p.o = c.o.base;
    p.lse = c.lse;
    p.os_token = c.o.token;
    p.os_head = c.o.head;
    p.scale_log2 = c.scale * kLog2e;
    p.k_steps = (a.head_dim + 15) / 16;
    const int64_t items = static_cast<int64_t>(a.row_capacity) * a.kv_heads;
    p.one_half = 2 * items <= kNumSMs;
    p.wide = on_wide_grid(c.o, a.head_dim, a.tokens, a.q_heads);
    p.by_group = FastDiv(static_cast<uint32_t>(a.group));
    static std::atomic<bool> allowed[64];
    auto kernel = packed_attention_kernel<D, BF16>;
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), L::kTotal, allowed)) return st;
    const unsigned grid = static_cast<unsigned>(items * (p.one_half ? 2 : 1));
    const cudaError_t e = launch_dependent(kernel, dim3(grid), dim3(kThreads), L::kTotal, stream, 1, grid < kNumSMs, mq, mk, mv, p);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of packed_attention failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("packed_attention");
    return MHLO_CUDA_OK;
}

}  // namespace

int packed_attention_tc(const PackedCall& c, cudaStream_t stream) {
    const bool bf16 = c.dtype == MHLO_DT_BF16;
    if (c.a.head_dim <= 64) return bf16 ? launch<64, true>(c, stream) : launch<64, false>(c, stream);
    return bf16 ? launch<128, true>(c, stream) : launch<128, false>(c, stream);
}

int packed_attention_tc_device_error() { return take_kv_error(); }

}  // namespace mhlo
