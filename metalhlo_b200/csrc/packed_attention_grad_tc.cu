// Gradients of attention over packed sequences on tcgen05, bf16 / f16, head dimensions up to 128: two kernels, each of which takes the scores
// again and sums in the order of its blocks, so that no atomics are needed and the same inputs give the same bits:
//   key_grads    128 keys a CTA, over the blocks of stacked query rows that see them (all heads of the group, one below the other):
//                S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//   query_grads  128 query rows, over the blocks of keys that they see: S = Q K^T, dP = dO V^T, dQ += dS K
// with P = 2^(scale log2(e) S - lse log2(e)) and dS = P (dP - delta). That is seven products where five would do; the two more cost less than
// adding dQ up in memory, and nothing of them depends on an order of arrival.
//
// Threads hold a row of the tile in tensor memory. P and dS go over the scores and dP they came from and are the A operands of the products that
// follow, so they never pass through shared memory.
//   warp 0             producer (bulk tensor loads; rows behind a sequence's end become zeros, as they would be summed over)
//   warp 1             MMA issuer
//   warps 2-5, 6-9     exponentials: columns 0-63 / 64-127 of a block
// At D = 64 a block goes in two steps of 64 columns with warps 2-5 alone, in half of the tensor memory: two CTAs share an SM, and each works while the other
// waits for its chain - scores, exponentials, dP, dS, sums.
//
// Times: 3 causal sequences of up to 8192 tokens, 32 query heads of 128 on 8, bf16: 1.18 ms the keys, 0.86 to 0.92 the queries (1260 TFLOP/s of what they compute
// where the mask leaves something; the tensor pipe is busy for 67 %). 32 of 1024, 12 heads of 64, f16: 0.192 and 0.137 ms (0.181 and 0.128 with one power of two for all of the call, see below); 0.200 and
// 0.147 with one CTA to an SM, which
// none of these changed by more than a few percent: products of the next tile issued ahead with results stored under them (keys 0, queries -5 %, at D = 128
// +5 %), the two warpgroups' exponentials in turn, loads of tensor memory a half ahead (0), a quarter of the exponentials by a polynomial (+2 %), sixteen warps
// of exponentials (0), results through shared memory or by warps of their own (0).
// P and dS are rounded to the type of q and of the gradient, as operands of one product are of one type: 2^-8 of each at most in bf16, 2^-11 in f16, beside which
// the results' own rounding counts the same.
// f16 keeps numbers between 2^-14 and 2^16 whole. P goes to the product times 2^14, dS times a power of two that brings the largest possible one below 2^15; both are
// undone in the results. The power is a result row's own, as the sum over a row of dS or of dS^T has to have one: for a query 2 |grad| max|v|, for a key
// max|grad| (|v| + max|v|), each maximum over its sequence (delta is grad times weighted values). Taken over all of the call, sequences whose gradients are 2^20 smaller
// than another's were left with no bits.
#include <algorithm>

#include "packed_tc.cuh"

namespace mhlo {
namespace {

constexpr int kWaitKeys = 70, kWaitQueries = 90;
constexpr float kUnit = 16384.f;  // of P in fp16

// A block of 128 goes in kParts steps of kWide columns.
template <int D>
struct Shape {
    static constexpr int kParts = D == 64 ? 2 : 1, kWide = 128 / kParts, kWarps = 8 / kParts, kThreads = 64 + 32 * kWarps, kCtas = kParts;
    static constexpr uint32_t kTmem = 4 * kWide;  // columns
};

struct GradParams {
    PackedArgs a;
    const float2* stats;
    const float2* largest;  // f16: see PackedCall
    const float *grad_norms, *value_norms;
    void *dq, *dk, *dv;
    float* shares;   // where the rows of a tile of keys are cut into splits: their sums, [splits][dk, dv][tokens][kv_heads][head_dim]
    int32_t splits;
    int64_t dq_token, dq_head, dk_token, dk_head, dv_token, dv_head;
    float scale, scale_log2;
    int32_t k_steps;  // head_dim / 16, rounded up
    int32_t wide;     // results 32 bytes at a time
};

// The power of two that brings numbers of up to `most` below 2^15.
__device__ __forceinline__ float unit_of(float most) {
    if (!(most > 0.f) || most > 1e38f) return 1.f;
    const int exponent = static_cast<int>(__float_as_uint(most) >> 23) - 127;  // most < 2^(exponent + 1)
    return ldexpf(1.f, min(14 - exponent, 100));
}

// Weights of 32 scores: 2^(s scale_log2 + offset), offset(c) of column pair c.
template <typename Offset>
__device__ __forceinline__ void weights(const uint32_t* s, float scale_log2, float* w, Offset offset) {
    const float2 c2 = make_float2(scale_log2, scale_log2);
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
        const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), c2, offset(c));
        w[c] = ex2(x.x);
        w[c + 1] = ex2(x.y);
    }
}
template <bool BF16>
__device__ __forceinline__ void store_packed(uint32_t taddr, const float* w) {
    uint32_t packed[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) packed[c] = pack16<BF16>(w[2 * c], w[2 * c + 1]);
    tmem_st16(taddr, packed);
}

// One thread's products of a warp-uniform schedule.
struct Issuer {
    int k_steps;
    __device__ __forceinline__ void commit(uint64_t* bar) const {
        if (elect_one()) umma_commit(bar);
        __syncwarp();
    }
    // d = a b^T over head_dim, both tiles [128][head_dim] in shared memory; bar is arrived on when all products so far are done. One thread
    // issues all of a product's instructions: with an election for each the issuer was what bounded D = 64.
    template <int D>
    __device__ __forceinline__ void rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint64_t* bar) const {
        tc_fence_after();
        if (elect_one()) {
            const uint64_t da = make_smem_desc(a, 16, 1024), db = make_smem_desc(b, 16, 1024);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                if (kk >= k_steps) break;
                const uint32_t at = ((kk / 4) * kPanelBytes + (kk % 4) * 32) >> 4;
                umma_f16(d, da + at, db + at, idesc, kk != 0 ? 1u : 0u);
            }
            umma_commit(bar);
        }
        __syncwarp();
    }
    // d += a b over COLUMNS columns of a: a in tensor memory, 64 packed columns from a on and 64 from a + 64 on; b [COLUMNS][head_dim] in shared memory
    template <int COLUMNS>
    __device__ __forceinline__ void columns(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool more) const {
        tc_fence_after();
        if (elect_one()) {
            const uint64_t db = make_smem_desc(b, kPanelBytes, 1024);
#pragma unroll
            for (int kk = 0; kk < COLUMNS / 16; ++kk) umma_ts(d, a + (kk / 4) * 64 + (kk % 4) * 8, db + (kk * 16 * 128 >> 4), idesc, more || kk != 0 ? 1u : 0u);
        }
        __syncwarp();
    }
};

// ---- keys and values ------------------------------------------------------------------------------------------------------------------
// The pipe runs dV(j), S(j + 1) while the threads turn dP(j) into dS(j), and dK(j), dP(j + 1) under the exponentials of j + 1: with two
// regions of a step's columns beside the two sums each product finds its region free.
template <int D>
struct KeySmem {
    static constexpr int kTile = 128 * D * 2, kStages = 2;
    static constexpr int kK = 0, kV = kTile, kQ = 2 * kTile, kG = kQ + kStages * kTile, kEnd = kG + kStages * kTile, kTotal = kEnd + 1024;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(Shape<D>::kThreads, Shape<D>::kCtas) key_grads_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                                                                const __grid_constant__ GradParams p) {
    using L = KeySmem<D>;
    constexpr int kPanels = D / 64, kStages = L::kStages, kParts = Shape<D>::kParts, kWide = Shape<D>::kWide, kWarps = Shape<D>::kWarps, kThreads = Shape<D>::kThreads;
    constexpr uint32_t kS = 0, kP = kWide, kDv = 2 * kWide, kDk = 2 * kWide + D, kPartBytes = kWide * 128;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ __align__(16) float minus_lse[kStages][128];
    __shared__ __align__(16) float minus_delta[kStages][128];
    __shared__ uint64_t bars[9 + 4 * kStages];
    __shared__ uint32_t tmem_slot;
    __shared__ ItemRing ring;
    uint64_t* const kv_full = bars;
    uint64_t* const kv_empty = bars + 1;
    uint64_t* const s_full = bars + 2;    // scores of a block are in tensor memory
    uint64_t* const p_full = bars + 3;    // its weights are
    uint64_t* const dp_full = bars + 4;
    uint64_t* const ds_full = bars + 5;
    uint64_t* const sums_full = bars + 6; // the tile's sums are complete
    uint64_t* const sums_free = bars + 7; // they have been read
    uint64_t* const own = bars + 8;
    uint64_t* const q_full = bars + 9;
    uint64_t* const g_full = q_full + kStages;
    uint64_t* const stats_full = g_full + kStages;
    uint64_t* const empty = stats_full + kStages;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = p.a.half_tokens * p.a.group;
    if (tid == 0) {
        mbar_init(kv_full, 2);
        mbar_init(kv_empty, 1);
        mbar_init(s_full, 1);
        mbar_init(p_full, kWarps);
        mbar_init(dp_full, 1);
        mbar_init(ds_full, kWarps);
        mbar_init(sums_full, 1);
        mbar_init(sums_free, kWarps);
        mbar_init(own, 1);
        ring.init(1 + kWarps);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&g_full[s], 1);
            mbar_init(&stats_full[s], 1);
            mbar_init(&empty[s], 1);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, Shape<D>::kTmem);
        tmem_relinquish();
    }
    // rows that no box brings are summed over with weights of zero
    for (int i = rows * 8 + tid; i < 128 * 8; i += kThreads) {
#pragma unroll
        for (int pn = 0; pn < 2 * kStages * kPanels; ++pn) *reinterpret_cast<uint4*>(smem + L::kQ + pn * kPanelBytes + i * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    grid_dependency_wait();
    grid_dependency_release();
    KeyTile t;
    bool ok = true;
    int4 entry;
    int32_t part;
    ItemSink sink(ring);
    auto next = [&]() {
        const bool more = sink.next(&entry, &part, &ok);
        if (more) t = key_tile(p.a, p.splits, entry, part);
        else if (!ok) kv_report(kWaitKeys + 13);
        return more;
    };
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
        if (ok && !mbar_wait(bar, parity)) {
            kv_report(kWaitKeys + where);
            ok = false;
        }
        return ok;
    };

    if (warp == 0) {
        // ---- producer
        uint32_t item = 0, block = 0, own_phase = 0;
        auto failed = [&]() {
            kv_report(kWaitKeys + 9);
            ok = false;
        };
        ItemSource source(ring, p.a, true, p.a.kv_heads * p.splits);
        auto take = [&]() { return source.next(&entry, &part, &ok, [](const int4&, int32_t) { return true; }); };
        bool rest = take();
        while (rest && ok) {
            t = key_tile(p.a, p.splits, entry, part);
            rest = take();
            for (int32_t b = t.b0; b < t.b1 && ok; ++b, ++block) {
                const int stage = block % kStages;
                const int32_t token0 = b * p.a.half_tokens, valid = min(rows, (t.n - token0) * p.a.group);
                if (!wait(&empty[stage], (block / kStages & 1) ^ 1, 0)) break;
                if (!load_tile<kPanels>(smem + L::kQ + stage * L::kTile, &map_q, &q_full[stage], own, &own_phase, rows, valid, true, 0, t.head, t.first + token0)) failed();
                if (b == t.b0) {  // rows behind the end go no further than their own rows of the sums
                    if (!wait(kv_empty, (item & 1) ^ 1, 1)) break;
                    ++item;
                    load_tile<kPanels>(smem + L::kK, &map_k, kv_full, own, &own_phase, kKeyTile, kKeyTile, false, t.head, t.first + t.k0, 0);
                    load_tile<kPanels>(smem + L::kV, &map_v, kv_full, own, &own_phase, kKeyTile, kKeyTile, false, t.head, t.first + t.k0, 0);
                }
                if (ok && !load_tile<kPanels>(smem + L::kG + stage * L::kTile, &map_g, &g_full[stage], own, &own_phase, rows, valid, true, 0, t.head, t.first + token0)) failed();
                const float2* const from = p.stats + (static_cast<int64_t>(t.head) * p.a.tokens + t.first + token0) * p.a.group;
#pragma unroll
                for (int r = lane; r < 128; r += 32) {
                    const float2 s = r < valid ? from[r] : make_float2(-INFINITY, 0.f);
                    minus_lse[stage][r] = s.x + (BF16 ? 0.f : 14.f);
                    minus_delta[stage][r] = -s.y;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&stats_full[stage]);
            }
        }
        if (!ok) {
            kv_report(kWaitKeys + 14);
            source.drain();
        }
    } else if (warp == 1) {
        // ---- MMA issuer
        const Issuer mma{p.k_steps};
        const uint32_t idesc_rows = instruction(BF16, false, kWide), idesc_cols = instruction(BF16, true, static_cast<uint32_t>(p.k_steps * 16));
        const uint32_t k_addr = smem_u32(smem + L::kK), v_addr = smem_u32(smem + L::kV), q_addr = smem_u32(smem + L::kQ), g_addr = smem_u32(smem + L::kG);
        uint32_t item = 0, step = 0;
        auto tile = [&](uint32_t base, uint32_t at) { return base + at / kParts % kStages * L::kTile + at % kParts * kPartBytes; };
        auto scores = [&](uint32_t at) {
            if (!wait(&q_full[at / kParts % kStages], at / kParts / kStages & 1, 2)) return;
            mma.rows<D>(tmem + kS, k_addr, tile(q_addr, at), idesc_rows, s_full);
        };
        auto grads = [&](uint32_t at) {
            if (!wait(&g_full[at / kParts % kStages], at / kParts / kStages & 1, 3)) return;
            mma.rows<D>(tmem + kP, v_addr, tile(g_addr, at), idesc_rows, dp_full);
        };
        while (ok && next()) {
            const int32_t steps = (t.b1 - t.b0) * kParts;
            if (steps == 0) continue;
            if (!wait(kv_full, item & 1, 4)) break;
            scores(step);
            if (ok) grads(step);
            if (steps == 1) mma.commit(kv_empty);
            for (int32_t i = 0; i < steps && ok; ++i, ++step) {
                const bool more = i + 1 < steps;
                if (!wait(p_full, step & 1, 5)) break;
                if (i == 0 && item > 0 && !wait(sums_free, (item - 1) & 1, 6)) break;
                mma.columns<kWide>(tmem + kDv, tmem + kS, tile(g_addr, step), idesc_cols, i > 0);
                if (more) scores(step + 1);
                if (!wait(ds_full, step & 1, 7)) break;
                mma.columns<kWide>(tmem + kDk, tmem + kP, tile(q_addr, step), idesc_cols, i > 0);
                if (step % kParts == kParts - 1) mma.commit(&empty[step / kParts % kStages]);
                if (more) {
                    grads(step + 1);
                    if (i + 2 == steps) mma.commit(kv_empty);
                }
            }
            if (ok) mma.commit(sums_full);
            ++item;
        }
    } else {
        // ---- exponentials
        const int half = (warp - 2) >> 2, quarter = warp & 3, r = quarter * 32 + lane;  // half: 0 where there are four warps
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_taddr = tmem + lane_base + kS + half * 64, p_taddr = tmem + lane_base + kP + half * 64;
        uint32_t item = 0, step = 0;
        while (ok && next()) {
            const int32_t steps = (t.b1 - t.b0) * kParts;
            // this thread's key: the norm of its value, and the power of two of its sum
            const int64_t of_head = static_cast<int64_t>(t.head) * p.a.tokens + t.first;
            const float2 most = BF16 ? make_float2(0.f, 0.f) : p.largest[of_head];
            const float v = !BF16 && t.k0 + r < t.n ? p.value_norms[of_head + t.k0 + r] : 0.f;
            float unit = 1.f, from_dp = 1.f;
            for (int32_t i = 0; i < steps; ++i, ++step) {
                const uint32_t block = step / kParts, stage = block % kStages;
                const int32_t token0 = (t.b0 + i / kParts) * p.a.half_tokens, part = kParts == 2 ? step % 2 : half;
                // columns below hidden are rows of earlier tokens than this thread's key
                const int32_t hidden = p.a.causal && t.k0 + kKeyTile - 1 > token0 ? (t.k0 + r - token0) * p.a.group - part * 64 : 0;
                const bool mask = __any_sync(0xffffffffu, hidden > 0);
                if (!wait(&stats_full[stage], block / kStages & 1, 8) || !wait(s_full, step & 1, 10)) break;
                tc_fence_after();
                if (!BF16 && i == 0) {
                    unit = unit_of(most.x * (v + most.y));
                    from_dp = unit / kUnit;
                }
                const float *const lse = minus_lse[stage] + part * 64, *const delta = minus_delta[stage] + part * 64;
                float w[64];
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t s[32];
                    tmem_ld32(s_taddr + c0, s);
                    tmem_ld_wait();
                    if (mask) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (c0 + c < hidden) s[c] = 0xff800000u;
                    }
                    weights(s, p.scale_log2, w + c0, [&](int c) { return *reinterpret_cast<const float2*>(lse + c0 + c); });
                }
                // over the scores that this thread has read
                store_packed<BF16>(s_taddr, w);
                store_packed<BF16>(s_taddr + 16, w + 32);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
                if (!wait(dp_full, step & 1, 11)) break;
                tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t g[32];
                    tmem_ld32(p_taddr + c0, g);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        float2 x = *reinterpret_cast<const float2*>(delta + c0 + c);
                        x = __fadd2_rn(make_float2(__uint_as_float(g[c]), __uint_as_float(g[c + 1])), x);
                        if (!BF16) x = __fmul2_rn(x, make_float2(from_dp, from_dp));
                        x = __fmul2_rn(x, make_float2(w[c0 + c], w[c0 + c + 1]));
                        w[c0 + c] = x.x;
                        w[c0 + c + 1] = x.y;
                    }
                    store_packed<BF16>(p_taddr + c0 / 2, w + c0);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_full);
            }
            // ---- results: dV, dK; of two warpgroups each takes one
            const bool any = t.b0 < t.b1, mine = t.k0 + r < t.n;
            if (!ok || (any && !wait(sums_full, item & 1, 12))) break;
            tc_fence_after();
            const int64_t token = t.first + t.k0 + r;
#pragma unroll 1
            for (int which = half; which < (kParts == 2 ? 2 : half + 1); ++which) {
                const float factor = which == 0 ? (BF16 ? 1.f : 1.f / kUnit) : p.scale / unit;
                const uint32_t sums = tmem + lane_base + (which == 0 ? kDv : kDk);
                if (p.splits > 1) {
                    float* const to = p.shares + (((static_cast<int64_t>(t.split) * 2 + 1 - which) * p.a.tokens + token) * p.a.kv_heads + t.head) * p.a.head_dim;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        if (c0 >= p.a.head_dim) break;
                        uint32_t x[32];
                        if (any) {
                            tmem_ld32(sums + c0, x);
                            tmem_ld_wait();
                        }
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (any) v = make_float4(__uint_as_float(x[c]) * factor, __uint_as_float(x[c + 1]) * factor, __uint_as_float(x[c + 2]) * factor, __uint_as_float(x[c + 3]) * factor);
                            if (mine && c0 + c < p.a.head_dim) *reinterpret_cast<float4*>(to + c0 + c) = v;
                        }
                    }
                } else {
                    uint8_t* const to = which == 0 ? static_cast<uint8_t*>(p.dv) + (token * p.dv_token + t.head * p.dv_head) * 2
                                                   : static_cast<uint8_t*>(p.dk) + (token * p.dk_token + t.head * p.dk_head) * 2;
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        if (c0 >= p.a.head_dim) break;
                        uint32_t x[32];
                        tmem_ld32(sums + c0, x);
                        tmem_ld_wait();
                        if (mine) store_result<BF16>(to, x, factor, c0, p.a.head_dim, p.wide != 0);
                    }
                }
            }
            if (!any) continue;
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sums_free);
            ++item;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Shape<D>::kTmem);
    }
}

// ---- queries ----------------------------------------------------------------------------------------------------------------------------
// Three regions of a step's columns beside dQ take turns: S(t) in region 2 t, dP(t) and dS(t) in 2 t + 1 (mod 3). Scores of the next step are
// there before the threads get to it, and its dP goes where this step's scores were as soon as they have been read.
template <int D>
struct QuerySmem {
    static constexpr int kTile = 128 * D * 2, kKStages = D == 64 ? 2 : 3, kVStages = 2;
    static constexpr int kQ = 0, kG = kTile, kK = 2 * kTile, kV = kK + kKStages * kTile, kEnd = kV + kVStages * kTile, kTotal = kEnd + 1024;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(Shape<D>::kThreads, Shape<D>::kCtas) query_grads_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g,
                                                                  const __grid_constant__ GradParams p) {
    using L = QuerySmem<D>;
    constexpr int kPanels = D / 64, kKS = L::kKStages, kVS = L::kVStages, kParts = Shape<D>::kParts, kWide = Shape<D>::kWide, kWarps = Shape<D>::kWarps;
    constexpr uint32_t kDq = 0, kRegion = D, kPartBytes = kWide * 128;
    static_assert(kRegion + 3 * kWide <= Shape<D>::kTmem, "columns of tensor memory");
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t bars[14 + 2 * kKS + 2 * kVS];
    __shared__ uint32_t tmem_slot;
    __shared__ ItemRing ring;
    uint64_t* const q_full = bars;
    uint64_t* const g_full = bars + 1;
    uint64_t* const qg_empty = bars + 2;
    // Steps take turns at two barriers each: products of the next one may complete before a warp has looked for this one's, and a
    // wait knows a phase only from its neighbours.
    uint64_t* const s_full = bars + 3;
    uint64_t* const s_free = bars + 5;  // the scores of a block have been read
    uint64_t* const dp_full = bars + 7;
    uint64_t* const ds_full = bars + 9;
    uint64_t* const sums_full = bars + 11;
    uint64_t* const sums_free = bars + 12;
    uint64_t* const own = bars + 13;
    uint64_t* const k_full = bars + 14;
    uint64_t* const k_empty = k_full + kKS;
    uint64_t* const v_full = k_empty + kKS;
    uint64_t* const v_empty = v_full + kVS;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = p.a.half_tokens * p.a.group;
    if (tid == 0) {
        mbar_init(q_full, 1);
        mbar_init(g_full, 1);
        mbar_init(qg_empty, 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&s_full[s], 1);
            mbar_init(&s_free[s], kWarps);
            mbar_init(&dp_full[s], 1);
            mbar_init(&ds_full[s], kWarps);
        }
        mbar_init(sums_full, 1);
        mbar_init(sums_free, kWarps);
        mbar_init(own, 1);
        ring.init(1 + kWarps);
        for (int s = 0; s < kKS; ++s) {
            mbar_init(&k_full[s], 1);
            mbar_init(&k_empty[s], 1);
        }
        for (int s = 0; s < kVS; ++s) {
            mbar_init(&v_full[s], 1);
            mbar_init(&v_empty[s], 1);
        }
        fence_barrier_init();
    }
    if (warp == 1) {
        tmem_alloc(&tmem_slot, Shape<D>::kTmem);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    grid_dependency_wait();
    grid_dependency_release();
    RowTile t;
    bool ok = true;
    int4 entry;
    int32_t part;
    ItemSink sink(ring);
    auto next = [&]() {
        const bool more = sink.next(&entry, &part, &ok);
        if (more) t = row_tile(p.a, true, entry, part);
        else if (!ok) kv_report(kWaitQueries + 14);
        return more;
    };
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
        if (ok && !mbar_wait(bar, parity)) {
            kv_report(kWaitQueries + where);
            ok = false;
        }
        return ok;
    };

    if (warp == 0) {
        // ---- producer
        uint32_t item = 0, block = 0, own_phase = 0;
        auto failed = [&]() {
            kv_report(kWaitQueries + 9);
            ok = false;
        };
        ItemSource source(ring, p.a, false, p.a.kv_heads * 2);
        auto take = [&]() { return source.next(&entry, &part, &ok, [&](const int4& e, int32_t i) { return row_tile(p.a, true, e, i).nblk > 0; }); };
        bool rest = take();
        while (rest && ok) {
            t = row_tile(p.a, true, entry, part);
            rest = take();
            for (int32_t b = 0; b < t.nblk && ok; ++b, ++block) {
                const int32_t valid = t.n - b * kKeyTile, ks = block % kKS, vs = block % kVS;
                if (!wait(&k_empty[ks], (block / kKS & 1) ^ 1, 0)) break;
                if (!load_tile<kPanels>(smem + L::kK + ks * L::kTile, &map_k, &k_full[ks], own, &own_phase, kKeyTile, valid, true, t.head, t.first + b * kKeyTile, 0)) failed();
                if (b == 0) {  // rows that are not the tile's go no further than their own rows of dQ
                    if (!wait(qg_empty, (item & 1) ^ 1, 1)) break;
                    ++item;
                    load_tile<kPanels>(smem + L::kQ, &map_q, q_full, own, &own_phase, rows, rows, false, 0, t.head, t.first + t.t0);
                    load_tile<kPanels>(smem + L::kG, &map_g, g_full, own, &own_phase, rows, rows, false, 0, t.head, t.first + t.t0);
                }
                if (!wait(&v_empty[vs], (block / kVS & 1) ^ 1, 2)) break;
                if (!load_tile<kPanels>(smem + L::kV + vs * L::kTile, &map_v, &v_full[vs], own, &own_phase, kKeyTile, valid, true, t.head, t.first + b * kKeyTile, 0)) failed();
            }
        }
        if (!ok) {
            kv_report(kWaitQueries + 9);
            source.drain();
        }
    } else if (warp == 1) {
        // ---- MMA issuer
        const Issuer mma{p.k_steps};
        const uint32_t idesc_rows = instruction(BF16, false, kWide), idesc_cols = instruction(BF16, true, static_cast<uint32_t>(p.k_steps * 16));
        const uint32_t k_addr = smem_u32(smem + L::kK), v_addr = smem_u32(smem + L::kV), q_addr = smem_u32(smem + L::kQ), g_addr = smem_u32(smem + L::kG);
        uint32_t item = 0, step = 0;
        auto region = [&](uint32_t i) { return tmem + kRegion + i % 3 * kWide; };
        auto key_tile_at = [&](uint32_t at) { return k_addr + at / kParts % kKS * L::kTile + at % kParts * kPartBytes; };
        auto scores = [&](uint32_t at) {
            if (!wait(&k_full[at / kParts % kKS], at / kParts / kKS & 1, 3)) return;
            mma.rows<D>(region(2 * at), q_addr, key_tile_at(at), idesc_rows, &s_full[at & 1]);
        };
        auto grads = [&](uint32_t at) {
            const uint32_t stage = at / kParts % kVS;
            if (!wait(&v_full[stage], at / kParts / kVS & 1, 4)) return;
            mma.rows<D>(region(2 * at + 1), g_addr, v_addr + stage * L::kTile + at % kParts * kPartBytes, idesc_rows, &dp_full[at & 1]);
            if (at % kParts == kParts - 1) mma.commit(&v_empty[stage]);
        };
        while (ok && next()) {
            const int32_t steps = t.nblk * kParts;
            if (!wait(q_full, item & 1, 5)) break;
            scores(step);
            if (!wait(g_full, item & 1, 6)) break;
            // the region of this dP held the last item's last scores, which were read before its last dS
            if (ok) grads(step);
            if (steps == 1) mma.commit(qg_empty);
            for (int32_t i = 0; i < steps && ok; ++i, ++step) {
                if (i + 1 < steps) {
                    scores(step + 1);
                    if (!wait(&s_free[step & 1], step >> 1 & 1, 7)) break;
                    grads(step + 1);
                    if (i + 2 == steps) mma.commit(qg_empty);
                }
                if (!wait(&ds_full[step & 1], step >> 1 & 1, 8)) break;
                if (i == 0 && item > 0 && !wait(sums_free, (item - 1) & 1, 10)) break;
                mma.columns<kWide>(tmem + kDq, region(2 * step + 1), key_tile_at(step), idesc_cols, i > 0);
                if (step % kParts == kParts - 1) mma.commit(&k_empty[step / kParts % kKS]);
            }
            if (ok) mma.commit(sums_full);
            ++item;
        }
    } else {
        // ---- exponentials
        const int half = (warp - 2) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const int32_t row_token = r / p.a.group, row_head = r - row_token * p.a.group;
        uint32_t item = 0, step = 0;
        while (ok && next()) {
            const int32_t i = t.t0 + row_token, steps = t.nblk * kParts, last = p.a.causal ? min(t.n - 1, i) : t.n - 1;
            const bool mine = r < rows && i < t.n;
            const int64_t token = t.first + i;
            const float2 stat = mine ? p.stats[(static_cast<int64_t>(t.head) * p.a.tokens + token) * p.a.group + row_head] : make_float2(-INFINITY, 0.f);
            // this thread's row: the norm of its gradient, and the power of two of its sum
            const int64_t of_head = static_cast<int64_t>(t.head) * p.a.tokens;
            const float most_v = BF16 ? 0.f : p.largest[of_head + t.first].y, g = !BF16 && mine ? p.grad_norms[(of_head + token) * p.a.group + row_head] : 0.f;
            float unit = 1.f;
            const float2 lse2 = make_float2(stat.x, stat.x);
            for (int32_t at = 0; at < steps; ++at, ++step) {
                const uint32_t s_taddr = tmem + lane_base + kRegion + 2 * step % 3 * kWide + half * 64, p_taddr = tmem + lane_base + kRegion + (2 * step + 1) % 3 * kWide + half * 64;
                const int32_t seen = last + 1 - at * kWide - half * 64;  // columns that this thread's row sees
                const bool mask = __any_sync(0xffffffffu, seen < 64);
                if (!wait(&s_full[step & 1], step >> 1 & 1, 11)) break;
                tc_fence_after();
                if (!BF16 && at == 0) unit = unit_of(2.f * g * most_v);
                float w[64];
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t s[32];
                    tmem_ld32(s_taddr + c0, s);
                    tmem_ld_wait();
                    if (mask) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (c0 + c >= seen) s[c] = 0xff800000u;
                    }
                    if (c0 == 32) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&s_free[step & 1]);
                    }
                    weights(s, p.scale_log2, w + c0, [&](int) { return lse2; });
                }
                if (!wait(&dp_full[step & 1], step >> 1 & 1, 12)) break;
                tc_fence_after();
                const float minus_delta = -stat.y * unit;
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 32) {
                    uint32_t dp[32];
                    tmem_ld32(p_taddr + c0, dp);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 32; c += 2) {
                        float2 x = __ffma2_rn(make_float2(__uint_as_float(dp[c]), __uint_as_float(dp[c + 1])), make_float2(unit, unit), make_float2(minus_delta, minus_delta));
                        x = __fmul2_rn(x, make_float2(w[c0 + c], w[c0 + c + 1]));
                        w[c0 + c] = x.x;
                        w[c0 + c + 1] = x.y;
                    }
                    store_packed<BF16>(p_taddr + c0 / 2, w + c0);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ds_full[step & 1]);
            }
            // ---- results: of two warpgroups each takes half of the elements
            if (!wait(sums_full, item & 1, 13)) break;
            tc_fence_after();
            const int64_t head = t.head * p.a.group + row_head;
            uint8_t* const to = static_cast<uint8_t*>(p.dq) + (token * p.dq_token + head * p.dq_head) * 2;
            const float factor = p.scale / unit;
#pragma unroll 1
            for (int c0 = half * (D / 2); c0 < (kParts == 2 ? D : (half + 1) * (D / 2)); c0 += 32) {
                if (c0 >= p.a.head_dim) break;
                uint32_t x[32];
                tmem_ld32(tmem + lane_base + kDq + c0, x);
                tmem_ld_wait();
                if (mine) store_result<BF16>(to, x, factor, c0, p.a.head_dim, p.wide != 0);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sums_free);
            ++item;
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Shape<D>::kTmem);
    }
}

template <int D, bool BF16>
int launch(const PackedCall& c, cudaStream_t stream) {
    const PackedArgs& a = c.a;
    CUtensorMap mq, mk, mv, mg;
    if (int st = query_map(&mq, c.q, a)) return st;
    if (int st = query_map(&mg, c.grad, a)) return st;
    if (int st = key_map(&mk, c.k, a)) return st;
    if (int st = key_map(&mv, c.v, a)) return st;
    GradParams p;
    p.a = a;
    p.stats = c.stats();
    p.largest = c.largest();
    p.grad_norms = c.grad_norms();
    p.value_norms = c.value_norms();
    p.dq = c.dq.base, p.dk = c.dk.base, p.dv = c.dv.base;
    p.dq_token = c.dq.token, p.dq_head = c.dq.head;
    p.dk_token = c.dk.token, p.dk_head = c.dk.head;
    p.dv_token = c.dv.token, p.dv_head = c.dv.head;
    p.scale = c.scale;
    p.scale_log2 = c.scale * kLog2e;
    p.k_steps = (a.head_dim + 15) / 16;
    p.wide = on_wide_grid(c.dq, a.head_dim, a.tokens, a.q_heads) && on_wide_grid(c.dk, a.head_dim, a.tokens, a.kv_heads) && on_wide_grid(c.dv, a.head_dim, a.tokens, a.kv_heads);
    p.splits = key_splits_tc(a);
    p.shares = c.shares();
    static std::atomic<bool> keys_allowed[64], queries_allowed[64];
    auto keys = key_grads_kernel<D, BF16>;
    auto queries = query_grads_kernel<D, BF16>;
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(keys), KeySmem<D>::kTotal, keys_allowed)) return st;
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(queries), QuerySmem<D>::kTotal, queries_allowed)) return st;
    const auto grid = [](int64_t items) { return dim3(static_cast<unsigned>(items)); };
    cudaError_t e = launch_dependent(keys, grid(static_cast<int64_t>(a.key_capacity) * a.kv_heads * p.splits), dim3(Shape<D>::kThreads), KeySmem<D>::kTotal, stream, 1, true, mq, mk, mv, mg, p);
    if (e == cudaSuccess)
        e = launch_dependent(queries, grid(2 * static_cast<int64_t>(a.row_capacity) * a.kv_heads), dim3(Shape<D>::kThreads), QuerySmem<D>::kTotal, stream, 1, true, mq, mk, mv, mg, p);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of packed_attention_grad failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("packed_attention_grad");
    return p.splits > 1 ? packed_join_shares(c, p.splits, stream) : MHLO_CUDA_OK;
}

}  // namespace

int packed_attention_grad_tc(const PackedCall& c, cudaStream_t stream) {
    const bool bf16 = c.dtype == MHLO_DT_BF16;
    if (c.a.head_dim <= 64) return bf16 ? launch<64, true>(c, stream) : launch<64, false>(c, stream);
    return bf16 ? launch<128, true>(c, stream) : launch<128, false>(c, stream);
}

int packed_attention_grad_tc_device_error() { return take_kv_error(); }

}  // namespace mhlo
