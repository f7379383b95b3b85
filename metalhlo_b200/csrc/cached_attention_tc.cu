// Attention over the paged 8-bit cache for sequences with many rows (chunks of a prompt, long drafts): the products on tcgen05, bf16
// and fp16, head dimension 64 or 128.
//
// A CTA owns 256 rows of a segment as two halves of 128 and walks the keys in blocks of 128:
//   warp 0             MMA issuer: S_h = Q_h K^T (both operands in shared memory), O_h += P_h V (P read from tensor memory)
//   warps 1-3, 12-15   producers: codes of keys and values from global memory a block ahead (asynchronous copies into slots of their
//                      own lanes), then into the 128-byte-swizzled layout as fp16, exactly
//   warps 4-7, 8-11    softmax of half 0 / 1, a thread per row: it puts its row of q into shared memory as fp16 at a piece's start and
//                      writes P over the scores in tensor memory
// The scales do not touch the codes: a key's scale multiplies its column of scores (16 keys at a time share one), a value's scale goes
// into the exponent of the weights as its ratio to the largest of the piece, so the products run on integers up to 127.
// Rows that are fp16 stay as they are; bf16 rows are brought to the same size by powers of two, which is exact.
//
// Per block and CTA the tensor pipe needs about 2050 clocks (4096 multiply-adds a clock), the exponentials as many (16 a clock), and
// the producers some 2000 warp instructions beside the 6000 of the softmax, out of 4 a clock: three limits close together. Decoding
// steps would fill 128 rows to a few percent and pay the producers' instructions all the same; they have a kernel of their own.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cached_attention.cuh"
#include "tc_ptx.cuh"

namespace mhlo {
namespace {

constexpr int kBlockM = 128, kHalves = 2, kRows = kHalves * kBlockM, kBlockN = 128, kStages = 2, kThreads = 512, kProducers = 7, kSlots = 4;
constexpr int kGroups = kBlockN / 16;  // keys with one scale
constexpr int kLeast = 3;              // blocks of a CTA's share where there is little to do: 384 keys, as in the kernel of few rows
constexpr float kUnitLog2 = 6.f;       // weights are held times 2^6, so that those far below the largest keep some bits of fp16
constexpr float kUnit = 64.f;
constexpr float kGrowth = 8.f;         // log2 of what scores may exceed the last maximum by before it moves
// Registers: 512 threads are launched with 128 each, 512 for every four lanes of the four warpgroups. The softmax holds a row's 128
// scores and weights; the others have little.
constexpr int kSoftmaxRegs = 168, kOtherRegs = 88;
static_assert(2 * kSoftmaxRegs + 2 * kOtherRegs <= 4 * 128, "register shares above what the CTA is launched with wait forever");
constexpr int kWaitError = 50;         // + where a bounded wait ran out

struct Scales {  // of a block's groups
    float key[kGroups], ratio_log2[kGroups], out_again[kGroups];
    uint32_t missing;  // groups without a page
};

template <int D>
struct Smem {
    static constexpr int kPanels = D / 64;
    static constexpr int kQHalf = kBlockM * D * 2, kTile = kBlockN * D * 2;
    static constexpr int kQ = 0, kK = kQ + kHalves * kQHalf, kV = kK + kStages * kTile, kRaw = kV + kStages * kTile,
                         kRawTile = kBlockN * D, kEnd = kRaw + 2 * kRawTile;
    static constexpr int kTotal = kEnd + 1024;  // the layout starts on 1024 bytes
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { return pack_out<false>(a, b); }

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

// Four codes as four fp16 numbers: 0x64xx is 1024 + xx, xx = code + 128.
__device__ __forceinline__ uint2 codes_f16(uint32_t w) {
    w ^= 0x80808080u;
    const uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342), bias = 0x64806480u;
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&bias));
    const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&hi), *reinterpret_cast<const __half2*>(&bias));
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// What the roles need of a piece: blocks from kb0 on, how many each half takes part in (a half whose rows see nothing of the last ones
// leaves them out; the second may have no rows at all).
struct Blocks {
    int32_t kb0, count, of_half[kHalves], limit;
    __device__ __forceinline__ Blocks(const Segment& s, int32_t group) {
        kb0 = s.t0;
        count = 0;
        limit = s.seen_by(s.rows - 1, group);
        for (int h = 0; h < kHalves; ++h) {
            const int32_t rows = min(kBlockM, s.rows - h * kBlockM);
            const int32_t seen = rows > 0 ? s.seen_by(h * kBlockM + rows - 1, group) : 0;
            of_half[h] = max(0, min(s.t1, (seen + kBlockN - 1) / kBlockN) - kb0);
            count = max(count, of_half[h]);
        }
    }
};

// The weights of 64 of a row's scores, packed; *sum: what they add to the row's sum. MASK: some columns are hidden.
template <bool MASK>
__device__ __forceinline__ void weights_of(const uint32_t* sr, const Scales& sc, int g0, float factor, float m, int32_t key0, int32_t seen, uint32_t* packed, float* total) {
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) {
        const int g = g0 + gi;
        const float f = factor * sc.key[g], off = sc.ratio_log2[g] + (kUnitLog2 - m);
        const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
        const bool hidden = MASK && (sc.missing >> g & 1);
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
            const int at = gi * 16 + c;
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(sr[at]), __uint_as_float(sr[at + 1])), f2, off2);
            float2 e = make_float2(ex2(x.x), ex2(x.y));
            if (MASK) {
                if (hidden || key0 + at >= seen) e.x = 0.f;
                if (hidden || key0 + at + 1 >= seen) e.y = 0.f;
            }
            sum = __fadd2_rn(sum, e);
            packed[at / 2] = pack_f16(e.x, e.y);
        }
        const float s = sum.x + sum.y;
        *total = MASK && s == 0.f ? *total : fmaf(s, sc.out_again[g], *total);
    }
}

// The largest of 64 scores in units of log2(e); hidden ones are not looked at.
template <bool MASK>
__device__ __forceinline__ float largest_of(const uint32_t* sr, const Scales& sc, int g0, float factor, int32_t key0, int32_t seen) {
    float mx = -INFINITY;
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) {
        float gm = -INFINITY;
        if (MASK) {
            const bool hidden = sc.missing >> (g0 + gi) & 1;
#pragma unroll
            for (int c = 0; c < 16; ++c) gm = hidden || key0 + gi * 16 + c >= seen ? gm : fmaxf(gm, __uint_as_float(sr[gi * 16 + c]));
            mx = gm == -INFINITY ? mx : fmaxf(mx, gm * (factor * sc.key[g0 + gi]));
        } else {
#pragma unroll
            for (int c = 0; c < 16; c += 2) gm = fmax3(gm, __uint_as_float(sr[gi * 16 + c]), __uint_as_float(sr[gi * 16 + c + 1]));
            mx = fmaxf(mx, gm * (factor * sc.key[g0 + gi]));
        }
    }
    return mx;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) cached_attention_tc_kernel(const __grid_constant__ CachedParams<T> p) {
    using L = Smem<D>;
    using Works = Work<kRows, kBlockN, kLeast, true>;
    constexpr int kPanels = L::kPanels;
    constexpr uint32_t kTmemCols = 512, kSCol = 0, kOCol = kHalves * kBlockN;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t bars[4 * kHalves + 4 * kStages];
    __shared__ uint32_t tmem_slot;
    __shared__ typename Works::Scratch scratch;
    __shared__ Scales scales[kSlots];
    __shared__ float v_most[kSlots];  // the largest value scale of the piece that a slot's block is of
    uint64_t* const q_full = bars;
    uint64_t* const s_full = q_full + kHalves;    // scores of the half's block are in tensor memory
    uint64_t* const p_full = s_full + kHalves;    // its weights are, and O is rescaled if need be
    uint64_t* const pv_done = p_full + kHalves;   // every product with values so far has completed
    uint64_t* const k_full = pv_done + kHalves;
    uint64_t* const k_empty = k_full + kStages;
    uint64_t* const v_full = k_empty + kStages;
    uint64_t* const v_empty = v_full + kStages;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int h = 0; h < kHalves; ++h) {
            mbar_init(&q_full[h], 4);
            mbar_init(&s_full[h], 1);
            mbar_init(&p_full[h], 4);
            mbar_init(&pv_done[h], 1);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&k_full[s], kProducers);
            mbar_init(&k_empty[s], 1);
            mbar_init(&v_full[s], kProducers);
            mbar_init(&v_empty[s], 1);
        }
        fence_barrier_init();
    }
    Works work;
    const bool any = work.template start<kThreads>(p, scratch);  // synchronises the CTA
    grid_dependency_release();
    if (!any) return;
    if (warp == 0) {
        tmem_alloc(&tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, int where) {
        if (!ok) return;
        if (!mbar_wait(bar, parity)) {
            kv_report(kWaitError + where);
            ok = false;
        }
    };
    Segment seg;
    if (warp < 4 || warp >= 12) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));

    if (warp == 0) {
        // ---- MMA issuer. Order on the pipe: for each half P.V of this block, then S of the next (of this piece, or the first of the
        // next one): S overwrites the half's scores and weights only after its P.V has read them.
        const uint32_t idesc_s = (1u << 4) | (static_cast<uint32_t>(kBlockN >> 3) << 17) | (static_cast<uint32_t>(kBlockM >> 4) << 24);
        const uint32_t idesc_o = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(kBlockM >> 4) << 24);
        const uint32_t q_addr = smem_u32(smem + L::kQ), k_addr = smem_u32(smem + L::kK), v_addr = smem_u32(smem + L::kV);
        auto commit_to = [&](uint64_t* bar) {
            if (elect_one()) umma_commit(bar);
            __syncwarp();
        };
        auto issue_s = [&](int h, int stage) {
            const uint32_t qa = q_addr + h * L::kQHalf, ka = k_addr + stage * L::kTile;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint64_t da = make_smem_desc(qa + (kk / 4) * kBlockM * 128 + (kk % 4) * 32, 16, 1024);
                const uint64_t db = make_smem_desc(ka + (kk / 4) * kBlockN * 128 + (kk % 4) * 32, 16, 1024);
                if (elect_one()) umma_f16(tmem + kSCol + h * kBlockN, da, db, idesc_s, kk != 0 ? 1u : 0u);
            }
            commit_to(&s_full[h]);
        };
        auto issue_pv = [&](int h, int stage, bool accumulate) {
            const uint32_t va = v_addr + stage * L::kTile;
#pragma unroll
            for (int kk = 0; kk < kBlockN / 16; ++kk) {
                const uint64_t db = make_smem_desc(va + kk * 16 * 128, kBlockN * 128, 1024);
                if (elect_one()) umma_ts(tmem + kOCol + h * D, tmem + kSCol + h * kBlockN + kk * 8, db, idesc_o, accumulate || kk != 0 ? 1u : 0u);
            }
            commit_to(&pv_done[h]);
        };
        auto next_blocks = [&](Blocks* out) {
            while (work.next(p, &seg)) {
                *out = Blocks(seg, p.group);
                if (out->count > 0) return true;
            }
            return false;
        };
        Blocks cur(Segment{}, 1), nxt(Segment{}, 1);
        bool has = next_blocks(&cur);
        int stage = 0;
        uint32_t phase = 0, it[kHalves] = {0, 0}, q_of[kHalves] = {0, 0};  // q_of: pieces the half has had blocks of
        // scores of half h in block j of a piece
        auto scores = [&](const Blocks& of, int j, int h, int st, uint32_t ph) {
            const bool takes_part = j < of.of_half[h];
            if (takes_part && j == 0) wait(&q_full[h], q_of[h]++ & 1, 1);
            if (h == 0) wait(&k_full[st], ph, 2);
            if (!ok) return;
            if (takes_part) {
                tc_fence_after();
                issue_s(h, st);
            }
            if (h == kHalves - 1) commit_to(&k_empty[st]);
        };
        if (has)
            for (int h = 0; h < kHalves; ++h) scores(cur, 0, h, 0, 0);
        while (has && ok) {
            const bool more_pieces = next_blocks(&nxt);
            for (int j = 0; j < cur.count && ok; ++j) {
                const bool last = j + 1 == cur.count;
                const int next_stage = stage + 1 == kStages ? 0 : stage + 1;
                const uint32_t next_phase = stage + 1 == kStages ? phase ^ 1 : phase;
                wait(&v_full[stage], phase, 3);
                for (int h = 0; h < kHalves && ok; ++h) {
                    if (j < cur.of_half[h]) {
                        wait(&p_full[h], it[h] & 1, 4);
                        if (!ok) break;
                        tc_fence_after();
                        issue_pv(h, stage, j > 0);
                        ++it[h];
                    }
                    if (h == kHalves - 1) commit_to(&v_empty[stage]);
                    if (!last) scores(cur, j + 1, h, next_stage, next_phase);
                }
                // the next piece's q comes only when the half is through with this one
                for (int h = 0; h < kHalves && ok && last && more_pieces; ++h) scores(nxt, 0, h, next_stage, next_phase);
                stage = next_stage;
                phase = next_phase;
            }
            cur = nxt;
            has = more_pieces;
        }
    } else if (warp < 4 || warp >= 12) {
        // ---- producers
        const KvArgs& a = p.kv;
        const int wp = warp < 4 ? warp - 1 : warp - 9;
        constexpr int kChunks = D / 16, kPassRows = 32 / kChunks, kPasses = kBlockN / kPassRows, kMine = (kPasses + kProducers - 1) / kProducers;
        // 16 codes a lane: four lanes of a quarter warp on one row and four on the next keep the stores free of bank conflicts
        const int chunk = D == 128 ? (lane & 3) | (lane >> 4) << 2 : lane & 3, row_in_pass = D == 128 ? (lane >> 2) & 3 : lane >> 2;
        int stage = 0;
        uint32_t phase = 0, block = 0;
        while (ok && work.next(p, &seg)) {
            const Blocks bl(seg, p.group);
            if (bl.count == 0) continue;
            // pages and scales of a block's groups, one per lane
            struct Groups {
                int64_t base;
                float ks, vs;
            };
            auto look_up = [&](int j) {
                Groups g{-1, 0.f, 0.f};
                const int32_t key = (bl.kb0 + j) * kBlockN + lane * 16;
                if (lane < kGroups && j < bl.count && key < bl.limit) {
                    const int32_t page = kv_page(a, seg.b, key >> a.page_shift);
                    if (page >= 0) {
                        const int64_t at = static_cast<int64_t>(page) * a.heads + seg.head;
                        g.base = ((at << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * D;
                        g.ks = a.k_scales[at];
                        g.vs = a.v_scales[at];
                    }
                }
                return g;
            };
            Groups now = look_up(0), next = look_up(1);
            // the largest value scale of the piece
            float most = 0.f;
            const int32_t keys_end = min(bl.limit, (bl.kb0 + bl.count) * kBlockN);
#pragma unroll 4
            for (int32_t i = (bl.kb0 * kBlockN >> a.page_shift) + lane; i <= (keys_end - 1) >> a.page_shift; i += 32) {
                const int32_t page = kv_page(a, seg.b, i);
                if (page >= 0) most = fmaxf(most, a.v_scales[static_cast<int64_t>(page) * a.heads + seg.head]);
            }
            most = warp_reduce<MaxOp>(most);
            // Codes wait in shared memory, in slots that only the lane that copies them reads: in registers a block of both would not fit,
            // and half a block ahead they were late (chunks of 512 tokens on 8192: 300 us that way, 215 with no copies at all).
            auto load = [&](const int8_t* codes, int64_t from, int slots) {
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int pass = wp + i * kProducers, row = pass * kPassRows + row_in_pass;
                    const int64_t b = __shfl_sync(0xffffffffu, from, (pass * kPassRows / 16) & 7);
                    if (pass < kPasses && b >= 0) copy16(smem_u32(smem + slots + (pass * 32 + lane) * 16), codes + b + (row & 15) * D + chunk * 16);
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            // zeros: groups whose rows are stored as zeros (no page, or a value scale that is nothing)
            auto store = [&](int offset, int slots, uint32_t zeros) {
                asm volatile("cp.async.wait_group 1;" ::: "memory");  // all but the newest: keys and values take turns
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int pass = wp + i * kProducers, row = pass * kPassRows + row_in_pass;
                    if (pass >= kPasses) break;
                    const bool zero = zeros >> (pass * kPassRows / 16) & 1;
                    const uint4 raw = *reinterpret_cast<const uint4*>(smem + slots + (pass * 32 + lane) * 16);
                    const uint2 c0 = codes_f16(raw.x), c1 = codes_f16(raw.y), c2 = codes_f16(raw.z), c3 = codes_f16(raw.w);
                    uint8_t* const at = smem + offset + (chunk >> 2) * kBlockN * 128 + row * 128;
                    const int c = (chunk & 3) * 2;
                    *reinterpret_cast<uint4*>(at + ((c ^ (row & 7)) << 4)) = zero ? make_uint4(0, 0, 0, 0) : make_uint4(c0.x, c0.y, c1.x, c1.y);
                    *reinterpret_cast<uint4*>(at + (((c + 1) ^ (row & 7)) << 4)) = zero ? make_uint4(0, 0, 0, 0) : make_uint4(c2.x, c2.y, c3.x, c3.y);
                }
                fence_proxy_async();
                __syncwarp();
            };
            load(a.k_codes, now.base, L::kRaw);
            load(a.v_codes, now.base, L::kRaw + L::kRawTile);
            for (int j = 0; j < bl.count && ok; ++j, ++block) {
                const Groups after = look_up(j + 2);
                const float ratio = most > 0.f ? now.vs / most : now.vs * 0.f;  // NaN stays
                const bool nothing = ratio < 1e-18f;
                const uint32_t missing = __ballot_sync(0xffffffffu, now.base < 0) & ((1u << kGroups) - 1), no_value = missing | __ballot_sync(0xffffffffu, nothing);
                wait(&k_empty[stage], phase ^ 1, 6);
                if (!ok) break;
                if (wp == 0 && lane < kGroups) {
                    // Four slots: k_empty says that the scores of two blocks ago are done, and they were asked for only after both halves
                    // had the weights of the block before those.
                    Scales& s = scales[block % kSlots];
                    s.key[lane] = now.base < 0 ? 0.f : now.ks;
                    s.ratio_log2[lane] = nothing ? 0.f : __log2f(ratio);
                    s.out_again[lane] = nothing ? 1.f / kUnit : __fdividef(1.f / kUnit, ratio);
                    if (lane == 0) {
                        s.missing = missing;
                        v_most[block % kSlots] = most;
                    }
                }
                store(L::kK + stage * L::kTile, L::kRaw, missing);
                if (lane == 0) mbar_arrive(&k_full[stage]);
                load(a.k_codes, next.base, L::kRaw);
                wait(&v_empty[stage], phase ^ 1, 7);
                if (!ok) break;
                store(L::kV + stage * L::kTile, L::kRaw + L::kRawTile, no_value);
                if (lane == 0) mbar_arrive(&v_full[stage]);
                load(a.v_codes, next.base, L::kRaw + L::kRawTile);
                now = next;
                next = after;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
        // ---- softmax
        const int h = (warp - 4) >> 2, quarter = warp & 3, r = h * kBlockM + quarter * 32 + lane;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_taddr = tmem + lane_base + kSCol + h * kBlockN, o_taddr = tmem + lane_base + kOCol + h * D;
        const float to_log2 = p.scale * 1.4426950408889634f;
        uint32_t it = 0, block0 = 0;
        while (ok && work.next(p, &seg)) {
            const Blocks bl(seg, p.group);
            const int nb = bl.of_half[h];
            const int32_t seen = r < seg.rows ? seg.seen_by(r, p.group) : 0x7fffffff;  // rows that are none hide nothing
            float m_ref = -INFINITY, l = 0.f, factor = 0.f, largest = 0.f;
            if (nb > 0) {
                // This row of q. The half's last scores of the piece before are done (this thread has seen them): q may be replaced.
                uint4 raw[D / 8];
                const T* const x = r < seg.rows ? p.q + seg.token(p, r) * p.qs[0] + seg.q_head(p, r) * p.qs[1] : nullptr;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    raw[c] = make_uint4(0, 0, 0, 0);
                    if (x == nullptr) continue;
                    if (p.q_vec) {
                        raw[c] = __ldcs(reinterpret_cast<const uint4*>(x + c * 8));  // not the read-only path: o may be q
                    } else {
                        float f[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = VecTraits<T>::to_float(x[c * 8 + e]);
                        raw[c] = VecTraits<T>::pack(f);
                    }
                }
                int shift = 0;
                if (kBf16) {
                    float big = 0.f;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        float f[8];
                        VecTraits<T>::unpack(raw[c], f);
#pragma unroll
                        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(f[e]));
                    }
                    if (big > 0.f && big < INFINITY) shift = max(-120, ilogbf(big) - 13);
                }
                const float unit = scalbnf(1.f, -shift);
                factor = scalbnf(to_log2, shift);
                const int row = r - h * kBlockM;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    uint4 w = raw[c];
                    if (kBf16) {
                        float f[8];
                        VecTraits<T>::unpack(raw[c], f);
                        w = make_uint4(pack_f16(f[0] * unit, f[1] * unit), pack_f16(f[2] * unit, f[3] * unit), pack_f16(f[4] * unit, f[5] * unit), pack_f16(f[6] * unit, f[7] * unit));
                    }
                    *reinterpret_cast<uint4*>(smem + L::kQ + h * L::kQHalf + (c >> 3) * kBlockM * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = w;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[h]);
            }
            for (int j = 0; j < nb && ok; ++j, ++it) {
                wait(&s_full[h], it & 1, 8);
                if (!ok) break;
                tc_fence_after();
                if (j == 0) largest = v_most[block0 % kSlots];
                const Scales& sc = scales[(block0 + j) % kSlots];
                const int32_t key0 = (bl.kb0 + j) * kBlockN;
                const bool mask = __any_sync(0xffffffffu, key0 + kBlockN > seen) || sc.missing != 0;
                // Two chunks of 64 keys, the loop not unrolled: instruction fetch was a third of the stalls with both and a variant that
                // took the maximum of earlier blocks for granted. A chunk looks at its own maximum first; where it would push weights out of
                // fp16 (a piece's first chunk, rarely later) everything so far is scaled anew. Every product with values so far completed
                // before these scores were signalled.
#pragma unroll 1
                for (int ci = 0; ci < 2; ++ci) {
                    const int32_t first = key0 + ci * 64;
                    uint32_t sr[64], packed[32];
                    tmem_ld32(s_taddr + ci * 64, sr);
                    tmem_ld32(s_taddr + ci * 64 + 32, sr + 32);
                    tmem_ld_wait();
                    const float mx = mask ? largest_of<true>(sr, sc, ci * 4, factor, first, seen) : largest_of<false>(sr, sc, ci * 4, factor, first, seen);
                    const bool grow = mx > m_ref + kGrowth;
                    if (__any_sync(0xffffffffu, grow)) {
                        float alpha = 1.f;
                        if (grow) {
                            alpha = m_ref == -INFINITY ? 0.f : ex2(m_ref - mx);
                            m_ref = mx;
                            l *= alpha;
                        }
                        // O of earlier blocks (j > 0), then this block's first weights (ci > 0)
#pragma unroll 1
                        for (int c0 = j > 0 ? 0 : D; c0 < D + (ci > 0 ? 32 : 0); c0 += 32) {
                            const uint32_t at = c0 < D ? o_taddr + c0 : s_taddr;
                            uint32_t w[32];
                            if (c0 >= D) tmem_st_wait();  // this thread's own store of them
                            tmem_ld32(at, w);
                            tmem_ld_wait();
                            if (c0 < D) {
#pragma unroll
                                for (int c = 0; c < 32; ++c) w[c] = __float_as_uint(__uint_as_float(w[c]) * alpha);
                            } else {
                                const __half2 by = __float2half2_rn(alpha);
#pragma unroll
                                for (int c = 0; c < 32; ++c) {
                                    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&w[c]), by);
                                    w[c] = *reinterpret_cast<const uint32_t*>(&x);
                                }
                            }
                            tmem_st32(at, w);
                        }
                    }
                    const float m = m_ref == -INFINITY ? 0.f : m_ref;
                    if (mask) weights_of<true>(sr, sc, ci * 4, factor, m, first, seen, packed, &l);
                    else weights_of<false>(sr, sc, ci * 4, factor, m, first, seen, packed, &l);
                    tmem_st32(s_taddr + ci * 32, packed);  // over columns that have been read
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[h]);
            }
            if (!ok) break;
            // The next piece's first product with values waits for this warp's weights, which come after these reads.
            if (nb > 0) {
                wait(&pv_done[h], (it - 1) & 1, 9);
                if (!ok) break;
                tc_fence_after();
            }
            const bool nothing = l == 0.f;
            const float unit = largest * (1.f / kUnit), by = seg.cut ? unit : nothing ? 0.f : unit / l;
            float* const out = work.partial(p, seg, D);
            T* const y = r < seg.rows ? p.o + seg.token(p, r) * p.os[0] + seg.q_head(p, r) * p.os[1] : nullptr;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
                uint32_t o[32];
                if (nb > 0) {
                    tmem_ld32(o_taddr + c0, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int c = 0; c < 32; ++c) o[c] = nb == 0 || nothing ? 0u : __float_as_uint(__uint_as_float(o[c]) * by);
                if (r < seg.rows && seg.cut) {
#pragma unroll
                    for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(out + 2 * kRows + r * D + c0 + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                } else if (r < seg.rows) {
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        if (p.o_vec == 2) {
                            *reinterpret_cast<uint4*>(y + c0 + c) =
                                make_uint4(pack_out<kBf16>(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), pack_out<kBf16>(__uint_as_float(o[c + 2]), __uint_as_float(o[c + 3])),
                                           pack_out<kBf16>(__uint_as_float(o[c + 4]), __uint_as_float(o[c + 5])), pack_out<kBf16>(__uint_as_float(o[c + 6]), __uint_as_float(o[c + 7])));
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[c0 + c + e] = VecTraits<T>::from_float(__uint_as_float(o[c + e]));
                        }
                    }
                }
                __syncwarp();  // loads from tensor memory are the whole warp's
            }
            if (r < seg.rows) {
                if (seg.cut) {
                    out[r] = m_ref;
                    out[kRows + r] = l;
                } else if (p.lse != nullptr) {
                    p.lse[seg.token(p, r) * p.q_heads + seg.q_head(p, r)] = nothing ? -INFINITY : (m_ref + log2f(l)) * 0.6931471805599453f;
                }
            }
            if (seg.cut && r == 0) work.leave_piece(p, seg);
            __syncwarp();
            block0 += bl.count;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <typename T, int D>
int launch(CachedParams<T> p, void* scratch, cudaStream_t stream) {
    p.pieces = static_cast<int32_t*>(scratch);
    p.partial = reinterpret_cast<float*>(p.pieces + kGrid * 8);
    auto kernel = cached_attention_tc_kernel<T, D>;
    static std::atomic<bool> smem_set[64];
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), Smem<D>::kTotal, smem_set)) return st;
    kernel<<<kGrid, kThreads, Smem<D>::kTotal, stream>>>(p);
    MHLO_CUDA_CHECK_LAUNCH("cached_attention (tcgen05)");
    if (p.whole) return MHLO_CUDA_OK;
    const cudaError_t e = launch_dependent(join_kernel<T, D, kRows>, dim3(kGrid, kRows / kJoinRows), dim3(32 * kJoinRows), 0, stream, 1, true, p);
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of cached_attention failed: %s", cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH("cached_attention (joining)");
    return MHLO_CUDA_OK;
}

}  // namespace

template <typename T>
int cached_attention_long(CachedParams<T> p, void* scratch, cudaStream_t stream) {
    return p.kv.head_dim == 64 ? launch<T, 64>(p, scratch, stream) : launch<T, 128>(p, scratch, stream);
}
template int cached_attention_long<__half>(CachedParams<__half>, void*, cudaStream_t);
template int cached_attention_long<__nv_bfloat16>(CachedParams<__nv_bfloat16>, void*, cudaStream_t);

int64_t cached_attention_long_scratch(int head_dim) { return kGrid * (8 * 4 + 2 * kRows * (head_dim + 2) * int64_t{4}); }
int cached_attention_long_device_error() { return take_kv_error(); }

}  // namespace mhlo
