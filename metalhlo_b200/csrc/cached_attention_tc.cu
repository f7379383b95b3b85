// Attention over the paged 8-bit cache for sequences with many rows (chunks of a prompt, long drafts): the products on tcgen05, bf16
// and fp16, head dimension 64 or 128.
//
// A CTA owns 256 rows of a segment as two halves of 128 and walks the keys in blocks of 128, two steps of 64 each:
//   warp 0             MMA issuer: S_h = Q_h K^T (both operands in shared memory), O_h += P_h V (P read from tensor memory)
//   warps 1-3, 12-15   producers: codes of keys and values from global memory a block ahead (asynchronous copies into slots of their
//                      own lanes), then into the 128-byte-swizzled layout as fp16, exactly
//   warps 4-7, 8-11    softmax of half 0 / 1, a thread per row: it puts its row of q into shared memory as fp16 at a piece's start and
//                      writes P over the scores in tensor memory
// The scales do not touch the codes: a key's scale multiplies its column of scores (16 keys at a time share one), a value's scale goes
// into the exponent of the weights, 2^(z + log2 vs - M), so the products run on integers up to 127. M is a row's own, of the keys that it
// has seen.
// Rows that are fp16 stay as they are; bf16 rows are brought to the same size by powers of two, which is exact.
//
// A half has two sets of scores (64 columns of tensor memory, O another head_dim): while the softmax works on step t the scores of
// t + 1 are there already, and those of t + 2 go out behind P.V of t, whose weights lie in the same columns. With one set of 128
// columns the softmax stood and waited for a third of the time; now it is what bounds a block, about 1 us a step of either half.
//
// Per block and CTA the tensor pipe needs about 2050 clocks (4096 multiply-adds a clock), the exponentials as many (16 a clock), and
// the producers some 2000 warp instructions beside the 6000 of the softmax, out of 4 a clock: three limits close together. Decoding
// steps would fill 128 rows to a few percent and pay the producers' instructions all the same; they have a kernel of their own.
// Chunks of 512 tokens of four sequences behind 7680 others, 32 query heads of 128 on 8, bf16: 365 us, 730 TFLOP/s. With
// a pass over all its pages first a piece had 17 us besides its steps: 2.5 until it knows its work, 7 for the first page, its codes and q, 4.5
// for its results, 3 for the first steps; without that pass 64 new tokens of one sequence behind 7680 take 44.4 us instead of 46.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cached_attention.cuh"
#include "tc_ptx.cuh"

namespace mhlo {
namespace {

constexpr int kStep = 64;  // keys whose scores are taken at once
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

struct __align__(16) Scales {  // of a block's groups
    float key[kGroups], value_log2[kGroups], out_again[kGroups];  // out_again: 1 / (kUnit value scale)
    float least[2];    // of each step, the least value_log2; -infinity where one is beyond 2^+-kReach or 2^30 of another, zero or no number
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

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]),
                 "r"(r[6]), "r"(r[7])
                 : "memory");
}

// Four codes as four fp16 numbers: 0x64xx is 1024 + xx, xx = code + 128.
__device__ __forceinline__ uint2 codes_f16(uint32_t w) {
    w ^= 0x80808080u;
    const uint32_t lo = __byte_perm(w, 0x64646464u, 0x4140), hi = __byte_perm(w, 0x64646464u, 0x4342), bias = 0x64806480u;
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), *reinterpret_cast<const __half2*>(&bias));
    const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&hi), *reinterpret_cast<const __half2*>(&bias));
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// What the roles need of a piece: blocks from kb0 on, and how many steps each half takes part in (a half whose rows see nothing of the
// last ones leaves them out; the second may have no rows at all).
struct Blocks {
    int32_t kb0, count, steps, of_half[kHalves], limit;
    __device__ __forceinline__ Blocks(const Segment& s, int32_t group) {
        kb0 = s.t0;
        steps = 0;
        limit = s.seen_by(s.rows - 1, group);
        for (int h = 0; h < kHalves; ++h) {
            const int32_t rows = min(kBlockM, s.rows - h * kBlockM);
            const int32_t seen = rows > 0 ? s.seen_by(h * kBlockM + rows - 1, group) : 0;
            of_half[h] = max(0, min(2 * s.t1, (seen + kStep - 1) / kStep) - 2 * kb0);
            steps = max(steps, of_half[h]);
        }
        count = (steps + 1) / 2;
    }
};

__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

struct Step {  // the groups of a step as a row takes them
    float f[4], value_log2[4];  // f: what turns a product into a score in units of log2(e)
    __device__ __forceinline__ Step(const Scales& sc, int set, float factor) {
        load_f32<4>(sc.key + set * 4, f);
        load_f32<4>(sc.value_log2 + set * 4, value_log2);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] *= factor;
    }
};

// The weights of 64 of a row's scores, packed; *total: the row's sum, which they are added to: it is one of 2^(z - m) and gets the weights
// times conv / value scale, conv = 2^d, big_m = m + d. MASK: some columns are hidden.
template <bool MASK>
__device__ __forceinline__ void weights_of(const uint32_t* sr, const Step& st, const float* out_again, uint32_t missing, float big_m, float conv, int32_t key0, int32_t seen,
                                           uint32_t* packed, float* total) {
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) {
        const float f = st.f[gi], off = st.value_log2[gi] + (kUnitLog2 - big_m);
        const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
        const bool hidden = MASK && (missing >> gi & 1);
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
        *total = fmaf(sum.x + sum.y, out_again[gi] * conv, *total);
    }
}

// The largest z + log2 vs of 64 scores, in units of log2(e); hidden ones are not looked at, and neither are those that are no number.
template <bool MASK>
__device__ __forceinline__ float largest_of(const uint32_t* sr, const Step& st, uint32_t missing, int32_t key0, int32_t seen) {
    float mx = -INFINITY;
#pragma unroll
    for (int gi = 0; gi < 4; ++gi) {
        float gm = -INFINITY;
        if (MASK) {
            const bool hidden = missing >> gi & 1;
#pragma unroll
            for (int c = 0; c < 16; ++c) gm = hidden || key0 + gi * 16 + c >= seen ? gm : fmaxf(gm, __uint_as_float(sr[gi * 16 + c]));
            if (gm == -INFINITY) continue;
        } else {
#pragma unroll
            for (int c = 0; c < 16; c += 2) gm = fmax3(gm, __uint_as_float(sr[gi * 16 + c]), __uint_as_float(sr[gi * 16 + c + 1]));
        }
        mx = fmaxf(mx, fmaf(gm, st.f[gi], st.value_log2[gi]));
    }
    return mx;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1) cached_attention_tc_kernel(const __grid_constant__ CachedParams<T> p) {
    using L = Smem<D>;
    using Works = Work<kRows, kBlockN, kLeast, true>;
    constexpr int kPanels = L::kPanels;
    constexpr uint32_t kTmemCols = 512, kSCol = 0, kOCol = kHalves * 2 * kStep;  // scores: [half][set][64]
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint64_t bars[7 * kHalves + 4 * kStages];
    __shared__ uint32_t tmem_slot;
    __shared__ typename Works::Scratch scratch;
    __shared__ Scales scales[kSlots];
    uint64_t* const q_full = bars;
    uint64_t* const s_full = q_full + kHalves;      // [half][set]: scores of a step are in tensor memory
    uint64_t* const p_full = s_full + 2 * kHalves;  // [half][set]: its weights are, and O is rescaled if need be
    // [half][set]: the step's product with values, and every one before it, has completed. A wait knows a phase only from its
    // neighbours: with one barrier for both sets the last two products of a piece could complete before anybody looked.
    uint64_t* const pv_done = p_full + 2 * kHalves;
    uint64_t* const k_full = pv_done + 2 * kHalves;
    uint64_t* const k_empty = k_full + kStages;
    uint64_t* const v_full = k_empty + kStages;
    uint64_t* const v_empty = v_full + kStages;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int h = 0; h < kHalves; ++h) {
            mbar_init(&q_full[h], 4);
            for (int set = 0; set < 2; ++set) {
                mbar_init(&pv_done[2 * h + set], 1);
                mbar_init(&s_full[2 * h + set], 1);
                mbar_init(&p_full[2 * h + set], 4);
            }
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
        // ---- MMA issuer. Order on the pipe: for each half P.V of step t, then the scores of step t + 2, which overwrite the weights
        // that this P.V has read.
        const uint32_t idesc_s = (1u << 4) | (static_cast<uint32_t>(kStep >> 3) << 17) | (static_cast<uint32_t>(kBlockM >> 4) << 24);
        const uint32_t idesc_o = (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17) | (static_cast<uint32_t>(kBlockM >> 4) << 24);
        const uint32_t q_addr = smem_u32(smem + L::kQ), k_addr = smem_u32(smem + L::kK), v_addr = smem_u32(smem + L::kV);
        auto commit_to = [&](uint64_t* bar) {
            if (elect_one()) umma_commit(bar);
            __syncwarp();
        };
        auto issue_s = [&](int h, int t, int stage) {
            const uint32_t qa = q_addr + h * L::kQHalf, ka = k_addr + stage * L::kTile + (t & 1) * kStep * 128;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint64_t da = make_smem_desc(qa + (kk / 4) * kBlockM * 128 + (kk % 4) * 32, 16, 1024);
                const uint64_t db = make_smem_desc(ka + (kk / 4) * kBlockN * 128 + (kk % 4) * 32, 16, 1024);
                if (elect_one()) umma_f16(tmem + kSCol + (2 * h + (t & 1)) * kStep, da, db, idesc_s, kk != 0 ? 1u : 0u);
            }
            commit_to(&s_full[2 * h + (t & 1)]);
        };
        auto issue_pv = [&](int h, int t, int stage) {
            const uint32_t va = v_addr + stage * L::kTile + (t & 1) * kStep * 128;
#pragma unroll
            for (int kk = 0; kk < kStep / 16; ++kk) {
                const uint64_t db = make_smem_desc(va + kk * 16 * 128, kBlockN * 128, 1024);
                if (elect_one()) umma_ts(tmem + kOCol + h * D, tmem + kSCol + (2 * h + (t & 1)) * kStep + kk * 8, db, idesc_o, t > 0 || kk != 0 ? 1u : 0u);
            }
            commit_to(&pv_done[2 * h + (t & 1)]);
        };
        uint32_t k_block = 0, v_block = 0;  // blocks so far: stage and parity
        uint32_t weights[2 * kHalves] = {0, 0, 0, 0}, q_of[kHalves] = {0, 0};
        while (ok && work.next(p, &seg)) {
            const Blocks bl(seg, p.group);
            if (bl.count == 0) continue;
            // scores of step t, both halves or one (they come in order); the block's last scores free its keys
            auto scores = [&](int t, int h) {
                if (t >= bl.steps) return;
                const uint32_t block = k_block + static_cast<uint32_t>(t >> 1);
                if (h == 0 && (t & 1) == 0) wait(&k_full[block % kStages], block / kStages & 1, 2);
                if (t == 0 && bl.of_half[h] > 0) wait(&q_full[h], q_of[h]++ & 1, 1);
                if (!ok) return;
                if (t < bl.of_half[h]) {
                    tc_fence_after();
                    issue_s(h, t, block % kStages);
                }
                if (h == kHalves - 1 && ((t & 1) == 1 || t + 1 == bl.steps)) commit_to(&k_empty[block % kStages]);
            };
            for (int t = 0; t < 2; ++t)
                for (int h = 0; h < kHalves; ++h) scores(t, h);
            for (int t = 0; t < bl.steps && ok; ++t) {
                const int stage = v_block % kStages;
                if ((t & 1) == 0) wait(&v_full[stage], v_block / kStages & 1, 3);
                for (int h = 0; h < kHalves && ok; ++h) {
                    if (t < bl.of_half[h]) {
                        const int set = 2 * h + (t & 1);
                        wait(&p_full[set], weights[set]++ & 1, 4);
                        if (!ok) break;
                        tc_fence_after();
                        issue_pv(h, t, stage);
                    }
                    scores(t + 2, h);
                }
                if ((t & 1) == 1 || t + 1 == bl.steps) {
                    commit_to(&v_empty[stage]);
                    ++v_block;
                }
            }
            k_block += bl.count;
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
            // Groups without a page have whatever the slots held: their scores are hidden, and all codes are numbers.
            auto store = [&](int offset, int slots) {
                asm volatile("cp.async.wait_group 1;" ::: "memory");  // all but the newest: keys and values take turns
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int pass = wp + i * kProducers, row = pass * kPassRows + row_in_pass;
                    if (pass >= kPasses) break;
                    const uint4 raw = *reinterpret_cast<const uint4*>(smem + slots + (pass * 32 + lane) * 16);
                    const uint2 c0 = codes_f16(raw.x), c1 = codes_f16(raw.y), c2 = codes_f16(raw.z), c3 = codes_f16(raw.w);
                    uint8_t* const at = smem + offset + (chunk >> 2) * kBlockN * 128 + row * 128;
                    const int c = (chunk & 3) * 2;
                    *reinterpret_cast<uint4*>(at + ((c ^ (row & 7)) << 4)) = make_uint4(c0.x, c0.y, c1.x, c1.y);
                    *reinterpret_cast<uint4*>(at + (((c + 1) ^ (row & 7)) << 4)) = make_uint4(c2.x, c2.y, c3.x, c3.y);
                }
                fence_proxy_async();
                __syncwarp();
            };
            load(a.k_codes, now.base, L::kRaw);
            load(a.v_codes, now.base, L::kRaw + L::kRawTile);
            for (int j = 0; j < bl.count && ok; ++j, ++block) {
                const Groups after = look_up(j + 2);
                const uint32_t missing = __ballot_sync(0xffffffffu, now.base < 0) & ((1u << kGroups) - 1);
                wait(&k_empty[stage], phase ^ 1, 6);
                if (!ok) break;
                if (wp == 0) {
                    // Four slots: k_empty says that the scores of two blocks ago are done, and they were asked for only after both halves
                    // had the weights of the block before those.
                    Scales& s = scales[block % kSlots];
                    const float value_log2 = now.base < 0 ? 0.f : log2f(now.vs);
                    float least = now.base < 0 ? INFINITY : fabsf(value_log2) <= kReach ? value_log2 : -INFINITY, most = now.base < 0 ? -INFINITY : value_log2;
#pragma unroll
                    for (int i = 1; i < 4; i <<= 1) {
                        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, i));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, i));
                    }
                    if (most - least > 30.f) least = -INFINITY;
                    if (lane < kGroups) {
                        s.key[lane] = now.base < 0 ? 0.f : key_scale(now.ks, p.key_unit);
                        s.value_log2[lane] = value_log2;
                        s.out_again[lane] = now.base < 0 ? 0.f : __fdividef(1.f / kUnit, now.vs);
                        if ((lane & 3) == 0) s.least[lane >> 2] = least;
                        if (lane == 0) s.missing = missing;
                    }
                }
                store(L::kK + stage * L::kTile, L::kRaw);
                if (lane == 0) mbar_arrive(&k_full[stage]);
                load(a.k_codes, next.base, L::kRaw);
                wait(&v_empty[stage], phase ^ 1, 7);
                if (!ok) break;
                store(L::kV + stage * L::kTile, L::kRaw + L::kRawTile);
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
        const int h = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, r = h * kBlockM + row;
        const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_taddr = tmem + lane_base + kSCol + h * 2 * kStep, o_taddr = tmem + lane_base + kOCol + h * D;
        const float to_log2 = p.scale * 1.4426950408889634f;
        uint8_t* const q_smem = smem + L::kQ + h * L::kQHalf;  // this half's q; between pieces the way of its rows to and from memory
        constexpr int kRowLanes = D / 8, kAtOnce = 32 / kRowLanes;  // lanes of 16 bytes a row of 16-bit elements takes
        auto q_chunk = [&](int of_row, int c) { return q_smem + (c >> 3) * kBlockM * 128 + of_row * 128 + (((c & 7) ^ (of_row & 7)) << 4); };
        uint32_t sets[2] = {0, 0}, block0 = 0;  // sets: steps so far that used the set
        while (ok && work.next(p, &seg)) {
            const Blocks bl(seg, p.group);
            const int steps = bl.of_half[h];
            const int32_t seen = r < seg.rows ? seg.seen_by(r, p.group) : 0x7fffffff;  // rows that are none hide nothing
            const int64_t token = seg.token(p, min(r, seg.rows - 1)), q_head = seg.q_head(p, min(r, seg.rows - 1));
            // The row's sum is in units of 2^m_ref, O in units of 2^(m_ref + d - kUnitLog2), both whole numbers; the others follow from them.
            float m_ref = -INFINITY, d = -INFINITY, big_m = -INFINITY, l = 0.f, factor = 0.f, near = -kReach, conv = 0.f;
            if (steps > 0) {
                // This warp's 32 rows of q, whole rows at a time. The half's last scores of the piece before are done (its products with
                // values are, and they came later): q may be replaced.
                const int64_t from = token * p.qs[0] + q_head * p.qs[1];
                float factors = 0.f;
                uint4 raw[32 / kAtOnce];  // all on the way at once: four at a time took 8 us of a piece
#pragma unroll
                for (int i = 0; i < 32; i += kAtOnce) {
                    const int which = i + lane / kRowLanes;
                    const int64_t at = __shfl_sync(0xffffffffu, from, which);
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (h * kBlockM + quarter * 32 + which < seg.rows) {
                        const T* const x = p.q + at + lane % kRowLanes * 8;
                        if (p.q_vec) {
                            w = __ldcs(reinterpret_cast<const uint4*>(x));  // not the read-only path: o may be q
                        } else {
                            float f[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] = VecTraits<T>::to_float(x[e]);
                            w = VecTraits<T>::pack(f);
                        }
                    }
                    raw[i / kAtOnce] = w;
                }
#pragma unroll
                for (int i = 0; i < 32; i += kAtOnce) {
                    const int which = i + lane / kRowLanes, c = lane % kRowLanes;
                    float f[8];
                    VecTraits<T>::unpack(raw[i / kAtOnce], f);
                    float unit = 1.f, mine = to_log2;
                    if (kBf16) {
                        float big = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(f[e]));
#pragma unroll
                        for (int x = 1; x < kRowLanes; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, x));
                        // 2^13 / (the power of two below the largest), and its inverse for the scores; ordinary exponents only
                        const int e = min(max(static_cast<int>(__float_as_uint(big) >> 23), 24), 254) - 13;
                        if (big > 0.f && big < INFINITY) {
                            unit = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
                            mine = to_log2 * __uint_as_float(static_cast<uint32_t>(e) << 23);
                        }
                    }
                    *reinterpret_cast<uint4*>(q_chunk(quarter * 32 + which, c)) =
                        make_uint4(pack_f16(f[0] * unit, f[1] * unit), pack_f16(f[2] * unit, f[3] * unit), pack_f16(f[4] * unit, f[5] * unit), pack_f16(f[6] * unit, f[7] * unit));
                    // to the lane whose row it is
                    const float got = __shfl_sync(0xffffffffu, mine, (lane - i) * kRowLanes & 31);
                    if (lane >= i && lane < i + kAtOnce) factors = got;
                }
                factor = factors;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full[h]);
            }
            auto publish = [&](int set) {  // weights that are in tensor memory
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * h + set]);
            };
            auto measure = [&]() {
                const bool none = d == -INFINITY;  // nothing but hidden columns, if the step's scales are near
                big_m = none ? -INFINITY : m_ref + d;
                near = none ? -kReach : fabsf(d) <= kReach && fabsf(m_ref) <= kNearZero ? d - kBelow : INFINITY;
                conv = ex2(d);
            };
            // O times alpha. The scores of step t were asked for behind the product with values of t - 2, so only that of t - 1 may be under way.
            auto scale_o = [&](int t, float alpha) {
                const int other = (t & 1) ^ 1;
                wait(&pv_done[2 * h + other], (sets[other] - 1) & 1, 10);
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_taddr + c0, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
                    tmem_st32(o_taddr + c0, o);
                }
            };
            // Ordinary steps are the inner loop, one exponential a score; a step whose value scales lie too far from one another or from the
            // references is taken by itself behind it.
            for (int t = 0; t < steps && ok; ++t) {
                int set;
                uint32_t taddr, missing;
                int32_t first;
                for (; t < steps; ++t) {
                    set = t & 1;
                    wait(&s_full[2 * h + set], sets[set]++ & 1, 8);
                    if (!ok) break;
                    tc_fence_after();
                    taddr = s_taddr + set * kStep;
                    uint32_t sr[64], packed[32];
                    tmem_ld32(taddr, sr);
                    tmem_ld32(taddr + 32, sr + 32);
                    const Scales& sc = scales[(block0 + (t >> 1)) % kSlots];
                    first = bl.kb0 * kBlockN + t * kStep;
                    missing = sc.missing >> (set * 4) & 15u;
                    const Step st(sc, set, factor);
                    const bool mask = __any_sync(0xffffffffu, first + kStep > seen) || missing != 0;
                    const float least = sc.least[set];
                    tmem_ld_wait();
                    // A step looks at its own maximum first; where it would push weights out of fp16 (a piece's first step, rarely later)
                    // O is scaled anew. m_ref can stay: ordinary scores are within kBelow + kGrowth of it, and it need not be a maximum.
                    const float mx = mask ? largest_of<true>(sr, st, missing, first, seen) : largest_of<false>(sr, st, missing, first, seen);
                    const bool grow = mx > big_m + kGrowth;
                    if (__any_sync(0xffffffffu, grow)) {
                        if (__any_sync(0xffffffffu, grow && !(fabsf(mx) <= kNearZero && fabsf(least) <= kReach))) break;
                        const float to = floorf(mx), alpha = grow ? ex2(big_m - to) : 1.f;
                        if (grow) {
                            if (m_ref == -INFINITY) m_ref = to - floorf(least);
                            d = to - m_ref;
                        }
                        measure();
                        if (t > 0) scale_o(t, alpha);
                    }
                    if (__any_sync(0xffffffffu, !(least >= near))) break;
                    float out_again[4];
                    load_f32<4>(sc.out_again + set * 4, out_again);
                    if (mask) weights_of<true>(sr, st, out_again, missing, reference(big_m), conv, first, seen, packed, &l);
                    else weights_of<false>(sr, st, out_again, missing, big_m, conv, first, seen, packed, &l);
                    tmem_st32(taddr, packed);  // over scores that have been read
                    publish(set);
                }
                if (!ok || t >= steps) break;
                // Step t by itself, a group at a time: the largest z, the largest z - m + log2 vs, and then weights and the sum, which has
                // exponentials of its own.
                const Scales& sc = scales[(block0 + (t >> 1)) % kSlots];
                float top = -INFINITY, big_top = -INFINITY, sum = 0.f, m = 0.f;
#pragma unroll 1
                for (int i = 0; i < 12; ++i) {
                    const int g = i & 3;
                    const float f = factor * sc.key[set * 4 + g], plus = sc.value_log2[set * 4 + g];
                    const int32_t there = missing >> g & 1 ? 0 : seen - first - g * 16;  // columns of the group that the row sees
                    if (i == 4) {
                        if (top > m_ref + kGrowth) {
                            const float to = floorf(top);
                            l *= m_ref == -INFINITY ? 0.f : ex2(m_ref - to);
                            d += m_ref == -INFINITY ? 0.f : m_ref - to;
                            m_ref = to;
                        }
                        m = reference(m_ref);
                    }
                    if (i == 8) {
                        const bool grow = big_top > d + kGrowth;
                        const float to = floorf(big_top), alpha = !grow ? 1.f : ex2(d - to);
                        if (grow) d = to;
                        if (t > 0 && __any_sync(0xffffffffu, grow)) scale_o(t, alpha);
                    }
                    uint32_t x[16], packed[8];
                    tmem_ld16(taddr + g * 16, x);
                    tmem_ld_wait();
                    if (i < 4) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) top = c < there ? fmaxf(top, __uint_as_float(x[c]) * f) : top;
                    } else if (i < 8) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) big_top = c < there ? fmaxf(big_top, fmaf(__uint_as_float(x[c]), f, -m) + plus) : big_top;
                    } else {
                        const float off = plus + (kUnitLog2 - reference(d));
#pragma unroll
                        for (int c = 0; c < 16; c += 2) {
                            float e[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const float z = fmaf(__uint_as_float(x[c + j]), f, -m);
                                e[j] = c + j < there ? ex2(z + off) : 0.f;
                                sum += c + j < there ? ex2(z) : 0.f;
                            }
                            packed[c / 2] = pack_f16(e[0], e[1]);
                        }
                        tmem_st8(taddr + g * 8, packed);  // over scores that have been read
                    }
                }
                l += sum;
                measure();
                publish(set);
            }
            if (!ok) break;
            // The next piece's first product with values waits for this warp's weights, which come after these reads.
            const int last_set = (steps - 1) & 1;
            if (steps > 0) wait(&pv_done[2 * h + last_set], (sets[last_set] - 1) & 1, 9);
            if (!ok) break;
            if (steps > 0) tc_fence_after();
            const bool nothing = l == 0.f;
            // 2^d may be out of fp32 where the result is not: its root comes twice
            const float half = ex2(0.5f * (d - kUnitLog2)), by = half / l;
            float* const out = work.partial(p, seg, D);
            // Results leave through the warp's part of q (its scores are done), so that whole rows are written at a time: 64 fp32 elements of
            // a row, or all 16-bit ones, at once.
            const int64_t to = token * p.os[0] + q_head * p.os[1];
            constexpr int kPassElems = D == 128 ? 64 : 32;  // fp32 elements of a row that its bytes of q hold
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += kPassElems) {
#pragma unroll
                for (int part = 0; part < kPassElems; part += 32) {
                    uint32_t o[32];
                    if (steps > 0) {
                        tmem_ld32(o_taddr + c0 + part, o);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = steps == 0 || nothing ? 0u : __float_as_uint(__uint_as_float(o[c]) * half * by);
                    if (seg.cut) {
#pragma unroll
                        for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(q_chunk(row, (part + c) / 4)) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            *reinterpret_cast<uint4*>(q_chunk(row, (c0 + part + c) / 8)) =
                                make_uint4(pack_out<kBf16>(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), pack_out<kBf16>(__uint_as_float(o[c + 2]), __uint_as_float(o[c + 3])),
                                           pack_out<kBf16>(__uint_as_float(o[c + 4]), __uint_as_float(o[c + 5])), pack_out<kBf16>(__uint_as_float(o[c + 6]), __uint_as_float(o[c + 7])));
                    }
                }
                __syncwarp();
                if (seg.cut || c0 + kPassElems >= D) {
#pragma unroll 4
                    for (int i = 0; i < 32; i += kAtOnce) {
                        const int which = i + lane / kRowLanes, c = lane % kRowLanes, of_row = quarter * 32 + which;
                        const int64_t at = __shfl_sync(0xffffffffu, to, which);
                        const uint4 w = *reinterpret_cast<const uint4*>(q_chunk(of_row, c));
                        if (h * kBlockM + of_row >= seg.rows) continue;
                        if (seg.cut) {
                            *reinterpret_cast<uint4*>(out + 2 * kRows + (h * kBlockM + of_row) * D + c0 + c * 4) = w;
                        } else if (p.o_vec == 2) {
                            *reinterpret_cast<uint4*>(p.o + at + c * 8) = w;
                        } else {
                            const T* const x = reinterpret_cast<const T*>(&w);
#pragma unroll
                            for (int e = 0; e < 8; ++e) p.o[at + c * 8 + e] = x[e];
                        }
                    }
                    __syncwarp();
                }
            }
            if (r < seg.rows) {
                if (seg.cut) {  // the sum's power of two goes to its reference, which may have stayed behind: other pieces are weighed by that
                    const float up = whole_log2(l);
                    out[r] = m_ref + up;
                    out[kRows + r] = l * ex2(-up);
                } else if (p.lse != nullptr) {
                    p.lse[token * p.q_heads + q_head] = nothing ? -INFINITY : (m_ref + log2f(l)) * 0.6931471805599453f;
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
int launch(const CachedParams<T>& p, cudaStream_t stream) {
    auto kernel = cached_attention_tc_kernel<T, D>;
    static std::atomic<bool> smem_set[64];
    if (int st = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), Smem<D>::kTotal, smem_set)) return st;
    kernel<<<kLongGrid, kThreads, Smem<D>::kTotal, stream>>>(p);
    MHLO_CUDA_CHECK_LAUNCH("cached_attention (tcgen05)");
    return MHLO_CUDA_OK;
}

}  // namespace

template <typename T>
int cached_attention_long(const CachedParams<T>& p, cudaStream_t stream) {
    static_assert(kRows == kLongRows, "rows of a segment");
    return p.kv.head_dim == 64 ? launch<T, 64>(p, stream) : launch<T, 128>(p, stream);
}
template int cached_attention_long<__half>(const CachedParams<__half>&, cudaStream_t);
template int cached_attention_long<__nv_bfloat16>(const CachedParams<__nv_bfloat16>&, cudaStream_t);

int cached_attention_long_device_error() { return take_kv_error(); }

}  // namespace mhlo
