// What the tensor-core kernels of attention over packed sequences share: tensor maps, loads of tiles with the rows behind a sequence's
// end cleared, and the instructions that tc_ptx.cuh lacks.
#pragma once

#include <atomic>
#include <string>
#include <type_traits>

#include "packed_attention.cuh"
#include "tc_ptx.cuh"

namespace mhlo {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

// Instruction descriptor: fp32 accumulators, 128 rows, n columns; b_mn: B's rows (of the sum) lie one below the other in shared memory.
__device__ __forceinline__ uint32_t instruction(bool bf16, bool b_mn, uint32_t n) {
    const uint32_t fmt = bf16 ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);
}

// A tile of 128 rows of up to 64 PANELS elements in shared memory: panels of 64 elements, 128 bytes a row, swizzled.
constexpr int kPanelBytes = 128 * 128;

// Loads a tile, by a whole warp: `rows` rows that the box of `map` brings, of which the first `valid` belong to the sequence. c1, c2, c3: the box's
// coordinates. full: gets the bytes. Where rows are of another sequence, or of none, and the product would sum over them (clear), they become
// zeros: a weight of zero does not hide an infinity. The warp then waits for the bytes itself (on `own`, whose parity is *own_phase) and
// clears them before it arrives on full. False: the wait ran out.
template <int PANELS>
__device__ __forceinline__ bool load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* full, uint64_t* own, uint32_t* own_phase, int rows, int valid, bool clear, int c1,
                                          int c2, int c3) {
    const int lane = threadIdx.x & 31;
    const bool wait = clear && valid < rows;
    uint64_t* const bar = wait ? own : full;
    if (lane == 0) {
        mbar_expect_tx(bar, PANELS * rows * 128);
#pragma unroll
        for (int pn = 0; pn < PANELS; ++pn) tma_load_4d(dst + pn * kPanelBytes, map, bar, pn * 64, c1, c2, c3);
    }
    if (!wait) return true;
    const bool there = mbar_wait(own, *own_phase);
    *own_phase ^= 1;
    if (!there) return false;
    for (int i = valid * 8 + lane; i < rows * 8; i += 32) {
#pragma unroll
        for (int pn = 0; pn < PANELS; ++pn) *reinterpret_cast<uint4*>(dst + pn * kPanelBytes + i * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(full);
    return true;
}

__device__ __forceinline__ void load64(uint32_t taddr, uint32_t* r) {
    tmem_ld32(taddr, r);
    tmem_ld32(taddr + 32, r + 32);
    tmem_ld_wait();
}

// 32 bytes at once: a whole sector of L2. Halves of one, 16 bytes each, are as many requests as there are 16 bytes.
__device__ __forceinline__ void store32(void* to, const uint4& a, const uint4& b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}

// 32 elements of a row's result, those below dim. wide: rows and dim on the 32-byte grid.
template <bool BF16>
__device__ __forceinline__ void store_result(uint8_t* to, const uint32_t* x, float factor, int c0, int dim, bool wide) {
#pragma unroll
    for (int c = 0; c < 32; c += 16) {
        uint4 w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t* const e = x + c + 8 * i;
            w[i].x = pack16<BF16>(__uint_as_float(e[0]) * factor, __uint_as_float(e[1]) * factor);
            w[i].y = pack16<BF16>(__uint_as_float(e[2]) * factor, __uint_as_float(e[3]) * factor);
            w[i].z = pack16<BF16>(__uint_as_float(e[4]) * factor, __uint_as_float(e[5]) * factor);
            w[i].w = pack16<BF16>(__uint_as_float(e[6]) * factor, __uint_as_float(e[7]) * factor);
        }
        if (wide) {
            if (c0 + c < dim) store32(to + (c0 + c) * 2, w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (c0 + c + 8 * i < dim) *reinterpret_cast<uint4*>(to + (c0 + c + 8 * i) * 2) = w[i];
        }
    }
}
inline bool on_wide_grid(const PackedTensor& t, int32_t dim, int32_t tokens, int32_t heads) {
    return (reinterpret_cast<uintptr_t>(t.base) & 31) == 0 && dim % 16 == 0 && (tokens == 1 || t.token % 16 == 0) && (heads == 1 || t.head % 16 == 0);
}

// ---- items ------------------------------------------------------------------------------------------------------------------------------
// The grid has a CTA for every item there could be; those that run take over, one by one, the items of CTAs that have not been launched yet
// (cluster launch control). Items come in the order of the plan to whichever CTA is free: dealt out in advance, runs of sequences that share L2
// left CTAs idle for 6 to 35 percent of the time. The producer's warp asks, reads the plan's entry and hands it on through a ring, an item ahead
// of the one that it loads: the issuer wants to know whether there is a next one before it is through with this.
constexpr int kTileSlots = 4;
struct ItemRing {
    uint4 response;
    int4 entry[kTileSlots];
    int32_t part[kTileSlots];
    uint64_t asked, full[kTileSlots], empty[kTileSlots];
    __device__ __forceinline__ void init(int consumers) {  // one thread, before the barriers' fence
        mbar_init(&asked, 1);
        for (int s = 0; s < kTileSlots; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], consumers);
        }
    }
};

// The producer's side, for a whole warp.
struct ItemSource {
    ItemRing& ring;
    const PackedArgs& a;
    const int4* list;
    int64_t items;
    int32_t each;  // items of an entry
    uint32_t taken = 0, given = 0;
    __device__ __forceinline__ ItemSource(ItemRing& r, const PackedArgs& args, bool keys, int32_t items_of_entry)
        : ring(r), a(args), list(keys ? args.key_tiles() : args.row_tiles()), each(items_of_entry) {
        const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
        items = a.matches(h) ? static_cast<int64_t>(keys ? h.key_tiles : h.row_tiles) * each : 0;
    }
    __device__ __forceinline__ void ask() {
        fence_proxy_async();  // the answer before has been read
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            mbar_expect_tx(&ring.asked, 16);
            asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(&ring.response)),
                         "r"(smem_u32(&ring.asked))
                         : "memory");
        }
    }
    // The CTA whose item this one takes over, -1: none is left.
    __device__ __forceinline__ int64_t answer() const {
        uint32_t cancelled, x;
        asm volatile(
            "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
            "ld.shared.b128 r, [%2];\n\t"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "mov.u32 %1, 0;\n\t"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
            : "=r"(cancelled), "=r"(x)
            : "r"(smem_u32(&ring.response))
            : "memory");
        return cancelled ? static_cast<int64_t>(x) : -1;
    }
    // The next item, already handed on; false: no more (handed on as well), or a wait ran out (*ok). wanted(e, part): whether there is anything to do.
    template <typename Wanted>
    __device__ __forceinline__ bool next(int4* e, int32_t* part, bool* ok, Wanted wanted) {
        for (;;) {
            int64_t id = blockIdx.x;
            if (taken > 0) {
                if (!mbar_wait(&ring.asked, (taken - 1) & 1)) return *ok = false;
                id = answer();
            }
            if (id < 0) break;
            ++taken;
            ask();
            if (id >= items) continue;
            *e = list[static_cast<uint32_t>(id) / static_cast<uint32_t>(each)];
            *part = static_cast<int32_t>(static_cast<uint32_t>(id) % static_cast<uint32_t>(each));
            if (!a.inside(*e)) {
                kv_report(MHLO_CUDA_KV_ERROR_PLAN);
                continue;
            }
            if (wanted(*e, *part)) return give(*e, *part, ok);
        }
        give(make_int4(0, 0, 0, 0), 0, ok);
        return false;
    }
    // Behind a wait that ran out: no answer may come to shared memory that is no longer this CTA's.
    __device__ __forceinline__ void drain() const {
        if (taken > 0) mbar_wait(&ring.asked, (taken - 1) & 1);
    }
    __device__ __forceinline__ bool give(const int4& e, int32_t part, bool* ok) {
        const uint32_t slot = given % kTileSlots;
        if (!mbar_wait(&ring.empty[slot], (given / kTileSlots & 1) ^ 1)) return *ok = false;
        ++given;
        if ((threadIdx.x & 31) == 0) {
            ring.entry[slot] = e;
            ring.part[slot] = part;
            mbar_arrive(&ring.full[slot]);
        }
        __syncwarp();
        return true;
    }
};

// The others' side, for each of their warps.
struct ItemSink {
    ItemRing& ring;
    uint32_t taken = 0;
    __device__ __forceinline__ explicit ItemSink(ItemRing& r) : ring(r) {}
    __device__ __forceinline__ bool next(int4* e, int32_t* part, bool* ok) {
        const uint32_t slot = taken % kTileSlots;
        if (!mbar_wait(&ring.full[slot], taken / kTileSlots & 1)) return *ok = false;
        ++taken;
        *e = ring.entry[slot];
        *part = ring.part[slot];
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[slot]);
        return e->y > 0;
    }
};

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline int encode_map(CUtensorMap* map, const void* base, const cuuint64_t (&dims)[4], const int64_t (&strides)[3], const cuuint32_t (&box)[4]) {
    static std::atomic<EncodeFn> known{nullptr};
    EncodeFn encode = known.load(std::memory_order_acquire);
    if (encode == nullptr) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) != cudaSuccess || fn == nullptr)
            return fail(MHLO_CUDA_EXECUTION_FAILED, "packed_attention: cuTensorMapEncodeTiled is not available from this driver");
        encode = reinterpret_cast<EncodeFn>(fn);
        known.store(encode, std::memory_order_release);
    }
    cuuint64_t bytes[3];
    for (int i = 0; i < 3; ++i)  // the stride of a dimension of one entry does not matter
        bytes[i] = dims[i + 1] == 1 ? static_cast<cuuint64_t>((dims[0] * 2 + 15) / 16 * 16) : static_cast<cuuint64_t>(strides[i] * 2);
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, bytes, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MHLO_CUDA_OK : fail(MHLO_CUDA_EXECUTION_FAILED, "packed_attention: cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
}

// Rows of queries: {element, head of the group, head of keys, token}; elements behind head_dim arrive as zeros.
inline int query_map(CUtensorMap* map, const PackedTensor& t, const PackedArgs& a) {
    const auto n = [](int64_t x) { return static_cast<cuuint64_t>(x); };
    const cuuint64_t dims[4] = {n(a.head_dim), n(a.group), n(a.kv_heads), n(a.tokens)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(a.group), 1, static_cast<cuuint32_t>(a.half_tokens)};
    return encode_map(map, t.base, dims, {t.head, t.head * a.group, t.token}, box);
}
inline int key_map(CUtensorMap* map, const PackedTensor& t, const PackedArgs& a) {
    const auto n = [](int64_t x) { return static_cast<cuuint64_t>(x); };
    const cuuint64_t dims[4] = {n(a.head_dim), n(a.kv_heads), n(a.tokens), 1};
    const cuuint32_t box[4] = {64, 1, kKeyTile, 1};
    return encode_map(map, t.base, dims, {t.head, t.token, 0}, box);
}

}  // namespace
}  // namespace mhlo
