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
