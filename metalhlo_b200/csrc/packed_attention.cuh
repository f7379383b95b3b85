// What the kernels of attention over packed sequences share: the plan of a batch (its sequences cut into tiles, longest first), and how
// CTAs walk it.
//
// Query heads that read one head of keys are stacked: row r of a run of tokens is token r / group, query head head * group + r % group.
// A half tile holds the rows of kRows / group whole tokens, so that one tensor-map box of {64 elements, group heads, tokens} is its rows
// one below the other, a causal mask cuts the same keys off all heads of a token, and keys and values are fetched once for the group.
#pragma once

#include "kv_cache.cuh"

namespace mhlo {

constexpr int kRows = 128;        // of a half tile: stacked rows of queries
constexpr int kHalves = 2;
constexpr int kKeyTile = 128;     // keys of a block, and of a tile of the gradients of keys and values
constexpr int kPlanMagic = 0x506c616e;

// The plan in device memory: a header, then the tiles of query rows, then the tiles of keys, each {first token of the sequence, its tokens,
// first token of the tile inside it, 0}, in descending order of the tokens that they meet.
struct PlanHeader {
    int32_t magic, tokens, q_heads, kv_heads, causal, row_tiles, key_tiles;
    int32_t first, end;  // rows of the sequences
    int32_t reserved[3];
};

struct PackedArgs {
    const int32_t* starts;
    void* plan;
    int32_t seqs, tokens, q_heads, kv_heads, group, head_dim, causal;
    int32_t half_tokens;  // tokens whose rows a half tile holds
    int32_t row_capacity, key_capacity;  // entries of the two lists
    __host__ __device__ __forceinline__ const int4* row_tiles() const { return reinterpret_cast<const int4*>(static_cast<const char*>(plan) + sizeof(PlanHeader)); }
    __host__ __device__ __forceinline__ const int4* key_tiles() const { return row_tiles() + row_capacity; }
    // Whether the plan is one of such a batch; one thread reports.
    __device__ __forceinline__ bool matches(const PlanHeader& h) const {
        const bool ok = h.magic == kPlanMagic && h.tokens == tokens && h.q_heads == q_heads && h.kv_heads == kv_heads && h.causal == causal &&
                        h.row_tiles >= 0 && h.row_tiles <= row_capacity && h.key_tiles >= 0 && h.key_tiles <= key_capacity;
        if (!ok && threadIdx.x == 0) kv_report(MHLO_CUDA_KV_ERROR_PLAN);
        return ok;
    }
    __device__ __forceinline__ bool inside(const int4& e) const {
        return e.x >= 0 && e.y > 0 && e.y <= tokens - e.x && e.z >= 0 && e.z < e.y;
    }
};

// A [tokens, heads, head_dim] tensor: element strides {token, head}.
struct PackedTensor {
    void* base = nullptr;
    int64_t token = 0, head = 0;
};

// A call of the forward or backward half.
struct PackedCall {
    PackedArgs a;
    int32_t dtype;
    float scale;
    PackedTensor q, k, v, o, grad, dq, dk, dv;
    float* lse;
    void* scratch;
    // of scratch: what the backward half needs of a row, [kv_heads][tokens][group]: -lse log2(e), and grad . o
    float2* stats() const { return static_cast<float2*>(scratch); }
    // fp16: the largest squared norms of a row of grad and of a row of v, as bits
    uint32_t* norms() const { return reinterpret_cast<uint32_t*>(stats() + static_cast<int64_t>(a.tokens) * a.q_heads); }
};

// Whether the tensor-core kernels read or write the tensor in place: rows on the 16-byte grid, none that repeats itself.
inline bool packed_on_grid(const PackedTensor& t, int32_t tokens, int32_t heads) {
    return aligned16(t.base) && (tokens == 1 || (t.token > 0 && t.token % 8 == 0)) && (heads == 1 || (t.head > 0 && t.head % 8 == 0));
}

// 16-bit types, head dimensions that are multiples of 8 up to 128 (packed_attention_tc.cu, packed_attention_grad_tc.cu).
int packed_attention_tc(const PackedCall& c, cudaStream_t stream);
int packed_attention_grad_tc(const PackedCall& c, cudaStream_t stream);
int packed_attention_tc_device_error();
int packed_attention_grad_tc_device_error();

namespace {

// Work is dealt out in passes over the CTAs, forwards and backwards in turn: items come longest first, so the CTA that got the longest of
// one pass gets the shortest of the next.
struct Dealt {
    int32_t pass = 0;
    __device__ __forceinline__ int64_t next() {
        const int32_t g = gridDim.x, c = blockIdx.x;
        const int64_t i = static_cast<int64_t>(pass) * g + ((pass & 1) ? g - 1 - c : c);
        ++pass;
        return i;
    }
    // Item of a list of `items`, -1 behind the last pass that holds any.
    __device__ __forceinline__ int64_t next(int64_t items) {
        while (static_cast<int64_t>(pass) * gridDim.x < items) {
            const int64_t i = next();
            if (i < items) return i;
        }
        return -1;
    }
};

struct RowTile {
    int32_t first, n, t0, head;  // the sequence's first token and its tokens, the tile's first token inside it, head of keys
    int32_t nb[kHalves], nblk;   // key blocks of each half (0: it has no rows), and of the tile
};

// Items of query rows: a tile's two halves together, or each by itself (the second half of a RowTile is then empty).
struct RowWalk {
    Dealt dealt;
    const PackedArgs& a;
    int64_t items;
    int32_t one_half;
    __device__ __forceinline__ RowWalk(const PackedArgs& args, int32_t one) : a(args), one_half(one) {
        const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
        items = a.matches(h) ? static_cast<int64_t>(h.row_tiles) * a.kv_heads * (one ? 2 : 1) : 0;
    }
    __device__ __forceinline__ bool next(RowTile* t) {
        for (;;) {
            const int64_t i = dealt.next(items);
            if (i < 0) return false;
            const uint32_t entry = static_cast<uint32_t>(i) / static_cast<uint32_t>(a.kv_heads);
            t->head = static_cast<uint32_t>(i) - entry * a.kv_heads;
            const int4 e = a.row_tiles()[one_half ? entry >> 1 : entry];
            if (!a.inside(e)) {
                kv_report(MHLO_CUDA_KV_ERROR_PLAN);
                continue;
            }
            t->first = e.x;
            t->n = e.y;
            t->t0 = e.z + (one_half && (entry & 1) == 0 ? a.half_tokens : 0);  // the later half first: it is the longer one
            if (t->t0 >= t->n) continue;
            const int32_t all = (t->n + kKeyTile - 1) / kKeyTile;
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const int32_t from = t->t0 + h * a.half_tokens, to = min(t->n, from + a.half_tokens);
                t->nb[h] = from >= t->n || (h > 0 && one_half) ? 0 : a.causal ? (to + kKeyTile - 1) / kKeyTile : all;
            }
            t->nblk = max(t->nb[0], t->nb[1]);
            return true;
        }
    }
};

struct KeyTile {
    int32_t first, n, k0, head;
    int32_t b0, b1;  // half tiles of query rows that see the tile's keys
};

struct KeyWalk {
    Dealt dealt;
    const PackedArgs& a;
    int64_t items;
    __device__ __forceinline__ explicit KeyWalk(const PackedArgs& args) : a(args) {
        const PlanHeader h = *static_cast<const PlanHeader*>(a.plan);
        items = a.matches(h) ? static_cast<int64_t>(h.key_tiles) * a.kv_heads : 0;
    }
    __device__ __forceinline__ bool next(KeyTile* t) {
        for (;;) {
            const int64_t i = dealt.next(items);
            if (i < 0) return false;
            const uint32_t entry = static_cast<uint32_t>(i) / static_cast<uint32_t>(a.kv_heads);
            t->head = static_cast<uint32_t>(i) - entry * a.kv_heads;
            const int4 e = a.key_tiles()[entry];
            if (!a.inside(e)) {
                kv_report(MHLO_CUDA_KV_ERROR_PLAN);
                continue;
            }
            t->first = e.x;
            t->n = e.y;
            t->k0 = e.z;
            t->b0 = a.causal ? e.z / a.half_tokens : 0;
            t->b1 = (e.y + a.half_tokens - 1) / a.half_tokens;
            return true;
        }
    }
};

}  // namespace
}  // namespace mhlo
