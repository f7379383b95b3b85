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
// first token of the tile inside it, 0}: long tiles first, then runs of sequences whose keys and values stay in L2 together (run_tokens), inside
// a run in descending order of the tokens that they meet. In one order for all, 64 sequences of 512 tokens read 603 MB where they have 403.
struct PlanHeader {
    int32_t magic, tokens, q_heads, kv_heads, causal, row_tiles, key_tiles;
    int32_t first, end;  // rows of the sequences
    int32_t seqs;        // how far the second list lies behind the first goes by them
    int32_t reserved[2];
};

struct PackedArgs {
    const int32_t* starts;
    void* plan;
    int32_t seqs, tokens, q_heads, kv_heads, group, head_dim, causal;
    int32_t half_tokens;  // tokens whose rows a half tile holds
    int32_t row_capacity, key_capacity;  // entries of the two lists
    int32_t run_tokens;
    __host__ __device__ __forceinline__ const int4* row_tiles() const { return reinterpret_cast<const int4*>(static_cast<const char*>(plan) + sizeof(PlanHeader)); }
    __host__ __device__ __forceinline__ const int4* key_tiles() const { return row_tiles() + row_capacity; }
    // Whether the plan is one of such a batch; one thread reports (not in launches beside the tensor-core kernels of the same call, whose word is another: report).
    __device__ __forceinline__ bool matches(const PlanHeader& h, bool report = true) const {
        const bool ok = h.magic == kPlanMagic && h.seqs == seqs && h.tokens == tokens && h.q_heads == q_heads && h.kv_heads == kv_heads && h.causal == causal &&
                        h.row_tiles >= 0 && h.row_tiles <= row_capacity && h.key_tiles >= 0 && h.key_tiles <= key_capacity;
        if (!ok && report && threadIdx.x == 0) kv_report(MHLO_CUDA_KV_ERROR_PLAN);
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

// Floats of the norms that the backward half takes of f16 tensors.
inline int64_t packed_norms(int32_t dtype, const PackedArgs& a) {
    return dtype == MHLO_DT_F16 ? (static_cast<int64_t>(a.tokens) * (a.q_heads + 3 * a.kv_heads) + 3) / 4 * 4 : 0;
}

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
    // f16: the largest norms of a row of grad and of a row of v in a sequence, at its first token of [kv_heads][tokens]; norms of grad's rows, laid out like stats, and of
    // v's, [kv_heads][tokens]
    float2* largest() const { return stats() + (static_cast<int64_t>(a.tokens) * a.q_heads + 1) / 2 * 2; }
    float* grad_norms() const { return reinterpret_cast<float*>(largest() + static_cast<int64_t>(a.tokens) * a.kv_heads); }
    float* value_norms() const { return grad_norms() + static_cast<int64_t>(a.tokens) * a.q_heads; }
    // Gradients of keys and values that several CTAs share, [splits][dk, dv][tokens][kv_heads][head_dim]
    float* shares() const { return reinterpret_cast<float*>(largest()) + packed_norms(dtype, a); }
};

// Into how many shares the rows that see a tile of keys are cut where `items` tiles would leave most of `ctas` without work.
inline int32_t key_splits(int64_t items, int64_t ctas) {
    return static_cast<int32_t>(items >= ctas ? 1 : items < 1 ? 1 : (ctas + items - 1) / items > 16 ? 16 : (ctas + items - 1) / items);
}
inline int32_t key_splits_tc(const PackedArgs& a) { return key_splits(static_cast<int64_t>(a.key_capacity) * a.kv_heads, kNumSMs); }
// Joins them in order (packed_attention.cu).
int packed_join_shares(const PackedCall& c, int32_t splits, cudaStream_t stream);

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

struct RowTile {
    int32_t first, n, t0, head;  // the sequence's first token and its tokens, the tile's first token inside it, head of keys
    int32_t nb[kHalves], nblk;   // key blocks of each half (0: it has no rows), and of the tile (0: there is none)
};

// Item `part` of an entry of query rows, heads next to each other: a tile's two halves together, or (one_half) each by itself, the second half of the
// RowTile is then empty.
__device__ __forceinline__ RowTile row_tile(const PackedArgs& a, bool one_half, const int4& e, int32_t part) {
    RowTile t;
    const bool later = one_half && part < a.kv_heads;  // the later half first: it is the longer one
    t.head = part >= a.kv_heads ? part - a.kv_heads : part;
    t.first = e.x;
    t.n = e.y;
    t.t0 = e.z + (later ? a.half_tokens : 0);
    const int32_t all = (t.n + kKeyTile - 1) / kKeyTile;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        const int32_t from = t.t0 + h * a.half_tokens, to = min(t.n, from + a.half_tokens);
        t.nb[h] = from >= t.n || (h > 0 && one_half) ? 0 : a.causal ? (to + kKeyTile - 1) / kKeyTile : all;
    }
    t.nblk = max(t.nb[0], t.nb[1]);
    return t;
}

struct KeyTile {
    int32_t first, n, k0, head;
    int32_t b0, b1;  // half tiles of query rows that see the tile's keys: this share of them, which may be empty
    int32_t split;
};
__device__ __forceinline__ KeyTile key_tile(const PackedArgs& a, int32_t splits, const int4& e, int32_t part) {
    KeyTile t;
    t.split = splits > 1 ? part / a.kv_heads : 0;
    t.head = part - t.split * a.kv_heads;
    t.first = e.x;
    t.n = e.y;
    t.k0 = e.z;
    t.b0 = a.causal ? e.z / a.half_tokens : 0;
    t.b1 = (e.y + a.half_tokens - 1) / a.half_tokens;
    if (splits > 1) {
        const int64_t all = t.b1 - t.b0;
        t.b1 = t.b0 + static_cast<int32_t>(all * (t.split + 1) / splits);
        t.b0 += static_cast<int32_t>(all * t.split / splits);
    }
    return t;
}

}  // namespace
}  // namespace mhlo
