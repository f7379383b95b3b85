// The clipped policy loss with a KL term, and its gradient: for token t with log probability p, that of the policy it was sampled from, o, and
// optionally of a reference policy, f, its advantage a and its weight w (1 / counted tokens, or 1 / (counted tokens of its sequence * sequences)),
//   ratio = exp(p - o), x = f - p
//   loss = sum of w (-min(ratio a, clip(ratio, 1 - low, 1 + high) a) + kl_weight (exp(x) - x - 1))
//   dloss/dp = w ((clipped ? 0 : -ratio a) + kl_weight (1 - exp(x))).
//
// Bound by HBM for millions of tokens (21 bytes each; 0.9 million take 12 us, two launches of it), by launches below (4000: 7.6 us): up to kSmall tokens one CTA counts, weighs and sums; more take a
// launch that counts and one that does the rest. Counts are integers, sums are fp64 in a fixed order. Whether a ratio is clipped goes by
// p - o in fp64 against the logarithms of the borders: in fp32 one token in some million next to a border would get the other gradient.
#include <algorithm>
#include <cmath>

#include "kv_cache.cuh"

namespace mhlo {
namespace {

constexpr int kEach = 4;  // tokens of a thread
constexpr int kThreads = 256, kSmallThreads = 1024;
// One CTA up to here: with a KL term and a mask, 4000 tokens take 6.0 us in it and 6.5 in two launches, 8192 10.0 and 6.6, 16 384 16.5 and 7.7; in sequences of 500 tokens
// 8.4 and 12.5, 12.2 and 12.5, 21.6 and 14.3; of 8 tokens 11.3 and 14.5, 20.6 and 14.1, 38.5 and 14.7.
constexpr int64_t kSmall = 4096;
constexpr int kSmallSeqs = 2048;  // whose starts and counts it has in shared memory: 16 KB

struct PolicyParams {
    const float *logprobs, *old_logprobs, *ref, *advantages;
    const uint8_t* mask;    // null: all count
    const int32_t* starts;  // null: one mean over all tokens
    float* grad;
    float* results;         // loss, KL, share of clipped tokens
    int32_t* counts;        // [sequences], then sequences that count, tickets of the two launches; without starts a count of each CTA that counts
    int32_t counters;       // those CTAs
    double* partial;        // [CTAs][3]
    int64_t tokens;
    int32_t seqs;
    double low, high;       // log(1 - low), log(1 + high)
    float border_low, border_high, kl_weight;
    int32_t vec;
};

struct Sums {
    double loss = 0, kl = 0, clipped = 0;
    __device__ __forceinline__ void add(const Sums& o) { loss += o.loss, kl += o.kl, clipped += o.clipped; }
};

// Through fp32 and what it leaves of x. Where the result is 0 or infinite anyway that rest may be whole units, or no number.
__device__ __forceinline__ float exp_of(double x) {
    const float near = static_cast<float>(x), e = expf(near);
    return fabsf(near) <= 128.f ? e * (1.f + static_cast<float>(x - near)) : e;
}

// exp(x) - x - 1 and exp(x) - 1; up to 1 by the series, whose terms do not cancel.
__device__ __forceinline__ void kl_terms(double x64, float* k3, float* em1) {
    const float x = static_cast<float>(x64);
    if (fabsf(x) <= 1.f) {
        float s = 1.f / 479001600.f;
        s = fmaf(s, x, 1.f / 39916800.f);
        s = fmaf(s, x, 1.f / 3628800.f);
        s = fmaf(s, x, 1.f / 362880.f);
        s = fmaf(s, x, 1.f / 40320.f);
        s = fmaf(s, x, 1.f / 5040.f);
        s = fmaf(s, x, 1.f / 720.f);
        s = fmaf(s, x, 1.f / 120.f);
        s = fmaf(s, x, 1.f / 24.f);
        s = fmaf(s, x, 1.f / 6.f);
        s = fmaf(s, x, 0.5f);
        *k3 = s * x * x;
        *em1 = x + *k3;
    } else {
        const float e = exp_of(x64);
        *em1 = e - 1.f;
        *k3 = e == INFINITY ? INFINITY : *em1 - x;
    }
}

// One token that counts: its gradient, and its share of the sums.
__device__ __forceinline__ float token(const PolicyParams& p, float logprob, float old, float ref, float a, double w, Sums* sums) {
    const double d = static_cast<double>(logprob) - static_cast<double>(old);
    const bool over = a > 0.f && d > p.high, under = a < 0.f && d < p.low;
    float loss, grad;
    if (over || under) {
        loss = -(over ? p.border_high : p.border_low) * a;
        grad = 0.f;
        sums->clipped += w;
    } else {
        grad = loss = -exp_of(d) * a;
    }
    if (p.ref != nullptr) {
        float k3, em1;
        kl_terms(static_cast<double>(ref) - static_cast<double>(logprob), &k3, &em1);
        sums->kl += w * k3;
        if (p.kl_weight != 0.f) {
            loss = fmaf(p.kl_weight, k3, loss);
            grad = fmaf(-p.kl_weight, em1, grad);
        }
    }
    sums->loss += w * loss;
    return static_cast<float>(w) * grad;
}

__device__ __forceinline__ uint32_t counted(const PolicyParams& p, int64_t first) {  // bit i: token first + i counts
    if (first >= p.tokens) return 0;
    const int n = static_cast<int>(min(static_cast<int64_t>(kEach), p.tokens - first));
    if (p.mask == nullptr) return (1u << n) - 1;
    uint32_t bits = 0;
    if (p.vec && n == kEach) {
        const uint32_t m = *reinterpret_cast<const uint32_t*>(p.mask + first);
#pragma unroll
        for (int i = 0; i < kEach; ++i) bits |= (m >> (8 * i) & 255u) != 0 ? 1u << i : 0u;
        return bits;
    }
    for (int i = 0; i < n; ++i) bits |= p.mask[first + i] != 0 ? 1u << i : 0u;
    return bits;
}

// Where a run of tokens lies among the sequences. A warp finds the sequence of its first token, its lanes go on from there.
struct Place {
    int32_t b, end;  // sequence (-1: none), and its end
    __device__ __forceinline__ void find(const int32_t* starts, int32_t seqs, int64_t warp_first, int64_t first) {
        b = kv_search(seqs, warp_first, [&](int32_t i) { return static_cast<int64_t>(starts[i]); });
        go(starts, seqs, first);
    }
    __device__ __forceinline__ void go(const int32_t* starts, int32_t seqs, int64_t t) {
        while (b + 1 < seqs && starts[b + 1] <= t) ++b;
        end = starts[b + 1];
    }
    __device__ __forceinline__ bool holds(const int32_t* starts, int64_t t) const { return starts[b] <= t && t < end; }
};

struct Tokens {
    float logprob[kEach], old[kEach], ref[kEach], a[kEach];
    __device__ __forceinline__ void load(const PolicyParams& p, int64_t first) {
        auto get = [&](const float* from, float* to) {
            if (p.vec && first + kEach <= p.tokens) {
                const float4 v = *reinterpret_cast<const float4*>(from + first);
                to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < kEach; ++i) to[i] = first + i < p.tokens ? from[first + i] : 0.f;
            }
        };
        get(p.logprobs, logprob);
        get(p.old_logprobs, old);
        get(p.advantages, a);
        if (p.ref != nullptr) get(p.ref, ref);
    }
};

__device__ __forceinline__ void store(const PolicyParams& p, int64_t first, const float* grad) {
    if (p.vec && first + kEach <= p.tokens) {
        *reinterpret_cast<float4*>(p.grad + first) = make_float4(grad[0], grad[1], grad[2], grad[3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        if (first + i < p.tokens) p.grad[first + i] = grad[i];
}

// Gradients and sums of the tokens first .. first + 3. weight(b): of a token of sequence b; asked for once where all four are in one.
template <typename Weight>
__device__ __forceinline__ void step(const PolicyParams& p, const int32_t* starts, int64_t first, uint32_t bits, const Tokens& t, Place place, Sums* sums, Weight weight) {
    float grad[kEach];
    int32_t of = -1;
    double w = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        grad[i] = 0.f;
        if (!(bits >> i & 1)) continue;
        if (starts != nullptr) {
            place.go(starts, p.seqs, first + i);
            if (!place.holds(starts, first + i)) continue;
        }
        if (place.b != of) of = place.b, w = weight(of);
        grad[i] = token(p, t.logprob[i], t.old[i], t.ref[i], t.a[i], w, sums);
    }
    if (first < p.tokens) store(p, first, grad);
}

// Adds one to the counts of the tokens' sequences, up to four at once.
template <typename Add>
__device__ __forceinline__ void count(const PolicyParams& p, const int32_t* starts, int64_t first, uint32_t bits, Place place, Add add) {
    if (starts == nullptr) {
        const int32_t n = __reduce_add_sync(0xffffffffu, __popc(bits));
        if ((threadIdx.x & 31) == 0 && n > 0) add(0, n);
        return;
    }
    // ordinarily the whole warp is in one sequence
    const bool one = place.holds(starts, first) && first + kEach <= place.end;
    if (__all_sync(0xffffffffu, one) && __match_any_sync(0xffffffffu, place.b) == 0xffffffffu) {
        const int32_t n = __reduce_add_sync(0xffffffffu, __popc(bits));
        if ((threadIdx.x & 31) == 0 && n > 0) add(place.b, n);
        return;
    }
    for (int i = 0; i < kEach; ++i) {
        if (!(bits >> i & 1)) continue;
        place.go(starts, p.seqs, first + i);
        if (place.holds(starts, first + i)) add(place.b, 1);
    }
}

__device__ __forceinline__ double sum_over_warp(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// The CTA's sums, in its first thread.
__device__ __forceinline__ Sums sum_over_cta(Sums s, Sums* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    s.loss = sum_over_warp(s.loss);
    s.kl = sum_over_warp(s.kl);
    s.clipped = sum_over_warp(s.clipped);
    if (warps == 1) return s;
    __syncthreads();
    if (lane == 0) scratch[warp] = s;
    __syncthreads();
    if (warp != 0) return s;
    s = lane < warps ? scratch[lane] : Sums{};
    s.loss = sum_over_warp(s.loss);
    s.kl = sum_over_warp(s.kl);
    s.clipped = sum_over_warp(s.clipped);
    return s;
}

__device__ __forceinline__ double weight_of(int32_t n, int32_t sequences) { return n > 0 ? 1.0 / (static_cast<double>(n) * static_cast<double>(sequences)) : 0.0; }

__device__ __forceinline__ void results(const PolicyParams& p, const Sums& s) {
    p.results[0] = static_cast<float>(s.loss);
    p.results[1] = static_cast<float>(s.kl);
    p.results[2] = static_cast<float>(s.clipped);
}

__device__ __forceinline__ void check_starts(const PolicyParams& p, int32_t b) {
    const int32_t first = p.starts[b], end = p.starts[b + 1];
    if (first < 0 || end < first || end > p.tokens) kv_report(MHLO_CUDA_KV_ERROR_STARTS);
}

// Everything in one CTA.
__global__ void __launch_bounds__(kSmallThreads) policy_small_kernel(const __grid_constant__ PolicyParams p) {
    __shared__ int32_t counts[kSmallSeqs], starts[kSmallSeqs + 1], sequences;
    __shared__ Sums scratch[32];
    const int tid = threadIdx.x, threads = blockDim.x;
    const int32_t n = p.starts != nullptr ? p.seqs : 1;
    grid_dependency_wait();
    grid_dependency_release();
    Tokens ahead;  // the first ones of this thread
    const uint32_t ahead_bits = counted(p, tid * kEach);
    if (tid * kEach < p.tokens) ahead.load(p, tid * kEach);
    for (int32_t i = tid; i < n; i += threads) {
        counts[i] = 0;
        if (p.starts != nullptr) {
            starts[i] = p.starts[i];
            check_starts(p, i);
        }
    }
    if (tid == 0) {
        sequences = 0;
        if (p.starts != nullptr) starts[n] = p.starts[n];
    }
    __syncthreads();
    const int32_t* const from = p.starts != nullptr ? starts : nullptr;
    const int64_t all = (p.tokens + 32 * kEach - 1) / (32 * kEach) * (32 * kEach);  // warps stay whole
    for (int64_t first = tid * kEach; first < all; first += threads * kEach) {
        Place place{0, 0};
        if (from != nullptr) place.find(from, p.seqs, first - (tid & 31) * kEach, first);
        count(p, from, first, first == tid * kEach ? ahead_bits : counted(p, first), place, [&](int32_t b, int32_t k) { atomicAdd(&counts[b], k); });
    }
    __syncthreads();
    int32_t some = 0;
    for (int32_t i = tid; i < n; i += threads) some += counts[i] > 0;
    some = __reduce_add_sync(0xffffffffu, some);
    if ((tid & 31) == 0 && some > 0) atomicAdd(&sequences, some);
    __syncthreads();
    Sums sums;
    for (int64_t first = tid * kEach; first < all; first += threads * kEach) {
        Place place{0, 0};
        if (from != nullptr) place.find(from, p.seqs, first - (tid & 31) * kEach, first);
        uint32_t bits = ahead_bits;
        if (first != tid * kEach) {
            bits = counted(p, first);
            if (bits != 0) ahead.load(p, first);
        }
        step(p, from, first, bits, ahead, place, &sums, [&](int32_t b) { return weight_of(counts[b], sequences); });
    }
    sums = sum_over_cta(sums, scratch);
    if (tid == 0) results(p, sums);
}

// Whether this CTA is the last one to get here; what the others wrote before is then there.
__device__ __forceinline__ bool last_cta(int32_t* ticket) {
    __shared__ bool last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(ticket, 1) == static_cast<int32_t>(gridDim.x) - 1;
    __syncthreads();
    if (last) __threadfence();
    return last;
}

constexpr int64_t kOfCta = kThreads * kEach;

__global__ void __launch_bounds__(kThreads) policy_count_kernel(const __grid_constant__ PolicyParams p) {
    __shared__ int32_t sequences;
    const int tid = threadIdx.x;
    const int32_t n = p.seqs;
    grid_dependency_release();
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * kThreads + tid; b < p.seqs; b += static_cast<int64_t>(gridDim.x) * kThreads) check_starts(p, static_cast<int32_t>(b));
    for (int64_t base = blockIdx.x * kOfCta; base < p.tokens; base += gridDim.x * kOfCta) {
        const int64_t first = base + tid * kEach;
        Place place;
        place.find(p.starts, p.seqs, first - (tid & 31) * kEach, first);
        count(p, p.starts, first, counted(p, first), place, [&](int32_t b, int32_t k) { atomicAdd(&p.counts[b], k); });
    }
    if (tid == 0) sequences = 0;
    if (!last_cta(p.counts + n + 1)) return;
    int32_t some = 0;
    for (int32_t i = tid; i < n; i += kThreads) some += __ldcg(p.counts + i) > 0;
    some = __reduce_add_sync(0xffffffffu, some);
    if ((tid & 31) == 0 && some > 0) atomicAdd(&sequences, some);
    __syncthreads();
    if (tid == 0) p.counts[n] = sequences;
}

// Without sequences: a count a CTA, which the next launch adds up. (An atomic addition a warp, all to one word, took 9 us for a million tokens.)
__global__ void __launch_bounds__(kThreads) policy_count_all_kernel(const __grid_constant__ PolicyParams p, int32_t wide) {
    __shared__ int32_t sums[kThreads / 32];
    const int tid = threadIdx.x, step = gridDim.x * kThreads;
    grid_dependency_release();
    int32_t mine = 0;
    if (p.mask == nullptr) {
        mine = blockIdx.x == 0 && tid == 0 ? static_cast<int32_t>(p.tokens) : 0;
    } else {
        const int64_t vectors = wide ? p.tokens / 16 : 0;
        const uint4* const v = reinterpret_cast<const uint4*>(p.mask);
#pragma unroll 4
        for (int64_t i = blockIdx.x * kThreads + tid; i < vectors; i += step) {
            const uint4 m = v[i];
            mine += __popc(__vcmpne4(m.x, 0)) + __popc(__vcmpne4(m.y, 0)) + __popc(__vcmpne4(m.z, 0)) + __popc(__vcmpne4(m.w, 0));
        }
        mine >>= 3;
        for (int64_t i = vectors * 16 + blockIdx.x * kThreads + tid; i < p.tokens; i += step) mine += p.mask[i] != 0;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if ((tid & 31) == 0) sums[tid >> 5] = mine;
    __syncthreads();
    if (tid != 0) return;
    for (int w = 1; w < kThreads / 32; ++w) mine += sums[w];
    p.counts[blockIdx.x] = mine;
    if (blockIdx.x == 0) p.counts[p.counters] = 0;  // the next launch's ticket
}

// The tokens' values do not wait for the counts: everything in front of the launch that counts is done when this one begins.
__global__ void __launch_bounds__(kThreads) policy_loss_kernel(const __grid_constant__ PolicyParams p) {
    __shared__ Sums scratch[32];
    __shared__ int32_t all;
    const int tid = threadIdx.x;
    Sums sums;
    bool waited = false;
    int32_t sequences = 1;
    auto wait = [&]() {
        grid_dependency_wait();
        grid_dependency_release();
        if (p.starts != nullptr) {
            sequences = __ldcg(p.counts + p.seqs);
        } else {
            if (tid < 32) {
                int32_t mine = 0;
                for (int32_t i = tid; i < p.counters; i += 32) mine += __ldcg(p.counts + i);
                mine = __reduce_add_sync(0xffffffffu, mine);
                if (tid == 0) all = mine;
            }
            __syncthreads();
        }
        waited = true;
    };
    for (int64_t base = blockIdx.x * kOfCta; base < p.tokens; base += gridDim.x * kOfCta) {
        const int64_t first = base + tid * kEach;
        Tokens t;
        const uint32_t bits = counted(p, first);
        if (first < p.tokens) t.load(p, first);
        Place place{0, 0};
        if (p.starts != nullptr) place.find(p.starts, p.seqs, first - (tid & 31) * kEach, first);
        if (!waited) wait();
        step(p, p.starts, first, bits, t, place, &sums, [&](int32_t b) { return p.starts != nullptr ? weight_of(__ldcg(p.counts + b), sequences) : weight_of(all, 1); });
    }
    if (!waited) wait();
    sums = sum_over_cta(sums, scratch);
    if (tid == 0) {
        double* const to = p.partial + static_cast<int64_t>(blockIdx.x) * 3;
        to[0] = sums.loss, to[1] = sums.kl, to[2] = sums.clipped;
    }
    if (!last_cta(p.counts + (p.starts != nullptr ? p.seqs + 2 : p.counters))) return;
    Sums mine;
    for (int32_t i = tid; i < static_cast<int32_t>(gridDim.x); i += kThreads) mine.add({__ldcg(p.partial + i * 3), __ldcg(p.partial + i * 3 + 1), __ldcg(p.partial + i * 3 + 2)});
    mine = sum_over_cta(mine, scratch);
    if (tid == 0) results(p, mine);
}

constexpr int64_t kMostCtas = 4 * kNumSMs;

int64_t counts_bytes(int64_t seqs) { return ((std::max<int64_t>(seqs, kNumSMs) + 3) * 4 + 15) / 16 * 16; }
int64_t scratch_bytes(int64_t tokens, int64_t seqs) { return tokens <= kSmall && seqs <= kSmallSeqs ? 0 : counts_bytes(seqs) + kMostCtas * 24; }

}  // namespace

int policy_loss_device_error() { return take_kv_error(); }

}  // namespace mhlo

using namespace mhlo;

extern "C" {

int64_t mhlo_cuda_policy_loss_scratch_bytes(int64_t tokens, int64_t seqs) {
    return tokens < 0 || tokens > (1 << 30) || seqs < 0 || seqs > (1 << 24) ? 0 : scratch_bytes(tokens, seqs);
}

int mhlo_cuda_policy_loss(const mhlo_cuda_policy_batch* batch, float* grad_dev, float* results_dev, void* scratch_dev, int64_t bytes, mhlo_cuda_stream_t stream) {
    static const char* const what = "policy_loss";
    if (!batch) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null batch", what);
    const mhlo_cuda_policy_batch& b = *batch;
    if (b.tokens < 0 || b.tokens > (1 << 30) || b.seqs < 0 || b.seqs > (1 << 24))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld tokens, %lld sequences", what, static_cast<long long>(b.tokens), static_cast<long long>(b.seqs));
    if (!(b.clip_low >= 0.0 && b.clip_low < 1.0) || !(b.clip_high >= 0.0) || b.clip_high > 1e30)
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: clipped at 1 - %g and 1 + %g", what, b.clip_low, b.clip_high);
    if (!(std::fabs(b.kl_weight) <= 1e30) || (b.tokens > 0 && b.kl_weight != 0.0 && !b.ref_logprobs)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: KL weight %g%s", what, b.kl_weight, b.ref_logprobs ? "" : " without ref_logprobs");
    if (!results_dev) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null results", what);
    if (b.tokens > 0 && (!b.logprobs || !b.old_logprobs || !b.advantages || !grad_dev)) return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: null logprobs, old_logprobs, advantages or grad", what);
    const int64_t need = scratch_bytes(b.tokens, b.seqs);
    if (need > 0 && (!scratch_dev || !aligned16(scratch_dev) || bytes < need))
        return fail(MHLO_CUDA_INVALID_ARGUMENT, "%s: %lld bytes of scratch, %lld needed, on 16 bytes", what, static_cast<long long>(bytes), static_cast<long long>(need));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    PolicyParams p;
    p.logprobs = b.logprobs, p.old_logprobs = b.old_logprobs, p.ref = b.ref_logprobs, p.advantages = b.advantages;
    p.mask = b.mask;
    p.starts = b.starts;
    p.grad = grad_dev;
    p.results = results_dev;
    p.tokens = b.tokens;
    p.seqs = static_cast<int32_t>(b.seqs);
    p.low = std::log1p(-b.clip_low);
    p.high = std::log1p(b.clip_high);
    p.border_low = static_cast<float>(1.0 - b.clip_low);
    p.border_high = static_cast<float>(1.0 + b.clip_high);
    p.kl_weight = static_cast<float>(b.kl_weight);
    p.vec = aligned16(b.logprobs) && aligned16(b.old_logprobs) && aligned16(b.ref_logprobs) && aligned16(b.advantages) && aligned16(grad_dev) &&
            (reinterpret_cast<uintptr_t>(b.mask) & 3) == 0;
    if (b.starts && b.seqs == 0) {  // no token is of any sequence
        if (b.tokens > 0) MHLO_CUDA_TRY(cudaMemsetAsync(grad_dev, 0, b.tokens * 4, s), MHLO_CUDA_EXECUTION_FAILED);
        MHLO_CUDA_TRY(cudaMemsetAsync(results_dev, 0, 12, s), MHLO_CUDA_EXECUTION_FAILED);
        return MHLO_CUDA_OK;
    }
    cudaError_t e;
    if (need == 0) {
        p.counts = nullptr;
        p.counters = 0;
        p.partial = nullptr;
        const int64_t threads = std::min<int64_t>(kSmallThreads, std::max<int64_t>(1, (b.tokens + 32 * kEach - 1) / (32 * kEach)) * 32);
        e = launch_dependent(policy_small_kernel, dim3(1), dim3(static_cast<unsigned>(threads)), 0, s, 1, true, p);
    } else {
        p.counts = static_cast<int32_t*>(scratch_dev);
        p.partial = reinterpret_cast<double*>(static_cast<char*>(scratch_dev) + counts_bytes(b.seqs));
        const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min((b.tokens + kOfCta - 1) / kOfCta, kMostCtas)));
        p.counters = static_cast<int32_t>(std::min<unsigned>(grid, kNumSMs));
        if (p.starts) {
            MHLO_CUDA_TRY(cudaMemsetAsync(p.counts, 0, (b.seqs + 3) * 4, s), MHLO_CUDA_EXECUTION_FAILED);
            policy_count_kernel<<<grid, kThreads, 0, s>>>(p);
        } else {
            policy_count_all_kernel<<<static_cast<unsigned>(p.counters), kThreads, 0, s>>>(p, aligned16(b.mask));
        }
        MHLO_CUDA_CHECK_LAUNCH(what);
        e = launch_dependent(policy_loss_kernel, dim3(grid), dim3(kThreads), 0, s, 1, true, p);
    }
    if (e != cudaSuccess) return fail(MHLO_CUDA_EXECUTION_FAILED, "launch of %s failed: %s", what, cudaGetErrorString(e));
    MHLO_CUDA_CHECK_LAUNCH(what);
    return MHLO_CUDA_OK;
}

}  // extern "C"
