// Sampling one token per row of logits from one given uniform number (sm_100a); semantics in include/kore_b200.h.
//
// Every filter keeps a prefix of the order (logit descending, index ascending).  As an unsigned 64-bit number that order
// is comp = ~ordered_bits(logit) << 32 | index, so the kept set is "comp <= bound" and a filter only lowers the bound.
// Top-k and top-p find the element at which a running measure (count, or weight) reaches a target by radix descent: a
// histogram of the measure over 1024 bins of the order, the bin that the target falls into, and so on inside that bin.
// Weights are integers of 2^-44 (the largest is 2^44, 2^19 of them fit 63 bits), so their sums do not depend on the order
// in which atomics arrive, and 44 bits are enough that a token's border moves by less than 2^-44 * vocab of the total.
#include <math.h>

#include "common.cuh"
#include "device_utils.cuh"

namespace kb {

using u64 = unsigned long long;

constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_BINS = 1024;
constexpr size_t SAMPLE_MAX_VOCAB = (size_t)1 << 19;

struct SampleParams {
    const float *logits;
    size_t ld;
    int vocab;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
    long long *tokens;
    float *logprobs;
};

__device__ __forceinline__ float clean(float l) { return l == l ? l : -INFINITY; }
// position in the order: smaller is earlier
__device__ __forceinline__ u64 comp_of(float l, int idx) {
    uint32_t b = __float_as_uint(l == 0.0f ? 0.0f : l);  // -0 and +0 are equal logits
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((u64)(~b) << 32) | (uint32_t)idx;
}

struct Row {
    const float *l;
    int vocab;
    float top;  // largest logit
    double inv_t;
    __device__ __forceinline__ u64 weight(float x) const {
        if (x == top) return 1ull << 44;
        if (x == -INFINITY || top == INFINITY) return 0ull;
        return __double2ull_rn(exp(((double)x - (double)top) * inv_t) * 0x1p44);
    }
};

__device__ __forceinline__ u64 block_sum(u64 v, u64 *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    u64 r = scratch[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
    return r;
}
__device__ __forceinline__ u64 block_min(u64 v, u64 *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, o));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    u64 r = scratch[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r = min(r, __shfl_xor_sync(0xffffffffu, r, o));
    return r;
}

// The element (its comp) at which the measure of the elements kept by `bound`, added up in order, reaches `target`
// (1 <= target <= the measure of all of them).  WEIGHT: measure = weight, otherwise 1.
template <bool WEIGHT>
__device__ u64 reach(const Row &row, u64 bound, u64 target, u64 *hist, u64 *scratch) {
    __shared__ u64 s_before;
    __shared__ int s_bin;
    u64 lo = 0, hi = bound;  // the element lies in [lo, hi]
    for (int level = 0;; ++level) {
        // tighten to the elements that are there, then cut into bins of 2^shift
        u64 first = ~0ull, last = ~0ull;
        for (int i = threadIdx.x; i < row.vocab; i += SAMPLE_THREADS) {
            const u64 c = comp_of(clean(row.l[i]), i);
            if (c >= lo && c <= hi) {
                first = min(first, c);
                last = min(last, ~c);
            }
        }
        lo = block_min(first, scratch);
        hi = ~block_min(last, scratch);
        if (lo >= hi) return lo;
        const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 10);
        hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < row.vocab; i += SAMPLE_THREADS) {
            const float l = clean(row.l[i]);
            const u64 c = comp_of(l, i);
            if (c >= lo && c <= hi) atomicAdd(hist + ((c - lo) >> shift), WEIGHT ? row.weight(l) : 1ull);
        }
        __syncthreads();
        // running sum over the bins: thread = bin
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const u64 mine = hist[threadIdx.x];
        u64 inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 31) scratch[warp] = inc;
        __syncthreads();
        u64 base = 0;
        for (int wq = 0; wq < warp; ++wq) base += scratch[wq];
        inc += base;
        if (inc - mine < target && target <= inc) {
            s_bin = threadIdx.x;
            s_before = inc - mine;
        }
        __syncthreads();
        target -= s_before;
        lo += (u64)s_bin << shift;
        hi = min(hi, lo + ((1ull << shift) - 1));
        __syncthreads();
    }
}

__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(SampleParams p) {
    __shared__ u64 hist[SAMPLE_BINS], scratch[32];
    const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Row row;
    row.l = p.logits + (size_t)r * p.ld;
    row.vocab = p.vocab;
    u64 best = ~0ull;
    for (int i = threadIdx.x; i < row.vocab; i += SAMPLE_THREADS) best = min(best, comp_of(clean(row.l[i]), i));
    best = block_min(best, scratch);
    const int best_idx = (int)(uint32_t)best;
    row.top = clean(row.l[best_idx]);
    const float temp = p.temperature ? p.temperature[r] : 1.0f;
    if (row.top == -INFINITY || !(temp > 0.0f)) {
        if (threadIdx.x == 0) {
            p.tokens[r] = row.top == -INFINITY ? 0 : best_idx;
            if (p.logprobs) p.logprobs[r] = row.top == -INFINITY ? __uint_as_float(0x7fffffffu) : 0.0f;
        }
        return;
    }
    row.inv_t = 1.0 / (double)temp;
    u64 bound = ~0ull;
    const int k = p.top_k ? p.top_k[r] : 0;
    if (k > 0 && k < row.vocab) bound = reach<false>(row, bound, (u64)k, hist, scratch);
    const float mp = p.min_p ? p.min_p[r] : 0.0f;
    if (mp > 0.0f) {
        const double least = log((double)fminf(mp, 1.0f));
        u64 out = ~0ull;  // the first element below the border
        for (int i = threadIdx.x; i < row.vocab; i += SAMPLE_THREADS) {
            const float l = clean(row.l[i]);
            if (l != row.top && !(((double)l - (double)row.top) * row.inv_t >= least)) out = min(out, comp_of(l, i));
        }
        out = block_min(out, scratch);
        if (out != ~0ull) bound = min(bound, out - 1);
    }
    auto total_of = [&](u64 bnd) {
        u64 s = 0;
        for (int i = threadIdx.x; i < row.vocab; i += SAMPLE_THREADS) {
            const float l = clean(row.l[i]);
            if (comp_of(l, i) <= bnd) s += row.weight(l);
        }
        return block_sum(s, scratch);
    };
    const float tp = p.top_p ? p.top_p[r] : 1.0f;
    if (tp < 1.0f) {
        const u64 z = total_of(bound);
        u64 target = (u64)ceil((double)fmaxf(tp, 0.0f) * (double)z);
        target = min(max(target, 1ull), z);
        bound = reach<true>(row, bound, target, hist, scratch);
    }
    // the draw: warps sum contiguous segments, the segment that holds the number is walked in index order
    const int seg = (row.vocab + 31) / 32, i0 = min(row.vocab, warp * seg), i1 = min(row.vocab, i0 + seg);
    auto kept = [&](int i) {
        const float l = clean(row.l[i]);
        return comp_of(l, i) <= bound ? row.weight(l) : 0ull;
    };
    u64 s = 0;
    for (int i = i0 + lane; i < i1; i += 32) s += kept(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if (lane == 0) scratch[warp] = s;
    __syncthreads();
    u64 before = 0, z = 0;
    for (int wq = 0; wq < 32; ++wq) {
        if (wq < warp) before += scratch[wq];
        z += scratch[wq];
    }
    const float u = p.u[r];
    u64 draw = u > 0.0f ? (u64)((double)fminf(u, 1.0f) * (double)z) : 0ull;
    draw = min(draw, z - 1);
    if (draw < before || draw >= before + s) return;  // one warp goes on
    for (int i = i0; i < i1; i += 32) {
        const u64 mine = i + lane < i1 ? kept(i + lane) : 0ull;
        u64 inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        const u64 all = __shfl_sync(0xffffffffu, inc, 31);
        if (draw < before + all) {
            if (draw >= before + inc - mine && draw < before + inc) {
                p.tokens[r] = i + lane;
                if (p.logprobs) {
                    const float l = clean(row.l[i + lane]);
                    const double x = l == row.top ? 0.0 : ((double)l - (double)row.top) * row.inv_t;
                    p.logprobs[r] = (float)(x - log((double)z * 0x1p-44));
                }
            }
            return;
        }
        before += all;
    }
}

}  // namespace kb

using namespace kb;

extern "C" int kb_sample(const float *logits, size_t n, size_t vocab, size_t ld, const float *temperature, const int *top_k,
                         const float *top_p, const float *min_p, const float *u, long long *tokens, float *logprobs, kb_stream stream) {
    if (!logits || !u || !tokens) return fail(KB_ERR_INVALID, "null pointer");
    if (vocab == 0) return fail(KB_ERR_INVALID, "sample: empty vocabulary");
    if (vocab > SAMPLE_MAX_VOCAB) return fail(KB_ERR_UNSUPPORTED, "sample: vocabulary of %zu (at most %zu)", vocab, SAMPLE_MAX_VOCAB);
    if (ld == 0) ld = vocab;
    if (ld < vocab) return fail(KB_ERR_INVALID, "sample: row stride %zu below the vocabulary %zu", ld, vocab);
    if (n == 0) return KB_OK;
    if (n > 0x7fffffffu) return fail(KB_ERR_UNSUPPORTED, "sample: %zu rows", n);
    SampleParams p = {logits, ld, (int)vocab, temperature, top_k, top_p, min_p, u, tokens, logprobs};
    sample_kernel<<<(unsigned)n, SAMPLE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "sample launch");
}
