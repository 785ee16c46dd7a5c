// Sampling one token per row of logits from one given uniform number (sm_100a); semantics in include/kore_b200.h.
//
// Every filter keeps a prefix of the order (logit descending, index ascending).  As an unsigned 64-bit number that order
// is comp = ~ordered_bits(logit) << 32 | index, so the kept set is "comp <= bound" and a filter only lowers the bound.
// Weights are integers of 2^-44 (the largest is 2^44, 2^19 of them fit 63 bits): their sums do not depend on the order in
// which atomics arrive, and a token's border moves by at most vocab 2^-45 of the largest weight.
//
// Bound by the latency of the passes for a few rows and by the f64 exponentials for many (a logit is read once).  A row
// belongs to a cluster of 1 to 8 CTAs, each with a slice of it in shared memory.  Top-k and top-p look for the element at
// which a running measure (count, or weight) reaches a target: a histogram over 1024 steps of 1/32 in the exponent gives
// the bin, the candidates of that bin (a few dozen of 32000 normal logits) are collected, sorted and summed by every CTA
// alike.  A bin of more than SAMPLE_CAND candidates (ties, flat rows) is cut into 1024 parts of the order first, again and
// again.  The draw sums the kept weights by segment and walks the one that holds the number.
#include <math.h>
#include <stdlib.h>

#include "common.cuh"
#include "device_utils.cuh"
#include "tc_ptx.cuh"

namespace kb {

using u64 = unsigned long long;

constexpr int SAMPLE_THREADS = 512;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int SAMPLE_BINS = 1024;
constexpr int SAMPLE_CAND = 2048;
constexpr int SAMPLE_CTAS = 8;  // of a cluster, at most
constexpr int SAMPLE_SLICE = 40960;  // logits of a slice that shared memory holds (160 KB); a longer slice is read from L2
constexpr size_t SAMPLE_MAX_VOCAB = (size_t)1 << 19;

struct SampleParams {
    const float *logits;
    size_t ld;
    int vocab, slice;
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
    long long *tokens;
    float *logprobs;
};

struct SampleShared {
    u64 slot[8][SAMPLE_CTAS];  // one row per reduction over the cluster
    u64 scratch[SAMPLE_WARPS];
    uint32_t hist_lo[SAMPLE_BINS], hist_hi[SAMPLE_BINS];  // 64-bit sums in two words: 64-bit shared atomics are compare-and-swap loops
    u64 own[SAMPLE_CAND], all[SAMPLE_CAND];
    uint32_t n_own;
    int bin;
    u64 before, found;
};

__device__ __forceinline__ float clean(float l) { return l == l ? l : -INFINITY; }
// position in the order: smaller is earlier
__device__ __forceinline__ u64 comp_of(float l, int idx) {
    uint32_t b = __float_as_uint(l == 0.0f ? 0.0f : l);  // -0 and +0 are equal logits
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((u64)(~b) << 32) | (uint32_t)idx;
}
__device__ __forceinline__ float logit_of(u64 comp) {
    const uint32_t b = ~(uint32_t)(comp >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

// 2^44 2^y rounded to an integer, y <= 0: 2^f on [-1/2, 1/2] by its Taylor series to the 11th power (the next term is below
// 7e-15, 2^-47), times 2^n by the exponent field, rounded by adding 2^52
__device__ __forceinline__ u64 exp2_fixed(double y) {
    if (!(y > -46.0)) return 0ull;
    const double shift = 0x1.8p52, n = y + shift, f = y - (n - shift);
    double r = 4.44553827187081162491e-10;  // ln(2)^k / k!, k = 11 .. 0
    r = fma(r, f, 7.05491162080112335899e-09);
    r = fma(r, f, 1.01780860092396999224e-07);
    r = fma(r, f, 1.32154867901443095086e-06);
    r = fma(r, f, 1.52527338040598410828e-05);
    r = fma(r, f, 1.54035303933816087761e-04);
    r = fma(r, f, 1.33335581464284432841e-03);
    r = fma(r, f, 9.61812910762847687873e-03);
    r = fma(r, f, 5.55041086648215831190e-02);
    r = fma(r, f, 2.40226506959100721827e-01);
    r = fma(r, f, 6.93147180559945286227e-01);
    r = fma(r, f, 1.0);
    const double v = __hiloint2double(__double2hiint(r) + ((__double2loint(n) + 44) << 20), __double2loint(r));
    return (u64)__double_as_longlong(v + 0x1p52) & ((1ull << 52) - 1);
}

__device__ __forceinline__ uint32_t ld_cluster(const uint32_t *p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(ptx::mapa(ptx::smem_u32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ u64 ld_cluster(const u64 *p, uint32_t rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(ptx::mapa(ptx::smem_u32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ void st_cluster(u64 *p, uint32_t rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ptx::mapa(ptx::smem_u32(p), rank)), "l"(v) : "memory");
}

struct Row {
    SampleShared &sh;
    const float *l;  // this CTA's slice: shared memory, or the logits themselves
    int n, i0;       // its length and its first index
    uint32_t rank, ctas;
    float top;       // largest logit
    double per;      // log2(e) / temperature
    float bins;      // bins per unit of logit

    __device__ __forceinline__ u64 weight(float x) const {
        if (top == INFINITY) return x == top ? 1ull << 44 : 0ull;
        return exp2_fixed(((double)x - (double)top) * per);
    }
    __device__ __forceinline__ int bin_of(float x) const {  // falls with x
        return x == top ? 0 : (int)fminf((top - x) * bins, (float)(SAMPLE_BINS - 1));
    }

    template <typename F>
    __device__ __forceinline__ u64 block_reduce(u64 v, F f) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sh.scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        u64 r = sh.scratch[threadIdx.x % SAMPLE_WARPS];
#pragma unroll
        for (int o = SAMPLE_WARPS / 2; o > 0; o >>= 1) r = f(r, __shfl_xor_sync(0xffffffffu, r, o));
        return r;
    }
    // every CTA's value, then the join of all; `id` names a slot that no other reduction of the row still uses
    __device__ __forceinline__ void exchange(u64 v, int id) const {
        if (threadIdx.x < ctas) st_cluster(&sh.slot[id][rank], threadIdx.x, v);
        ptx::cluster_sync();
    }
    template <typename F>
    __device__ __forceinline__ u64 cluster_reduce(u64 v, int id, F f) const {
        exchange(block_reduce(v, f), id);
        u64 r = sh.slot[id][0];
        for (uint32_t c = 1; c < ctas; ++c) r = f(r, sh.slot[id][c]);
        return r;
    }
    // inclusive sum over the threads
    __device__ __forceinline__ u64 block_scan(u64 v, u64 &total) const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 up = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += up;
        }
        __syncthreads();
        if (lane == 31) sh.scratch[warp] = v;
        __syncthreads();
        total = 0;
        u64 base = 0;
#pragma unroll
        for (int w = 0; w < SAMPLE_WARPS; ++w) {
            if (w == warp) base = total;
            total += sh.scratch[w];
        }
        return v + base;
    }
    __device__ __forceinline__ void hist_add(int b, u64 m) const {
        const uint32_t old = atomicAdd(sh.hist_lo + b, (uint32_t)m);
        const uint32_t hi = (uint32_t)(m >> 32) + (old + (uint32_t)m < old ? 1u : 0u);
        if (hi) atomicAdd(sh.hist_hi + b, hi);
    }

    // The element (its comp) at which the measure of the elements kept by `bound`, added up in order, reaches
    // target(measure of all); WEIGHT: measure = weight, otherwise 1.  Where that is a matter of weights of 0: ~0.
    template <bool WEIGHT, typename T>
    __device__ u64 reach(u64 bound, T target_of) const {
        u64 lo = 0, hi = ~0ull, target = 0;
        int shift = 0;
        for (int level = 0;; ++level) {
            for (int b = threadIdx.x; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.hist_lo[b] = sh.hist_hi[b] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i - (int)threadIdx.x < n; i += SAMPLE_THREADS) {  // whole warps
                const float x = i < n ? clean(l[i]) : 0.0f;
                const u64 c = comp_of(x, i0 + i);
                const bool in = i < n && c <= bound && c >= lo && c <= hi;
                const u64 m = !in ? 0ull : (WEIGHT ? weight(x) : 1ull);
                const int b = !m ? -1 : (level == 0 ? bin_of(x) : (int)((c - lo) >> shift));
                const int b0 = __shfl_sync(0xffffffffu, b, 0);
                if (b0 >= 0 && __all_sync(0xffffffffu, b == b0)) {  // ties and flat rows: one addition for the warp
                    u64 sum = m;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if ((threadIdx.x & 31) == 0) hist_add(b0, sum);
                } else if (b >= 0) {
                    hist_add(b, m);
                }
            }
            ptx::cluster_sync();
            // thread t: bins 2t and 2t + 1 of the whole row
            u64 mine[2] = {};
            for (uint32_t c = 0; c < ctas; ++c)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    mine[k] += (u64)ld_cluster(sh.hist_hi + 2 * threadIdx.x + k, c) << 32 | ld_cluster(sh.hist_lo + 2 * threadIdx.x + k, c);
            u64 total;
            u64 upto = block_scan(mine[0] + mine[1], total);
            if (level == 0) target = target_of(total);
            if (threadIdx.x == 0) sh.n_own = 0;
#pragma unroll
            for (int k = 1; k >= 0; --k) {
                if (upto - mine[k] < target && target <= upto) {
                    sh.bin = 2 * threadIdx.x + k;
                    sh.before = upto - mine[k];
                }
                upto -= mine[k];
            }
            __syncthreads();
            const int bin = sh.bin;
            target -= sh.before;
            if (!WEIGHT && level == 0 && bin == SAMPLE_BINS - 1) {  // from 31.9 on in the exponent weights are 0: who is kept does not matter
                ptx::cluster_sync();  // the histograms have been read
                return ~0ull;
            }
            if (level > 0) {
                lo += (u64)bin << shift;
                hi = min(hi, lo + ((1ull << shift) - 1));
            }
            u64 first = ~0ull, last = ~0ull;
            for (int i = threadIdx.x; i < n; i += SAMPLE_THREADS) {
                const float x = clean(l[i]);
                const u64 c = comp_of(x, i0 + i);
                if (c <= bound && c >= lo && c <= hi && (level > 0 || bin_of(x) == bin)) {
                    const uint32_t at = atomicAdd(&sh.n_own, 1u);
                    if (at < SAMPLE_CAND) sh.own[at] = c;
                    first = min(first, c);
                    last = min(last, ~c);
                }
            }
            ptx::cluster_sync();
            uint32_t count = 0;
            for (uint32_t c = 0; c < ctas; ++c) {
                const uint32_t m = ld_cluster(&sh.n_own, c);
                if (count + m <= SAMPLE_CAND)
                    for (uint32_t i = threadIdx.x; i < m; i += SAMPLE_THREADS) sh.all[count + i] = ld_cluster(sh.own + i, c);
                count = count + m <= SAMPLE_CAND ? count + m : SAMPLE_CAND + 1;
            }
            if (count <= SAMPLE_CAND) return pick<WEIGHT>(count, target);
            // too many: the part of the order that they span, cut into bins
            const auto least = [](u64 a, u64 b) { return a < b ? a : b; };
            lo = cluster_reduce(first, 4 + 2 * (level & 1), least);
            hi = ~cluster_reduce(last, 5 + 2 * (level & 1), least);
            shift = max(0, 64 - __clzll((long long)(hi - lo)) - 10);
        }
    }
    // of the candidates in sh.all the one at which their measure, added up in order, reaches target
    template <bool WEIGHT>
    __device__ u64 pick(uint32_t count, u64 target) const {
        uint32_t size = 2;
        while (size < count) size *= 2;
        for (uint32_t i = count + threadIdx.x; i < size; i += SAMPLE_THREADS) sh.all[i] = ~0ull;
        __syncthreads();
        for (uint32_t k = 2; k <= size; k *= 2)  // bitonic sort
            for (uint32_t j = k / 2; j > 0; j /= 2) {
                for (uint32_t p = threadIdx.x; p < size / 2; p += SAMPLE_THREADS) {
                    const uint32_t a = 2 * p - (p & (j - 1)), b = a + j;
                    const u64 x = sh.all[a], y = sh.all[b];
                    if ((x > y) == ((a & k) == 0)) {
                        sh.all[a] = y;
                        sh.all[b] = x;
                    }
                }
                __syncthreads();
            }
        constexpr int PER = SAMPLE_CAND / SAMPLE_THREADS;
        u64 m[PER], mine = 0, total;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const uint32_t i = PER * threadIdx.x + k;
            m[k] = i < count ? (WEIGHT ? weight(logit_of(sh.all[i])) : 1ull) : 0ull;
            mine += m[k];
        }
        u64 upto = block_scan(mine, total) - mine;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            if (upto < target && target <= upto + m[k]) sh.found = sh.all[PER * threadIdx.x + k];
            upto += m[k];
        }
        __syncthreads();
        return sh.found;
    }
};

__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    uint32_t ctas;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t r = blockIdx.x / ctas;
    Row row = {sh, nullptr, 0, 0, ptx::cluster_ctarank(), ctas, 0.0f, 0.0, 0.0f};
    row.i0 = min(p.vocab, (int)row.rank * p.slice);
    row.n = min(p.slice, p.vocab - row.i0);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const float *src = p.logits + r * p.ld + row.i0;
    float *held = reinterpret_cast<float *>(smem + (sizeof(SampleShared) + 15) / 16 * 16);
    const bool hold = p.slice <= SAMPLE_SLICE;
    row.l = hold ? held : src;
    u64 best = ~0ull;
    if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        for (int i = threadIdx.x; i < row.n / 4; i += SAMPLE_THREADS) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(src) + i);
            if (hold) reinterpret_cast<float4 *>(held)[i] = v;
            best = min(min(best, min(comp_of(clean(v.x), row.i0 + 4 * i), comp_of(clean(v.y), row.i0 + 4 * i + 1))),
                       min(comp_of(clean(v.z), row.i0 + 4 * i + 2), comp_of(clean(v.w), row.i0 + 4 * i + 3)));
        }
        for (int i = (row.n & ~3) + threadIdx.x; i < row.n; i += SAMPLE_THREADS) {
            const float v = __ldcg(src + i);
            if (hold) held[i] = v;
            best = min(best, comp_of(clean(v), row.i0 + i));
        }
    } else {
        for (int i = threadIdx.x; i < row.n; i += SAMPLE_THREADS) {
            const float v = __ldcg(src + i);
            if (hold) held[i] = v;
            best = min(best, comp_of(clean(v), row.i0 + i));
        }
    }
    const auto least = [](u64 a, u64 b) { return a < b ? a : b; };
    best = row.cluster_reduce(best, 0, least);
    row.top = logit_of(best);
    const float temp = p.temperature ? p.temperature[r] : 1.0f;
    if (row.top == -INFINITY || !(temp > 0.0f)) {
        if (row.rank == 0 && threadIdx.x == 0) {
            p.tokens[r] = row.top == -INFINITY ? 0 : (long long)(uint32_t)best;
            if (p.logprobs) p.logprobs[r] = row.top == -INFINITY ? __uint_as_float(0x7fffffffu) : 0.0f;
        }
        return;
    }
    const double inv_t = 1.0 / (double)temp;
    row.per = inv_t * 1.4426950408889634074;
    row.bins = (float)(inv_t * (SAMPLE_BINS / 32));
    u64 bound = ~0ull;
    const int k = p.top_k ? p.top_k[r] : 0;
    if (k > 0 && k < p.vocab) bound = row.reach<false>(bound, [&](u64) { return (u64)k; });
    const float mp = p.min_p ? p.min_p[r] : 0.0f;
    if (mp > 0.0f) {
        const double border = log((double)fminf(mp, 1.0f));
        u64 out = ~0ull;  // the first element below the border
        for (int i = threadIdx.x; i < row.n; i += SAMPLE_THREADS) {
            const float x = clean(row.l[i]);
            if (x != row.top && !(((double)x - (double)row.top) * inv_t >= border)) out = min(out, comp_of(x, row.i0 + i));
        }
        out = row.cluster_reduce(out, 1, least);
        if (out != ~0ull) bound = min(bound, out - 1);
    }
    const float tp = p.top_p ? p.top_p[r] : 1.0f;
    if (tp < 1.0f)
        bound = row.reach<true>(bound, [&](u64 z) { return min(max((u64)ceil((double)fmaxf(tp, 0.0f) * (double)z), 1ull), z); });
    // ---- the draw: warps sum contiguous segments, the segment that holds the number is walked in index order
    const int seg = (row.n + SAMPLE_WARPS - 1) / SAMPLE_WARPS, s0 = min(row.n, warp * seg), s1 = min(row.n, s0 + seg);
    auto kept = [&](int i) {
        const float x = clean(row.l[i]);
        return comp_of(x, row.i0 + i) <= bound ? row.weight(x) : 0ull;
    };
    u64 s = 0;
    for (int i = s0 + lane; i < s1; i += 32) s += kept(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if (lane == 0) sh.scratch[warp] = s;
    __syncthreads();
    u64 before = 0, mine = 0, z = 0;
    for (int w = 0; w < SAMPLE_WARPS; ++w) {
        if (w < warp) before += sh.scratch[w];
        mine += sh.scratch[w];
    }
    row.exchange(mine, 2);  // nothing of another CTA is read from here on
    for (uint32_t c = 0; c < ctas; ++c) {
        if (c < row.rank) before += sh.slot[2][c];
        z += sh.slot[2][c];
    }
    const float u = p.u[r];
    u64 draw = u > 0.0f ? (u64)((double)fminf(u, 1.0f) * (double)z) : 0ull;
    draw = min(draw, z - 1);
    if (draw < before || draw >= before + s) return;  // one warp of the cluster goes on
    for (int i = s0; i < s1; i += 32) {
        const u64 w = i + lane < s1 ? kept(i + lane) : 0ull;
        u64 inc = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
        }
        const u64 all = __shfl_sync(0xffffffffu, inc, 31);
        if (draw < before + all) {
            if (draw >= before + inc - w && draw < before + inc) {
                p.tokens[r] = row.i0 + i + lane;
                if (p.logprobs) {
                    const float x = clean(row.l[i + lane]);
                    const double e = x == row.top ? 0.0 : ((double)x - (double)row.top) * inv_t;
                    p.logprobs[r] = (float)(e - log((double)z * 0x1p-44));
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
    if (n > 0x7fffffffu / SAMPLE_CTAS) return fail(KB_ERR_UNSUPPORTED, "sample: %zu rows", n);
    int dev = 0;
    KB_CUDA(cudaGetDevice(&dev));
    // CTAs per row: all eight for the few rows that leave SMs idle, otherwise slices of up to 16384 logits; at least 1024 each
    const size_t per = n * SAMPLE_CTAS <= (size_t)sm_count(dev) * 2 ? 1024 : 16384;
    int ctas = 1;
    while (ctas < SAMPLE_CTAS && vocab > per * ctas) ctas *= 2;
    const int slice = (int)(((vocab + ctas - 1) / ctas + 3) / 4 * 4);
    SampleParams p = {logits, ld, (int)vocab, slice, temperature, top_k, top_p, min_p, u, tokens, logprobs};
    const size_t fixed = (sizeof(SampleShared) + 15) / 16 * 16;
    const size_t smem = fixed + (slice <= SAMPLE_SLICE ? (size_t)slice * 4 : 0);
    if (int rc = set_dyn_smem_once(reinterpret_cast<const void *>(sample_kernel), dev, (int)(fixed + SAMPLE_SLICE * 4), "sample smem attribute")) return rc;
    static const bool pdl = [] { const char *v = getenv("KB_GEMV_PDL"); return !(v && *v == '0'); }();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n * ctas));
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, p);
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "sample launch");
}
