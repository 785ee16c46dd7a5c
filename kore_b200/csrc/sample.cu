// Sampling one token per row of logits from one given uniform number (sm_100a); semantics in include/kore_b200.h.
//
// Every filter keeps a prefix of the order (logit descending, index ascending).  As an unsigned 64-bit number that order
// is comp = ~ordered_bits(logit) << 32 | index; the kept set is "a logit above x, or equal to it up to index i".
// Weights are integers of 2^-44 (the largest is 2^44, 2^19 of them fit 63 bits): their sums do not depend on the order in
// which atomics arrive, and a token's border moves by at most vocab 2^-45 of the largest weight.
//
// Bound by the latency of the passes and of the exchanges between CTAs (one row of 32000: 2.9 us greedy, 6.3 without filters,
// 9.1 with a top-k of 50, 13.0 with one of 1000, 13.4 to 15.4 with top-p), for many rows by how many clusters fit next to the f64 exponentials (13 f64 operations each): 128 rows
// of 131072 with unlike settings take 76 us, the logits alone 10 us.  A row belongs to a cluster of 1 to 8 CTAs; each has a
// slice of the row, in shared memory where it fits, otherwise in L2.  Top-k and top-p look for the element at which a running
// measure (count, or weight) reaches a target:
//   1. a histogram over 1024 steps of 1/32 in the exponent.  Counts are exact.  Of a weight only its share of its bin's
//      largest, in 16 bits, goes through an atomic (the sum of a bin is good to 2^-15), while threads add up the exact
//      total: the bins that may hold the border are then known, one or two of them;
//   2. their elements (a few dozen of 32000 normal logits) are collected and what lies before them is summed exactly.  While
//      there are more than SAMPLE_CAND of them (flat distributions), the part of the order that they span is cut into 1024
//      bins of exact 64-bit sums; where a CTA has more than SAMPLE_OWN of them (ties) by going over its logits again;
//   3. every CTA finds the element among the candidates by counting.
// Where all that is kept down to there is a short list (top-k, most nuclei), the whole of it is collected in step 2 and the
// first CTA does the rest, the draw included, on the list; the others are done.  Otherwise step 2 has the sums of the kept
// weights by segment already, and the CTA that holds the number walks the segment that does.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "device_utils.cuh"
#include "tc_ptx.cuh"

namespace kb {

using u64 = unsigned long long;

constexpr int SAMPLE_THREADS = 512;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int SAMPLE_BINS = 1024;
constexpr int SAMPLE_OWN = 1024;  // elements that a CTA collects
constexpr int SAMPLE_CAND = 256;  // of a list: counting what lies before each of c elements takes c^2 / 512 steps of a thread
constexpr int SAMPLE_CTAS = 8;    // of a cluster, at most
constexpr size_t SAMPLE_MAX_VOCAB = (size_t)1 << 19;

struct SampleParams {
    const float *logits;
    size_t ld;
    int vocab, slice;
    bool held;  // slices in shared memory
    const float *temperature;
    const int *top_k;
    const float *top_p, *min_p, *u;
    long long *tokens;
    float *logprobs;
};

struct SampleShared {
    u64 slot[8][SAMPLE_CTAS];  // one row per exchange between the CTAs
    u64 scratch[SAMPLE_WARPS], segment[SAMPLE_WARPS];
    double scale[32];               // see exp2_fixed
    uint32_t hist[2][SAMPLE_BINS];  // counts or shares; 64-bit sums take both (64-bit shared atomics are compare-and-swap loops)
    u64 own[SAMPLE_OWN], chosen[SAMPLE_CAND];  // collected by this CTA, and what is left of them in a part of the order
    __align__(16) u64 comp[SAMPLE_CAND];       // of the whole row, in order after sort_list
    u64 weight[SAMPLE_CAND];
    uint32_t n_own, n_chosen;
    int bin[2];
    u64 before, upto, found;
};
constexpr size_t SAMPLE_FIXED = (sizeof(SampleShared) + 15) / 16 * 16;

// NaN counts as -inf, -0 is +0
__device__ __forceinline__ float clean(float l) { return l == l ? l + 0.0f : -INFINITY; }
// position in the order of a clean logit: smaller is earlier
__device__ __forceinline__ u64 comp_of(float l, int idx) {
    uint32_t b = __float_as_uint(l);
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((u64)(~b) << 32) | (uint32_t)idx;
}
__device__ __forceinline__ float logit_of(u64 comp) {
    const uint32_t b = ~(uint32_t)(comp >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

// The bits of 2^52 + (2^44 2^y rounded to an integer), y <= 0; 2^52 + 0 where not `in`.  y = e + j / 32 + f: 2^f on [-1/64,
// 1/64] by its Taylor series to the 5th power (the next term is below 2.3e-15, 2^-48) times 2^(44 + e + j/32), which comes
// from the table entry scale[j] = 2^(44 + j/32) with j << 15 taken off its upper word: adding (32 e + j) << 15 puts e into the
// exponent field.  Adding 2^52 rounds.  No branch, so that several can be under way in a thread.
constexpr u64 FIXED_ZERO = 0x433ull << 52;
__device__ __forceinline__ u64 exp2_fixed(double y, bool in, const double *scale) {
    // below -64 (0 from -46 on) by the sign and exponent bits
    y = __hiloint2double(in && (uint32_t)__double2hiint(y) <= 0xc0500000u ? __double2hiint(y) : (int)0xc0500000u, __double2loint(y));
    const double shift = 0x1.8p47, n = y + shift, f = y - (n - shift);
    double r = 1.33335581464284434234e-03;  // ln(2)^k / k!, k = 5 .. 0
    r = fma(r, f, 9.61812910762847716198e-03);
    r = fma(r, f, 5.55041086648215799531e-02);
    r = fma(r, f, 2.40226506959100712334e-01);
    r = fma(r, f, 6.93147180559945309417e-01);
    r = fma(r, f, 1.0);
    const int k = __double2loint(n);
    const double s = scale[k & 31];
    return (u64)__double_as_longlong(r * __hiloint2double(__double2hiint(s) + (k << 15), __double2loint(s)) + 0x1p52);
}

__device__ __forceinline__ uint2 ld_cluster(const uint2 *p, uint32_t rank) {
    uint2 v;
    asm volatile("ld.shared::cluster.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(ptx::mapa(ptx::smem_u32(p), rank)) : "memory");
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
__device__ __forceinline__ u64 least(u64 a, u64 b) { return a < b ? a : b; }
__device__ __forceinline__ u64 plus(u64 a, u64 b) { return a + b; }
template <typename T>
__device__ __forceinline__ T warp_scan(T v) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T up = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += up;
    }
    return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// what the filters keep: logits above `least`, and those equal to it up to index `last`; never a logit of -inf
struct Kept {
    float least;
    int last;
    __device__ __forceinline__ bool operator()(float x, int i) const { return x > least || (x == least && i <= last); }
    __device__ __forceinline__ void cut(float l, int i) {
        if (l > least) least = l, last = i;
        else if (l == least) last = min(last, i);
    }
    __device__ __forceinline__ void cut(u64 comp) { cut(logit_of(comp), (int)(uint32_t)comp); }
};

struct Row {
    SampleShared &sh;
    const float *l;     // this CTA's slice: shared memory (clean, filled up with -inf), or the logits themselves
    bool held, wide;    // wide: the logits are 16-byte aligned
    int n, i0;          // its length and its first index
    int q0, q1;         // this warp's segment of it, in quads
    uint32_t rank, ctas;
    float top;          // largest logit, at most FLT_MAX
    double per;         // log2(e) / temperature
    float bins;         // bins per two units of logit

    // exponent of a kept logit; infinite logits are all that is kept where there are any
    __device__ __forceinline__ double exponent(float x) const { return ((double)fminf(x, FLT_MAX) - (double)top) * per; }
    __device__ __forceinline__ u64 weight(float x) const { return exp2_fixed(exponent(x), true, sh.scale) - FIXED_ZERO; }
    // place in the histogram, 0 .. 1023, falling with x; half the difference, which the ends of the type do not take to infinity
    __device__ __forceinline__ float bin_at(float x) const {
        return fminf(fmaf(-0.5f, fminf(x, FLT_MAX), 0.5f * top) * bins, (float)(SAMPLE_BINS - 1));
    }

    __device__ __forceinline__ void load4(int i, float (&x)[4]) const {
        if (held || (wide && 4 * i + 3 < n)) {
            const float4 v = reinterpret_cast<const float4 *>(l)[i];
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = 4 * i + k < n ? l[4 * i + k] : -INFINITY;
        }
        if (!held) {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = clean(x[k]);
        }
    }
    // f(four logits, index of the first) for the quads of this warp's segment, in index order; elements behind the slice are
    // -inf.  WHOLE: all lanes go around.
    template <bool WHOLE, typename F>
    __device__ __forceinline__ void each4(F f) const {
        const int lane = threadIdx.x & 31;
#pragma unroll 1
        for (int i = q0 + lane; WHOLE ? i - lane < q1 : i < q1; i += 32) {
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (!WHOLE || i < q1) load4(i, x);
            f(x, i0 + 4 * i);
        }
    }
    // sum of the weights of the four where `in`, all under way at once; nothing is done where the warp has none
    __device__ __forceinline__ u64 weigh(const float (&x)[4], const bool (&in)[4]) const {
        u64 sum = 0;
        if (__any_sync(__activemask(), in[0] || in[1] || in[2] || in[3])) {
#pragma unroll
            for (int k = 0; k < 4; ++k) sum += exp2_fixed(exponent(x[k]), in[k], sh.scale);
            sum -= 4 * FIXED_ZERO;
        }
        return sum;
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
    // this CTA's value into slot `id` of every CTA (visible behind the next cluster_sync); an id is written again only when a
    // cluster_sync lies between its last reading and that
    __device__ __forceinline__ void tell(u64 v, int id) const {
        if (threadIdx.x < ctas) st_cluster(&sh.slot[id][rank], threadIdx.x, v);
    }
    template <typename F>
    __device__ __forceinline__ u64 told(int id, F f) const {
        u64 r = sh.slot[id][0];
        for (uint32_t c = 1; c < ctas; ++c) r = f(r, sh.slot[id][c]);
        return r;
    }
    template <typename F>
    __device__ __forceinline__ u64 cluster_reduce(u64 v, int id, F f) const {
        tell(block_reduce(v, f), id);
        ptx::cluster_sync();
        return told(id, f);
    }
    // inclusive sums over the threads
    template <typename... T>
    __device__ __forceinline__ void block_scan(T &...v) const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        ((v = warp_scan(v)), ...);
        __syncthreads();
        int at = 0;
        if (lane == 31) ((reinterpret_cast<T *>(at++ ? sh.segment : sh.scratch)[warp] = v), ...);
        __syncthreads();
        at = 0;
        auto add = [&](auto &x) {
            using V = std::remove_reference_t<decltype(x)>;
            const V upto = warp_scan(reinterpret_cast<V *>(at++ ? sh.segment : sh.scratch)[lane % SAMPLE_WARPS]);
            const V base = __shfl_sync(0xffffffffu, upto, warp ? warp - 1 : 0);
            if (warp) x += base;
        };
        (add(v), ...);
    }
    __device__ __forceinline__ void hist_add64(int b, u64 m) const {
        if (b < 0) return;
        const uint32_t old = atomicAdd(sh.hist[0] + b, (uint32_t)m);
        const uint32_t hi = (uint32_t)(m >> 32) + (old + (uint32_t)m < old ? 1u : 0u);
        if (hi) atomicAdd(sh.hist[1] + b, hi);
    }
    __device__ __forceinline__ void hist_clear() const {
        for (int b = threadIdx.x; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.hist[0][b] = sh.hist[1][b] = 0;
        __syncthreads();
    }
    // bins 2t and 2t + 1 of word array h over the whole row
    __device__ __forceinline__ void hist_row(int h, u64 (&out)[2]) const {
        static_assert(SAMPLE_BINS == 2 * SAMPLE_THREADS, "two bins a thread");
        uint2 v[SAMPLE_CTAS];
#pragma unroll
        for (int c = 0; c < SAMPLE_CTAS; ++c)  // all loads under way before the first sum
            if (c < (int)ctas) v[c] = ld_cluster(reinterpret_cast<const uint2 *>(sh.hist[h]) + threadIdx.x, c);
        out[0] = out[1] = 0;
#pragma unroll
        for (int c = 0; c < SAMPLE_CTAS; ++c)
            if (c < (int)ctas) {
                out[0] += v[c].x;
                out[1] += v[c].y;
            }
    }
    // the bin in which the running sum reaches target, the sum before it and with it
    __device__ __forceinline__ void find_bin(const u64 (&mine)[2], u64 target) const {
        u64 upto = mine[0] + mine[1];
        block_scan(upto);
#pragma unroll
        for (int k = 1; k >= 0; --k) {
            if (upto - mine[k] < target && target <= upto) {
                sh.bin[0] = sh.bin[1] = 2 * threadIdx.x + k;
                sh.before = upto - mine[k];
                sh.upto = upto;
            }
            upto -= mine[k];
        }
    }
    __device__ __forceinline__ void collect(u64 c) const {
        const uint32_t slot = atomicAdd(&sh.n_own, 1u);
        if (slot < SAMPLE_OWN) sh.own[slot] = c;
    }
    // CTAs that collected more than they have room for
    __device__ __forceinline__ bool overflown(int id) const {
        bool over = false;
        for (uint32_t c = 0; c < ctas; ++c) over |= sh.slot[id][c] > SAMPLE_OWN;
        return over;
    }

    // Top-k for a k that is small against the number of threads: a histogram of the threads' own largest logits (mine_top) is
    // enough.  k of them lie in the bins up to some b, so the k largest of all do, and hardly more than k others with them.
    // Returns the length of the list, or 0 where it would be too long or the maxima too few.
    __device__ int cut_few(Kept &kept, float mine_top, int k) const {
        hist_clear();
        if (threadIdx.x == 0) sh.bin[1] = SAMPLE_BINS - 1;
        if (mine_top >= -FLT_MAX) atomicAdd(sh.hist[0] + (int)bin_at(mine_top), 1u);
        ptx::cluster_sync();
        u64 mine[2];
        hist_row(0, mine);
        find_bin(mine, (u64)k);
        if (threadIdx.x == 0) sh.n_own = 0;
        __syncthreads();
        const int b1 = sh.bin[1];
        if (b1 < SAMPLE_BINS - 1) {
            const float to = (float)(b1 + 1);
            each4<false>([&](const float (&x)[4], int i) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (bin_at(x[j]) < to && kept(x[j], i + j)) collect(comp_of(x[j], i + j));
            });
        }
        __syncthreads();
        tell(sh.n_own, 5);
        ptx::cluster_sync();
        const u64 count = told(5, plus);
        if (count == 0 || count > SAMPLE_CAND) return 0;
        if (take_list(sh.own, count)) cut_list<false>(kept, (uint32_t)count, (u64)k);
        return (int)count;
    }
    // the candidates of all CTAs (their numbers in slot 5) into the list, with their weights
    __device__ void fetch_list(const u64 *from, u64 count) const {
        uint32_t c = 0;
        u64 base = 0;
        for (u64 i = threadIdx.x; i < count; i += SAMPLE_THREADS) {
            while (i >= base + sh.slot[5][c]) base += sh.slot[5][c++];
            const u64 e = ld_cluster(from + (i - base), c);
            sh.comp[i] = e;
            sh.weight[i] = weight(logit_of(e));
        }
    }
    // the list of all that is kept, by the first CTA; the others have nothing left to do
    __device__ bool take_list(const u64 *from, u64 count) const {
        if (rank == 0) fetch_list(from, count);
        ptx::cluster_sync();  // the others' candidates have been read
        return rank == 0;
    }
    // Cuts `kept` behind the element at which the measure of the kept elements, added up in order, reaches target(measure of
    // all); WEIGHT: measure = weight, otherwise 1.  Where only elements of weight 0 are at stake, nothing is cut.  Returns the
    // length of the list that holds all that is kept, or 0 where there is none; WEIGHT without a list: sh.segment
    // has the warps' sums of the kept weights.
    template <bool WEIGHT, typename T>
    __device__ int cut(Kept &kept, T target_of) const {
        u64 target, sum = 0;
        hist_clear();
        if (threadIdx.x == 0) sh.bin[0] = sh.bin[1] = SAMPLE_BINS - 1;
        each4<false>([&](const float (&x)[4], int i) {
            bool in[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) in[k] = kept(x[k], i + k);
            if (WEIGHT) sum += weigh(x, in);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float at = bin_at(x[k]), magic = __fadd_rd(at, 0x1p23f);  // the floor, in the low bits
                const int b = __float_as_int(magic) & (SAMPLE_BINS - 1);
                uint32_t m = 1;
                if (WEIGHT) {
                    // share of the bin's largest weight in 16 bits: e^-z for z = fraction / 32, to z^3 / 6 < 2^-17
                    const float z = (at - (magic - 0x1p23f)) * (32.0f / SAMPLE_BINS);
                    m = __float_as_uint(fmaf(fmaf(z, fmaf(z, 0.5f, -1.0f), 1.0f), 65535.0f, 0x1p23f)) & 0xffffu;
                }
                if (in[k] && !(WEIGHT && b == SAMPLE_BINS - 1)) atomicAdd(sh.hist[0] + b, m);
            }
        });
        if (WEIGHT) tell(block_reduce(sum, plus), 3);
        ptx::cluster_sync();
        u64 mine[2];
        hist_row(0, mine);
        if (threadIdx.x == 0) sh.n_own = 0;
        if (WEIGHT) {
            // sums of shares are off by less than 2^-15: the border lies in the bins that reach target - slack .. target + slack
            const u64 all = told(3, plus);
            target = target_of(all);
            // In whole units of 2^-40, which the scan adds exactly: every number then lies in one bin
            const u64 aim = target >> 4, slack = all >> 18, low = aim > slack ? aim - slack : 0ull, high = aim + slack;
            u64 w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                w[k] = (u64)((double)mine[k] * (0x1p40 / 65535) * (double)exp2f((float)(2 * threadIdx.x + k) * (-1.4426950408889634f * 32 / SAMPLE_BINS)));
            u64 upto = w[0] + w[1];
            u64 shares = mine[0] + mine[1];  // up to bin[1]: 0.969 to 1 of 65535 for every element
            block_scan(upto, shares);
            if (threadIdx.x == SAMPLE_THREADS - 1) sh.upto = shares;
            __syncthreads();
#pragma unroll
            for (int k = 1; k >= 0; --k) {
                if (upto - w[k] < low && low <= upto) sh.bin[0] = 2 * threadIdx.x + k;
                if (upto - w[k] < high && high <= upto) {
                    sh.bin[1] = 2 * threadIdx.x + k;
                    sh.upto = shares;
                }
                upto -= w[k];
                shares -= mine[k];
            }
            if (threadIdx.x == 0 && low == 0) sh.bin[0] = 0;
        } else {
            target = target_of(0);
            find_bin(mine, target);
        }
        __syncthreads();
        const int b1 = sh.bin[1];
        if (!WEIGHT && b1 == SAMPLE_BINS - 1) {  // from 31.9 on in the exponent weights are 0: who is kept does not matter
            ptx::cluster_sync();                 // the histograms have been read
            return 0;
        }
        const bool list = WEIGHT ? sh.upto <= (u64)(SAMPLE_CAND * 0.96 * 65535) : sh.upto <= SAMPLE_CAND;
        const int b0 = list ? 0 : sh.bin[0];
        if (!WEIGHT && !list) target -= sh.before;

        // ---- the elements of bins b0 .. b1, and the sum of what lies before
        sum = 0;
        // the last bin's weights are 0 and its shares not counted: no border there, and no place in a list
        const float from = (float)b0, to = (float)(WEIGHT ? min(b1 + 1, SAMPLE_BINS - 1) : b1 + 1);
        each4<false>([&](const float (&x)[4], int i) {
            bool above[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float at = bin_at(x[k]);
                const bool in = at < to && kept(x[k], i + k);
                above[k] = in && at < from;
                if (in && at >= from) collect(comp_of(x[k], i + k));
            }
            if (WEIGHT) sum += weigh(x, above);
        });
        if (WEIGHT) tell(block_reduce(sum, plus), 4);
        __syncthreads();
        tell(sh.n_own, 5);
        ptx::cluster_sync();
        if (WEIGHT) target -= told(4, plus);
        u64 count = told(5, plus);
        const bool over = overflown(5);  // then the logits are gone over again, otherwise what was collected
        const uint32_t n_own = min(sh.n_own, (uint32_t)SAMPLE_OWN);
        const u64 *from_list = sh.own;
        // the part of the order that they span: by the bins' ends, and a little more than their rounding on either side
        const double wide_bin = 2.0 / (double)bins;
        u64 lo = comp_of(nextafterf((float)((double)top - (b0 ? b0 * wide_bin * (1.0 - 0x1p-20) : 0.0)), INFINITY) + 0.0f, 0);
        u64 hi = b1 < SAMPLE_BINS - 1 ? comp_of(nextafterf((float)((double)top - (b1 + 1) * wide_bin * (1.0 + 0x1p-20)), -INFINITY) + 0.0f, -1) : ~0ull;
        const auto candidate = [&](float x, int i) {
            const float at = bin_at(x);
            return at >= from && at < to && kept(x, i);
        };
        while (count > SAMPLE_CAND) {  // that part is cut into bins of 64-bit sums
            const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 10);
            hist_clear();
            if (over) {
                each4<true>([&](const float (&x)[4], int i) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const u64 c = comp_of(x[k], i + k);
                        const bool in = candidate(x[k], i + k) && c >= lo && c <= hi;
                        if (!__any_sync(0xffffffffu, in)) continue;
                        u64 m = !in ? 0ull : (WEIGHT ? weight(x[k]) : 1ull);
                        int b = m ? (int)((c - lo) >> shift) : -1;
                        if (__all_sync(0xffffffffu, b == __shfl_sync(0xffffffffu, b, 0))) {  // ties: one addition for the warp
                            m = warp_sum(m);
                            if (threadIdx.x & 31) b = -1;
                        }
                        hist_add64(b, m);
                    }
                });
            } else {
                for (uint32_t i = threadIdx.x; i < n_own; i += SAMPLE_THREADS) {
                    const u64 c = sh.own[i];
                    if (c >= lo && c <= hi) hist_add64((int)((c - lo) >> shift), WEIGHT ? weight(logit_of(c)) : 1ull);
                }
            }
            ptx::cluster_sync();
            u64 high[2];
            hist_row(0, mine);
            hist_row(1, high);
            mine[0] += high[0] << 32;
            mine[1] += high[1] << 32;
            find_bin(mine, target);
            if (threadIdx.x == 0) sh.n_chosen = 0;
            __syncthreads();
            target -= sh.before;
            const u64 first = lo;
            lo += (u64)sh.bin[0] << shift;
            hi = min(hi, lo + ((1ull << shift) - 1));
            u64 new_lo = ~0ull, new_hi = 0;
            auto choose = [&](u64 c) {
                const uint32_t slot = atomicAdd(&sh.n_chosen, 1u);
                if (slot < SAMPLE_CAND) sh.chosen[slot] = c;
                new_lo = min(new_lo, c);
                new_hi = max(new_hi, c);
            };
            if (over) {
                each4<false>([&](const float (&x)[4], int i) {
                    bool above[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const u64 c = comp_of(x[k], i + k);
                        const bool in = candidate(x[k], i + k);
                        above[k] = in && c >= first && c < lo;
                        if (in && c >= lo && c <= hi) choose(c);
                    }
                    if (WEIGHT) sum += weigh(x, above);
                });
            } else {
                for (uint32_t i = threadIdx.x; i < n_own; i += SAMPLE_THREADS)
                    if (sh.own[i] >= lo && sh.own[i] <= hi) choose(sh.own[i]);
            }
            __syncthreads();
            tell(sh.n_chosen, 5);
            ptx::cluster_sync();
            count = told(5, plus);
            from_list = sh.chosen;
            if (count > SAMPLE_CAND) {
                lo = cluster_reduce(new_lo, 6, least);
                hi = ~cluster_reduce(~new_hi, 7, least);
            }
        }
        if (list) {
            if (take_list(from_list, count)) cut_list<WEIGHT>(kept, (uint32_t)count, target);
            return (int)count;
        }
        fetch_list(from_list, count);
        cut_list<WEIGHT>(kept, (uint32_t)count, target);
        if (WEIGHT) {  // what is kept of this CTA's candidates goes to its segment
            sum = warp_sum(sum);
            if ((threadIdx.x & 31) == 0) sh.segment[threadIdx.x >> 5] = sum;
            __syncthreads();
            auto put = [&](u64 e) {
                if (kept(logit_of(e), (int)(uint32_t)e))
                    atomicAdd(sh.segment + ((int)(uint32_t)e - i0) / 4 / quads_per_warp(), weight(logit_of(e)));
            };
            if (over) {
                for (uint32_t i = threadIdx.x; i < min(sh.n_chosen, (uint32_t)SAMPLE_CAND); i += SAMPLE_THREADS) put(sh.chosen[i]);
            } else {
                for (uint32_t i = threadIdx.x; i < n_own; i += SAMPLE_THREADS) put(sh.own[i]);
            }
            __syncthreads();
        }
        return 0;
    }
    __device__ __forceinline__ int quads_per_warp() const { return max(1, ((n + 3) / 4 + SAMPLE_WARPS - 1) / SAMPLE_WARPS); }

    // The first `count` elements of the list by key into the scratch space, comp and weight: an element's place is the number of
    // smaller keys, which several threads count (c^2 / 512 steps of 2 keys: 1 us for 256 elements).  The histograms' space is free
    // while there is a list.
    __device__ __forceinline__ u64 *scratch_list() const { return reinterpret_cast<u64 *>(sh.hist); }
    template <typename K>
    __device__ __forceinline__ void place(uint32_t count, K key) const {
        static_assert(sizeof(sh.hist) >= 2 * SAMPLE_CAND * sizeof(u64) && SAMPLE_CAND <= SAMPLE_THREADS, "");
        uint32_t per = 1;  // threads per element
        while (per < 32 && 2 * per * count <= SAMPLE_THREADS) per *= 2;
        __syncthreads();
        const uint32_t i = threadIdx.x / per;
        const u64 e = sh.comp[min(i, count - 1)];
        const auto c = key(e);
        uint32_t before = 0;
#pragma unroll 4
        for (uint32_t j = 2 * (threadIdx.x % per); j < count; j += 2 * per) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(sh.comp + j);
            before += (key(two.x) < c ? 1 : 0) + (j + 1 < count && key(two.y) < c ? 1 : 0);
        }
        for (uint32_t o = per / 2; o > 0; o /= 2) before += __shfl_xor_sync(0xffffffffu, before, o);
        if (i < count && threadIdx.x % per == 0) {
            scratch_list()[before] = e;
            scratch_list()[SAMPLE_CAND + before] = sh.weight[i];
        }
        __syncthreads();
    }
    // cuts behind the element of the list, one a thread, at which the running sum of v reaches target(sum of all)
    template <typename T>
    __device__ __forceinline__ void cut_at(Kept &kept, u64 v, T target_of) const {
        u64 upto = v;
        block_scan(upto);
        if (threadIdx.x == SAMPLE_THREADS - 1) sh.upto = upto;
        __syncthreads();
        const u64 target = target_of(sh.upto);
        if (upto - v < target && target <= upto) sh.found = sh.comp[threadIdx.x];
        __syncthreads();
        kept.cut(sh.found);
    }
    // puts the list in order and cuts behind the element at which the measure reaches target
    template <bool WEIGHT>
    __device__ void cut_list(Kept &kept, uint32_t count, u64 target) const {
        place(count, [](u64 c) { return c; });
        if (threadIdx.x < count) {
            sh.comp[threadIdx.x] = scratch_list()[threadIdx.x];
            sh.weight[threadIdx.x] = scratch_list()[SAMPLE_CAND + threadIdx.x];
        }
        __syncthreads();
        if (WEIGHT) cut_at(kept, threadIdx.x < count ? sh.weight[threadIdx.x] : 0ull, [&](u64) { return target; });
        else kept.cut(sh.comp[min(target, (u64)count) - 1]);
    }
    __device__ __forceinline__ bool keeps(const Kept &kept, uint32_t count) const {  // this thread's element of the list
        const u64 c = sh.comp[threadIdx.x % SAMPLE_CAND];
        return threadIdx.x < count && kept(logit_of(c), (int)(uint32_t)c);
    }
};

__device__ __forceinline__ u64 drawn(float u, u64 z) {  // u of z, below z
    const u64 d = u > 0.0f ? (u64)((double)fminf(u, 1.0f) * (double)z) : 0ull;
    return min(d, z - 1);
}

__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(smem);
    uint32_t ctas;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t r = blockIdx.x / ctas;
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA runs: the others may write to its slots
    Row row = {sh};
    row.held = p.held;
    row.rank = ptx::cluster_ctarank();
    row.ctas = ctas;
    row.i0 = min(p.vocab, (int)row.rank * p.slice);
    row.n = min(p.slice, p.vocab - row.i0);
    const int quads = (row.n + 3) / 4;
    row.q0 = min(quads, warp * row.quads_per_warp());
    row.q1 = min(quads, row.q0 + row.quads_per_warp());
    if (threadIdx.x < 32) {
        const double s = exp2(44.0 + (double)threadIdx.x * (1.0 / 32));
        sh.scale[threadIdx.x] = __hiloint2double(__double2hiint(s) - ((int)threadIdx.x << 15), __double2loint(s));
    }
    pdl_release_and_wait();
    const float *src = p.logits + r * p.ld + row.i0;
    row.l = src;
    row.wide = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
    float top = -INFINITY;
    int top_at = 0;  // the first quad of this thread that holds its largest
    const auto rise = [&](float m, int i) {
        if (m > top) top = m, top_at = i;
    };
    if (row.held) {
        float *held = reinterpret_cast<float *>(smem + SAMPLE_FIXED);
        row.l = held;
        const int body = row.wide ? row.n / 4 : 0;
#pragma unroll 8
        for (int i = threadIdx.x; i < body; i += SAMPLE_THREADS) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(src) + i);
            reinterpret_cast<float4 *>(held)[i] = make_float4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
            rise(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), i);  // passes over NaN
        }
#pragma unroll 4
        for (int i = 4 * body + threadIdx.x; i < 4 * quads; i += SAMPLE_THREADS) {
            const float v = i < row.n ? clean(__ldcg(src + i)) : -INFINITY;
            held[i] = v;
            rise(v, i / 4);
        }
    } else {
        row.each4<false>([&](const float (&x)[4], int i) { rise(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), (i - row.i0) / 4); });
    }
    const float mine_top = top, temp = p.temperature ? p.temperature[r] : 1.0f;
    // the smallest of ~ordered bits: one instruction a warp
    const uint32_t warp_top = __reduce_min_sync(0xffffffffu, (uint32_t)(comp_of(top + 0.0f, 0) >> 32));
    if (lane == 0) sh.scratch[warp] = warp_top;
    __syncthreads();  // the slice and the table are there, too
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    top = logit_of((u64)__reduce_min_sync(0xffffffffu, (uint32_t)sh.scratch[lane % SAMPLE_WARPS]) << 32);
    if (!(temp > 0.0f)) {  // the first of the largest: of the slice, then of all
        u64 best = ~0ull;
        if (mine_top + 0.0f == top && row.n > 0) {
            float x[4];
            row.load4(top_at, x);
#pragma unroll
            for (int k = 3; k >= 0; --k)
                if (x[k] == top) best = comp_of(top, row.i0 + 4 * top_at + k);
        }
        best = row.cluster_reduce(best, 0, least);
        row.top = logit_of(best);
        if (row.rank == 0 && threadIdx.x == 0) {
            p.tokens[r] = row.top == -INFINITY ? 0 : (long long)(uint32_t)best;
            if (p.logprobs) p.logprobs[r] = row.top == -INFINITY ? __uint_as_float(0x7fffffffu) : 0.0f;
        }
        return;
    }
    row.tell(comp_of(top, 0), 0);
    ptx::cluster_sync();
    top = logit_of(row.told(0, least));
    row.top = fminf(top, FLT_MAX);
    if (top == -INFINITY) {
        if (row.rank == 0 && threadIdx.x == 0) {
            p.tokens[r] = 0;
            if (p.logprobs) p.logprobs[r] = __uint_as_float(0x7fffffffu);
        }
        return;
    }
    const float temp_used = fmaxf(temp, 0x1p-100f);  // below that `bins` could leave f32
    const double inv_t = 1.0 / (double)temp_used;
    row.per = inv_t * 1.4426950408889634074;
    row.bins = (float)(inv_t * (SAMPLE_BINS / 16));
    Kept kept = {top == INFINITY ? INFINITY : -FLT_MAX, 0x7fffffff};
    const int k = p.top_k ? p.top_k[r] : 0;
    int list = 0;
    if (k > 0 && k < p.vocab) {
        if (k <= SAMPLE_CAND / 2) list = row.cut_few(kept, mine_top, k);
        if (!list) list = row.cut<false>(kept, [&](u64) { return (u64)k; });
        if (list && row.rank) return;
    }
    const float mp = p.min_p ? p.min_p[r] : 0.0f;
    if (mp > 0.0f && temp < INFINITY) {  // an infinite temperature makes all finite logits equal
        // the smallest f32 logit that passes: the border in f64 is within a rounding of it
        const double border = log((double)fminf(mp, 1.0f));
        const auto passes = [&](float x) { return x >= row.top || ((double)x - (double)row.top) * inv_t >= border; };
        float x = fminf((float)((double)row.top + border * (double)temp_used), row.top);
        for (int i = 0; i < 4 && !passes(x); ++i) x = nextafterf(x, INFINITY);
        for (int i = 0; i < 4 && x > -INFINITY && passes(nextafterf(x, -INFINITY)); ++i) x = nextafterf(x, -INFINITY);
        kept.cut(x, 0x7fffffff);
    }
    const float tp = p.top_p ? p.top_p[r] : 1.0f;
    const auto nucleus = [&](u64 all) { return min(max((u64)ceil((double)fmaxf(tp, 0.0f) * (double)all), 1ull), all); };
    bool summed = false;
    if (tp < 1.0f) {
        if (list) {
            row.cut_at(kept, row.keeps(kept, list) ? sh.weight[threadIdx.x] : 0ull, nucleus);
        } else {
            list = row.cut<true>(kept, nucleus);
            if (list && row.rank) return;
            summed = true;
        }
    }
    const float u = p.u[r];
    const auto chosen = [&](float x, int i, u64 all) {
        p.tokens[r] = i;
        if (p.logprobs) {
            const double e = ((double)fminf(x, FLT_MAX) - (double)row.top) * inv_t;
            p.logprobs[r] = (float)(e - log((double)all * 0x1p-44));
        }
    };
    if (list) {  // in order: the kept ones are its first
        const uint32_t many = __syncthreads_count(row.keeps(kept, list));
        row.place(many, [](u64 c) { return (uint32_t)c; });
        const u64 w = threadIdx.x < many ? row.scratch_list()[SAMPLE_CAND + threadIdx.x] : 0ull;
        u64 upto = w;
        row.block_scan(upto);
        if (threadIdx.x == SAMPLE_THREADS - 1) sh.upto = upto;
        __syncthreads();
        const u64 all = sh.upto, draw = drawn(u, all);
        if (draw >= upto - w && draw < upto) {
            const u64 c = row.scratch_list()[threadIdx.x];
            chosen(logit_of(c), (int)(uint32_t)c, all);
        }
        return;
    }
    // ---- the draw: the warps' sums of kept weights, then the segment that holds the number is walked in index order
    const auto kept4 = [&](const float (&x)[4], int i, bool (&in)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) in[j] = kept(x[j], i + j);
    };
    if (!summed) {
        u64 s = 0;
        row.each4<false>([&](const float (&x)[4], int i) {
            bool in[4];
            kept4(x, i, in);
            s += row.weigh(x, in);
        });
        s = warp_sum(s);
        if (lane == 0) sh.segment[warp] = s;
        __syncthreads();
    }
    // this CTA's sums up to each of its segments
    const u64 upto = warp_scan(lane < SAMPLE_WARPS ? sh.segment[lane] : 0ull), mine = __shfl_sync(0xffffffffu, upto, SAMPLE_WARPS - 1);
    row.tell(mine, 2);
    ptx::cluster_sync();  // nothing of another CTA is read from here on
    u64 before = 0, z = 0;
    for (uint32_t c = 0; c < ctas; ++c) {
        if (c < row.rank) before += sh.slot[2][c];
        z += sh.slot[2][c];
    }
    const u64 draw = drawn(u, z);
    if (draw < before || draw >= before + mine) return;  // one CTA of the cluster goes on, with one of its segments
    const int seg = __ffs(__ballot_sync(0xffffffffu, draw < before + upto)) - 1;
    if (seg > 0) before += __shfl_sync(0xffffffffu, upto, seg - 1);
    const int end = min(quads, (seg + 1) * row.quads_per_warp());
    for (int i0 = seg * row.quads_per_warp(); i0 < end; i0 += SAMPLE_THREADS) {
        const int i = i0 + threadIdx.x;
        float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i < end) row.load4(i, x);
        u64 w[4], own = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = kept(x[j], row.i0 + 4 * i + j) ? row.weight(x[j]) : 0ull;
            own += w[j];
        }
        u64 at = own;
        row.block_scan(at);
        if (threadIdx.x == SAMPLE_THREADS - 1) sh.upto = at;
        at += before - own;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (draw >= at && draw < at + w[j]) chosen(x[j], row.i0 + 4 * i + j, z);
            at += w[j];
        }
        __syncthreads();
        before += sh.upto;
        if (draw < before) return;
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
    // CTAs per row: slices of at least 1024 logits, and as many CTAs as there are: a batch of unlike rows (greedy ones next to
    // flat nuclei) fills the SMs better in many short CTAs than in one round of long ones (128 mixed rows of 131072: 76 us with
    // eight, 86 with four, 108 with two)
    const size_t sms = (size_t)sm_count(dev);
    int ctas = 1;
    while (ctas < SAMPLE_CTAS && vocab > (size_t)1024 * ctas) ctas *= 2;
    const int slice = (int)(((vocab + ctas - 1) / ctas + 3) / 4 * 4);
    // the slice in shared memory where one CTA per SM (few rows), or two, have the room
    const size_t room = n * ctas <= sms ? 200 * 1024 : 100 * 1024;
    const bool held = SAMPLE_FIXED + (size_t)slice * 4 <= room;
    SampleParams p = {logits, ld, (int)vocab, slice, held, temperature, top_k, top_p, min_p, u, tokens, logprobs};
    const size_t smem = SAMPLE_FIXED + (held ? (size_t)slice * 4 : 0);
    if (int rc = set_dyn_smem_once(reinterpret_cast<const void *>(sample_kernel), dev, 200 * 1024, "sample smem attribute")) return rc;
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
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, p);
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "sample launch");
}
