// A KV cache held in 4 bits: append (with the norms of queries and keys and the rotation), read-back, attention (sm_100a).
//
// Layout and arithmetic are those of include/kore_b200.h: one row per (sequence, KV head, position), 4-bit codes in
// natural dim order (dim 8w + i in bits 4i .. 4i+3 of word w) and one word (bfloat16 step | bfloat16 lo << 16); a code c
// stands for lo + c * step.  One pair per row keeps the unpacking out of the products: a score is
//     step_j * sum_d(q_d c_jd) + lo_j * sum_d(q_d)      and an output      sum_j (p_j step_j) c_jd + sum_j p_j lo_j,
// so both contractions run on bare codes and the pair touches one number per (query, position).
#include <cuda_fp16.h>

#include "common.cuh"
#include "device_utils.cuh"

namespace kb {

constexpr int KV4_MAX_HD = 128;
constexpr int KV4_MAX_LEN = 1 << 30;  // positions are 32-bit numbers, with room for a chunk behind the last one

__host__ __device__ inline int kv4_words(int hd) { return (hd + 7) / 8; }

__device__ __forceinline__ float kv4_step(uint32_t s) { return __uint_as_float(s << 16); }
__device__ __forceinline__ float kv4_lo(uint32_t s) { return __uint_as_float(s & 0xffff0000u); }

// ---- norm + rotation + append ------------------------------------------------------------------
struct AppendParams {
    const float *qkv;
    size_t ld;
    const int *positions;
    const long long *cache_rows;
    const float *cos_t, *sin_t;
    int max_pos;
    const float *q_gamma, *k_gamma;
    float eps;
    double per_dim;  // 1 / hd
    unsigned tasks, groups;  // tokens * groups of heads
    int n_heads, n_kv, hd;
    long long cache_len;  // n_seqs * lmax
    int lmax;
    float *q_out, *k_cache, *v_cache;
    uint32_t *k_codes, *k_steps, *v_codes, *v_steps;
};

// the bfloat16 at or below x (finite), and the one at or above x >= 0
__device__ __forceinline__ float bf16_below(float x) {
    const uint32_t i = __float_as_uint(x), cut = i & 0xffff0000u;
    return __uint_as_float(x < 0.0f && i != cut ? cut + 0x10000u : cut);
}
__device__ __forceinline__ float bf16_above_nonneg(float x) {
    const uint32_t i = __float_as_uint(x), cut = i & 0xffff0000u;
    return __uint_as_float(i != cut ? cut + 0x10000u : cut);
}
// minima and maxima that a NaN passes through
__device__ __forceinline__ float min_nan(float x, float y) {
    float z;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}
__device__ __forceinline__ float warp_min_nan(float x) {
    float y;
    asm volatile("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
// sequence and position of a cache row
__device__ __forceinline__ void split_row(long long row, int lmax, size_t &seq, size_t &pos) {
    if (row >> 32) {
        seq = (size_t)(row / lmax);
        pos = (size_t)(row - (long long)seq * lmax);
    } else {
        seq = (uint32_t)row / (uint32_t)lmax;
        pos = (uint32_t)row - (uint32_t)seq * (uint32_t)lmax;
    }
}
// 1 / sqrt(x) to 2^-52: an f32 estimate and two Newton steps, 9 f64 operations where division and root take ten times as many
__device__ __forceinline__ double rsqrt_f64(double x) {
    if (!(x > 1e-30 && x < 1e30)) return 1.0 / sqrt(x);
    double y = (double)rsqrtf((float)x);
#pragma unroll
    for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
    return y;
}
// Sum over the warp of one of HPW values, that of index lane / (32 / HPW): while a lane holds several it passes on half of
// them.  What follows on the sums is then done for all of them at once.
template <int HPW>
__device__ __forceinline__ double warp_sum_of(double (&v)[HPW]) {
    const int lane = threadIdx.x & 31;
    int o = 16;
#pragma unroll
    for (int left = HPW / 2; left > 0; left /= 2, o /= 2)
#pragma unroll
        for (int i = 0; i < left; ++i) {
            const double mine = lane & o ? v[left + i] : v[i], other = lane & o ? v[i] : v[left + i];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, other, o);
        }
#pragma unroll
    for (int k = 16 / HPW; k > 0; k /= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], k);
    return v[0];
}

// Bound by one memory round trip for a few tokens (16 tokens, 32 heads of 100, norms, f32 cache: 2.7 us) and for many by the
// bytes of the rows, which the quantiser does not quite hide: 8192 tokens of 32 + 2 x 8 heads of 128 with norms take 66 us for
// 344 MB of rows read and written (5.2 TB/s; 62 us for 402 MB, 6.5 TB/s, with an f32 cache).  A warp takes HPW heads of one token:
// its lane l owns the rotation pairs 2l and 2l + 1, dims {2l, 2l + 1} of each half, so that its codes are whole bytes of the
// row, a row needs no shared memory, and the token's angles are read once for all heads.
// PAIRS: rows and tables are 8-byte aligned and half is even, a lane's two neighbours come and go in one access.
// FULL: heads of 128, every lane owns its pairs, so nothing is predicated and addresses are shifts (66 us against 80 us for the
// 8192 tokens above, 62 and 72 us with an f32 cache).
template <bool Q4, int HPW, bool PAIRS, bool FULL = false>
__global__ void __launch_bounds__(256) append_kernel(AppendParams p) {
    const int lane = threadIdx.x & 31;
    const unsigned task = blockIdx.x * 8u + (threadIdx.x >> 5);
    pdl_release_and_wait();
    if (task >= p.tasks) return;
    const int heads = p.n_heads + 2 * p.n_kv, hd = FULL ? 128 : p.hd, half = hd / 2;
    const unsigned t = task / p.groups;
    const int head0 = (int)(task - t * p.groups) * HPW;
    const int i0 = 2 * lane;
    const bool own0 = FULL || i0 < half, own1 = FULL || i0 + 1 < half;
    float a[HPW][2], b[HPW][2];
    const float *row = p.qkv + (size_t)t * p.ld + (size_t)head0 * hd;
    auto load2 = [&](const float *src, float (&x)[2]) {
        if (PAIRS) {
            const float2 v = own0 ? *reinterpret_cast<const float2 *>(src + i0) : make_float2(0.0f, 0.0f);
            x[0] = v.x; x[1] = v.y;
        } else {
            x[0] = own0 ? src[i0] : 0.0f;
            x[1] = own1 ? src[i0 + 1] : 0.0f;
        }
    };
    auto store2 = [&](float *dst, const float (&x)[2]) {
        if (PAIRS) {
            if (own0) *reinterpret_cast<float2 *>(dst + i0) = make_float2(x[0], x[1]);
        } else {
            if (own0) dst[i0] = x[0];
            if (own1) dst[i0 + 1] = x[1];
        }
    };
#pragma unroll
    for (int j = 0; j < HPW; ++j) {
        a[j][0] = a[j][1] = b[j][0] = b[j][1] = 0.0f;
        if (head0 + j < heads) {
            load2(row + j * hd, a[j]);
            load2(row + j * hd + half, b[j]);
        }
    }
    const int pos = p.positions[t];
    const bool pos_ok = pos >= 0 && pos < p.max_pos;
    const long long crow = p.cache_rows[t];
    const bool stored = pos_ok && crow >= 0 && crow < p.cache_len;
    float c[2] = {}, s[2] = {};
    if (head0 < p.n_heads + p.n_kv && pos_ok) {
        load2(p.cos_t + (size_t)pos * half, c);
        load2(p.sin_t + (size_t)pos * half, s);
    }
    const bool normed = p.q_gamma || p.k_gamma;
    float inv_of = 0.0f;  // of head lane / (32 / HPW)
    if (normed) {
        // f64, in one order whatever HPW (lanes 16, 8, 4, 2, 1 apart), so that every launch gives the same codes.  A sum in
        // another order rounds inv differently in about one row of 2^28
        double ss[HPW];
#pragma unroll
        for (int j = 0; j < HPW; ++j) {
            ss[j] = 0.0;
#pragma unroll
            for (int i = 0; i < 2; ++i) ss[j] = fma((double)a[j][i], (double)a[j][i], fma((double)b[j][i], (double)b[j][i], ss[j]));
        }
        inv_of = (float)rsqrt_f64(warp_sum_of<HPW>(ss) * p.per_dim + (double)p.eps);
    }
    auto scale = [&](int j, const float (&ga)[2], const float (&gb)[2]) {
        const float inv = HPW == 1 ? inv_of : __shfl_sync(0xffffffffu, inv_of, 32 / HPW * j);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[j][i] = __fmul_rn(__fmul_rn(a[j][i], inv), ga[i]);
            b[j][i] = __fmul_rn(__fmul_rn(b[j][i], inv), gb[i]);
        }
    };
    auto rotate = [&](int j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = a[j][i], y = b[j][i];
            a[j][i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
            b[j][i] = __fadd_rn(__fmul_rn(x, s[i]), __fmul_rn(y, c[i]));
        }
    };
    const float bad = __uint_as_float(0x7fffffffu);
    float ga[2] = {}, gb[2] = {};
    if (HPW > 1 && head0 + HPW <= p.n_heads) {  // queries only
        if (p.q_gamma) {
            load2(p.q_gamma, ga);
            load2(p.q_gamma + half, gb);
#pragma unroll
            for (int j = 0; j < HPW; ++j) scale(j, ga, gb);
        }
        float *dst = p.q_out + ((size_t)t * p.n_heads + head0) * hd;
#pragma unroll
        for (int j = 0; j < HPW; ++j) {
            rotate(j);
            if (!pos_ok) a[j][0] = a[j][1] = b[j][0] = b[j][1] = bad;
            store2(dst + j * hd, a[j]);
            store2(dst + j * hd + half, b[j]);
        }
        return;
    }
    if (normed) {
        const float *held = nullptr;  // the gamma in ga and gb
#pragma unroll
        for (int j = 0; j < HPW; ++j) {
            const float *gamma = head0 + j < p.n_heads ? p.q_gamma : (head0 + j < p.n_heads + p.n_kv ? p.k_gamma : nullptr);
            if (!gamma) continue;
            if (gamma != held) {
                held = gamma;
                load2(gamma, ga);
                load2(gamma + half, gb);
            }
            scale(j, ga, gb);
        }
    }
    size_t seq = 0, cpos = 0;
    if (stored && head0 + HPW > p.n_heads) split_row(crow, p.lmax, seq, cpos);
    const size_t at0 = seq * p.n_kv * p.lmax + cpos;
    float mn_of = 0.0f, mx_of = 0.0f;  // lane j: of head j
#pragma unroll
    for (int j = 0; j < HPW; ++j) {
        const int head = head0 + j;
        if (head >= heads) break;
        const bool is_q = head < p.n_heads, is_v = head >= p.n_heads + p.n_kv;
        if (!is_v) rotate(j);
        if (!is_q && !stored) continue;
        if (is_q || !Q4) {
            const int kvh = is_v ? head - p.n_heads - p.n_kv : head - p.n_heads;
            float *dst = is_q ? p.q_out + ((size_t)t * p.n_heads + head) * hd : (is_v ? p.v_cache : p.k_cache) + (at0 + (size_t)kvh * p.lmax) * hd;
            if (is_q && !pos_ok) a[j][0] = a[j][1] = b[j][0] = b[j][1] = bad;
            store2(dst, a[j]);
            store2(dst + half, b[j]);
            continue;
        }
        // hd is a multiple of 4 here, so a lane owns both of its pairs or none
        const float mn = warp_min_nan(own0 ? min_nan(min_nan(a[j][0], a[j][1]), min_nan(b[j][0], b[j][1])) : INFINITY);
        const float mx = warp_max(own0 ? fmaxf(fmaxf(a[j][0], a[j][1]), fmaxf(b[j][0], b[j][1])) : -INFINITY);
        if (HPW == 1 || lane == j) mn_of = mn, mx_of = mx;
    }
    if (!Q4 || !stored || head0 + HPW <= p.n_heads) return;
    // the pair of each head, in lane j for head j; an infinity or a NaN in the row makes one of the two no number
    const float lo_of = bf16_below(mn_of);
    const float step_of = bf16_above_nonneg(fmaxf(__fdiv_rn(__fsub_rn(mx_of, lo_of), 15.0f), 0x1p-100f));
    const bool ok_of = fabsf(lo_of) < INFINITY && step_of < INFINITY;
    const float per_of = ok_of ? __frcp_rn(step_of) : 0.0f;  // 0: no row
    const int words = kv4_words(hd);
    if (lane < HPW && head0 + lane >= p.n_heads && head0 + lane < heads) {
        const int kvh = head0 + lane - p.n_heads;
        const size_t at = at0 + (size_t)(kvh >= p.n_kv ? kvh - p.n_kv : kvh) * p.lmax;
        (kvh >= p.n_kv ? p.v_steps : p.k_steps)[at] = ok_of ? (__float_as_uint(lo_of) | __float_as_uint(step_of) >> 16) : 0x7fc07fc0u;
    }
#pragma unroll
    for (int j = 0; j < HPW; ++j) {
        const int head = head0 + j;
        if (head >= heads) break;
        const float lo = __shfl_sync(0xffffffffu, lo_of, j), per = __shfl_sync(0xffffffffu, per_of, j);
        if (head < p.n_heads) continue;
        const bool is_v = head >= p.n_heads + p.n_kv;
        const size_t at = at0 + (size_t)(is_v ? head - p.n_heads - p.n_kv : head - p.n_heads) * p.lmax;
        // a code lies in 0 .. 15 already: x >= lo, and step is not below (max - lo) / 15.  Adding 1.5 2^23 rounds to even; two
        // of them make a byte of the sum's low bits
        auto whole = [&](float x) { return __fadd_rn(__fmul_rn(__fsub_rn(x, lo), per), 12582912.0f); };
        auto byte_of = [&](const float (&x)[2]) { return per == 0.0f ? (uint8_t)0 : (uint8_t)__float_as_uint(fmaf(whole(x[1]) - 12582912.0f, 16.0f, whole(x[0]))); };
        uint8_t *bytes = reinterpret_cast<uint8_t *>((is_v ? p.v_codes : p.k_codes) + at * words);
        if (own0) {
            bytes[lane] = byte_of(a[j]);
            bytes[half / 2 + lane] = byte_of(b[j]);
        }
        if (!FULL && lane < 4 * words - half) bytes[half + lane] = 0;  // tail of the last word
    }
}

// ---- read-back ---------------------------------------------------------------------------------
// Bound by the bytes written.  A warp takes one row and two heads of it; a lane writes 16 bytes of K and of V, so a
// store covers whole lines, and reads its 16 bits of codes from a word that it shares with its neighbour.
constexpr int READ_HEADS = 2;  // 4 x 8192 rows of 8 heads: 53 us with two, 59 with four, 71 with one
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint32_t *k_codes, const uint32_t *k_steps, const uint32_t *v_codes,
                                                       const uint32_t *v_steps, const long long *cache_rows, unsigned tasks, unsigned groups,
                                                       int n_kv, int hd, long long cache_len, int lmax, float *k_out, float *v_out) {
    const int lane = threadIdx.x & 31;
    const unsigned task = blockIdx.x * 8u + (threadIdx.x >> 5);
    pdl_release_and_wait();
    if (task >= tasks || 4 * lane >= hd) return;
    const unsigned i = task / groups;
    const int head0 = (int)(task - i * groups) * READ_HEADS, words = kv4_words(hd);
    const long long crow = cache_rows[i];
    const bool ok = crow >= 0 && crow < cache_len;
    size_t seq = 0, pos = 0;
    if (ok) split_row(crow, lmax, seq, pos);
    uint32_t c[2][READ_HEADS], s[2][READ_HEADS];
#pragma unroll
    for (int j = 0; j < READ_HEADS; ++j) {
        const bool live = ok && head0 + j < n_kv;
        const size_t at = (seq * n_kv + (live ? head0 + j : 0)) * lmax + pos;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const bool get = live && (side ? v_out : k_out);
            c[side][j] = get ? (side ? v_codes : k_codes)[at * words + (lane >> 1)] >> (16 * (lane & 1)) : 0u;
            s[side][j] = get ? (side ? v_steps : k_steps)[at] : 0u;  // a row outside the cache: lo + 0 * 0 = 0
        }
    }
#pragma unroll
    for (int j = 0; j < READ_HEADS; ++j) {
        if (head0 + j >= n_kv) return;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float *out = side ? v_out : k_out;
            if (!out) continue;
            const float step = kv4_step(s[side][j]), lo = kv4_lo(s[side][j]);
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = fmaf(__uint_as_float(0x4b000000u | (c[side][j] >> (4 * k) & 15u)) - 8388608.0f, step, lo);
            *reinterpret_cast<float4 *>(out + ((size_t)i * n_kv + head0 + j) * hd + 4 * lane) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

// ---- attention ---------------------------------------------------------------------------------
// Bound by the bytes of the cache as long as the unpacking keeps up (8 sequences of 8191 .. 32768 positions, 8 KV heads of 128:
// 46.6 us, 3.8 TB/s; 16 sequences of 513 .. 640, 32 KV heads of 100: 13.6 us, 6.5 of them in the five tiles of a warp): at the
// copy bandwidth an SM receives a position (K and V, 136 bytes for heads of 128) every 6 clocks, too few for a multiply-add per
// value on the FP32 lanes.  So both products run on the matrix instruction m16n8k16 with f16 operands and f32 sums, and a 4-bit
// code becomes an operand by masking alone: the bits 0x00f0 of a 16-bit lane ARE the f16 number code * 2^-20 (subnormal, exact,
// taken as such by the instruction).  The factor goes into the end of the sums.  The bits 0x000f would do as well (code *
// 2^-24, two shifts fewer per eight codes), but the instruction aligns its products by the operands' exponent fields, so
// leading zeros cost bits of the sum: results were 1e-5 off that way.
//   The other operand must keep f32 accuracy: queries and softmax weights are split into two f16 terms, x = hi + lo, 22
// bits of x, for which rows are scaled by powers of two.
//   Codes are the 16-row operand, queries and weights the 8-column one (S^T = K Q^T, O^T = V^T P^T): the two terms of four
// query rows fill the columns, so four rows are served at the price of one, and the accumulators of 128 dims, both terms in
// one, take 16 registers.  Up to eight rows take a second set of columns (NT = 2) over the same unpacked codes.
//   Lane (g, t) = (lane / 4, lane % 4).  The contraction over dims runs in any order as long as queries and keys agree, so
// a lane takes whole words of key rows 2g and 2g + 1.  It gets hi and lo of query t at these positions, adds them, and after
// the softmax packs hi and lo of the weight in the same place; a transposition of 8 x 8 tiles (movmatrix) makes them the
// operand of the second product, where lane t meets positions 4t .. 4t+3 and row g of tile j is dim 8 word(g) + j.
//   The largest score is a reference only: weights up to 2^8 above it are allowed before sums are rescaled, so a tile
// costs two votes and most tiles nothing else.
//   A warp streams its own 32-position tiles through a ring of 16-byte asynchronous copies (no barrier between warps) and
// the warps of a CTA deal the tiles of a chunk.  A CTA costs about three tiles of a warp before and behind its loop, so long
// caches are cut into as many chunks as fill the GPU once, of one size for all sequences: the CTAs work that out from the
// lengths, and a second kernel joins the chunks.
constexpr int ATT4_WARPS = 4;
constexpr int ATT4_STAGES = 2;   // with 16 warps on an SM a second tile in flight each is enough
constexpr int ATT4_PER_SM = 4;   // resident CTAs: 128 registers a thread (five with 96 take 2.3 us longer for 16 sequences of 640)
constexpr int ATT4_TILE = 32;  // positions of a warp's tile
constexpr int ATT4_ROWS = 4;   // query rows of a set of columns
constexpr int ATT4_GRAIN = ATT4_WARPS * ATT4_TILE;  // positions that give every warp a tile
// A cache with room for so many grains is not split, so that the call is one launch without a search for work and a join: 577
// positions of one sequence and 32 KV heads take 6.4 us, and 7.2 us split, in a cache of 1024; from ATT4_MANY units on two grains more
// (4 sequences of 760 positions, 8 KV heads, five tokens: 10.8 us whole, 14.2 split).  By capacity, because the host does not know
// the lengths: in a larger cache both kernels run, and sequences of these lengths are then better split than kept whole (the 577: 7.2
// and 7.9 us; 16 sequences of 513 .. 640, 8 KV heads: 12.8 and 13.6 us), but for the shortest (16 of 100 .. 200: 9.9 and 8.0 us)
constexpr int ATT4_WHOLE = 5, ATT4_MANY = 32;
constexpr int ATT4_ROUND = 32;  // chunks that the second kernel takes in a round
constexpr float ATT4_SLACK = 8.0f;  // log2 of how far a weight may rise above the reference

struct AttnParams {
    const float *q;
    const uint32_t *k_codes, *k_steps, *v_codes, *v_steps;
    const int *lens;
    int t, n_heads, n_kv, rep, hd, lmax, words;
    int batch, row_tiles, tile_rows;
    int least_ctas;  // sequences * units, where slots > 0 and that is below it; otherwise slots
    int slots;  // CTAs that the GPU holds; 0: nothing is split, a CTA per unit (sequence, KV head, tile of query rows)
    float scale;
    float *out;
    float *part;      // [CTAs][tile_rows][hd] unnormalised sums
    float2 *part_ml;  // [CTAs][tile_rows] (largest score, sum of weights)
    int2 *part_of;    // [units] (first CTA, CTAs) of a unit
};

__device__ __forceinline__ int kv4_len(const AttnParams &p, int b) { return min(max(p.lens[b], 0), p.lmax); }

// What a CTA works on.  In a split launch every unit (KV head, tile of query rows) of sequence b is cut into ceil(grains of
// b / size) chunks, at least one; every warp works that out alike from the lengths.
struct AttnWork {
    int b, len, unit, chunk, chunks, size;  // unit: of the sequence; size in grains
};
__device__ __forceinline__ bool find_attn_work(const AttnParams &p, AttnWork &w) {
    const int lane = threadIdx.x & 31, units = p.n_kv * p.row_tiles;
    if (p.slots == 0) {
        w.b = blockIdx.x / units;
        w.unit = blockIdx.x - w.b * units;
        w.len = kv4_len(p, w.b);
        w.chunk = 0; w.chunks = 1; w.size = (p.lmax + ATT4_GRAIN - 1) / ATT4_GRAIN;
        return true;
    }
    const int len0 = lane < p.batch ? kv4_len(p, lane) : 0;
    unsigned grains = (len0 + ATT4_GRAIN - 1) / ATT4_GRAIN, longest = grains;
    for (int b = lane + 32; b < p.batch; b += 32) {
        const unsigned g = (kv4_len(p, b) + ATT4_GRAIN - 1) / ATT4_GRAIN;
        grains += g;
        longest = max(longest, g);
    }
    const unsigned long long total = (unsigned long long)__reduce_add_sync(0xffffffffu, grains) * units;
    // sum of ceil(g / size) <= total / size + sequences * units, which is at most `slots` for the first size.  Where the
    // units alone take most of the slots the second one is used, and up to a CTA per unit more than the GPU holds
    const bool once = p.slots - p.least_ctas > p.slots / 2;
    const auto shares = [&](unsigned n) { return total >> 31 ? (unsigned)((total + n - 1) / n) : ((unsigned)total + n - 1) / n; };
    unsigned even = shares(once ? p.slots - p.least_ctas : p.slots);
    // The smallest size (to 3 %) with which the CTAs still are all resident: chunks of 19 grains instead of 20 for 8 sequences of
    // 8191 .. 32768 positions, of 4 instead of 5 for 4 of 1501 .. 4001 with 24 units each (46.6 and 48.0 us, 19.9 and 21.9 us).
    // Where units take more than half of the slots, chunks of one round are larger and take 2 to 7 % longer than two rounds
    if (once && p.batch <= 32) {
        unsigned low = shares(p.slots);
        while (even - low > even / 32) {
            const unsigned mid = (low + even) / 2, c = lane < p.batch ? max((grains + mid - 1) / mid, 1u) : 0u;
            if (__reduce_add_sync(0xffffffffu, c) * units <= (unsigned)p.slots) even = mid;
            else low = mid + 1;
        }
    }
    // Sequences hardly longer than an even share stay whole: 16 sequences of 1020 positions and 32 KV heads, 8 grains of 7, take
    // 22.8 us, and 32 us with second chunks of one grain.  Otherwise a tile per warp is enough for a chunk (16 sequences of 641
    // positions and 8 KV heads: 12.6 us, in chunks of five 18); more than a round of them costs more than a second tile does (one
    // sequence of 8000: 12.4 us, and 11.3).  No larger than the cache: many units over a long one would take the products below
    // past 32 bits
    longest = __reduce_max_sync(0xffffffffu, longest);
    const unsigned least = 3 * longest <= 4 * even ? longest : longest > ATT4_ROUND ? 2 : 1;
    w.size = min(max(max(even, least), 1u), (unsigned)(p.lmax + ATT4_GRAIN - 1) / ATT4_GRAIN);
    int first = 0;  // running sum of CTAs over the sequences
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        const int b = b0 + lane, len = b0 == 0 ? len0 : b < p.batch ? kv4_len(p, b) : 0;
        const int c = b < p.batch ? max((int)((unsigned)(len + w.size * ATT4_GRAIN - 1) / (unsigned)(w.size * ATT4_GRAIN)), 1) : 0;
        int upto = c * units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += up;
        }
        const unsigned in = __ballot_sync(0xffffffffu, first + upto > (int)blockIdx.x);
        if (in) {
            const int at = __ffs(in) - 1, r = (int)blockIdx.x - first - __shfl_sync(0xffffffffu, upto, at) + __shfl_sync(0xffffffffu, c, at) * units;
            w.chunks = __shfl_sync(0xffffffffu, c, at);
            w.len = __shfl_sync(0xffffffffu, len, at);
            w.b = b0 + at; w.unit = r / w.chunks; w.chunk = r - w.unit * w.chunks;
            return true;
        }
        first += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;  // more CTAs than work
}

__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// x -> (hi, lo), two f16 terms of it
__device__ __forceinline__ uint32_t split_f16(float x) {
    const __half2 r = __floats2half2_rn(x, x - __half2float(__float2half_rn(x)));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; a result below 2^-126 is 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max_over_g(float x) {  // over the eight lanes of equal t
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float sum_over_g(float x) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint32_t *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const uint32_t *src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// W = 32-bit words of a row, a constant, so that every address inside a tile is one; NT = sets of four query rows
template <int W, int NT>
struct Attn4 {
    static constexpr int ROWS = ATT4_ROWS * NT;
    static constexpr int KC = (W + 3) / 4;      // words of a row per lane (4 lanes a row)
    static constexpr bool VEC = W % 4 == 0;     // lane t takes words KC t .., otherwise t, t + 4, ..
    static constexpr int NBK = (W + 7) / 8;     // blocks of 8 words = 64 dims = 4 tiles of 16 dims of the output
    // 64-byte rows meet in the same banks: rows 4a+2 and 4a+3 of K change places, 16-byte pieces of V are dealt over the banks
    static constexpr bool SWZ = W == 16;
    static constexpr int STAGE = 2 * ATT4_TILE * W + 2 * ATT4_TILE;  // words: K codes, V codes, K pairs, V pairs
    static constexpr int OLD = 64 * NBK + 4;    // row stride of the partial sums in shared memory
    static constexpr size_t RING = (size_t)ATT4_WARPS * ATT4_STAGES * STAGE * 4;
    static constexpr size_t JOINED = (size_t)ATT4_WARPS * ROWS * OLD * 4;
    static constexpr size_t SMEM = RING > JOINED ? RING : JOINED;
    __device__ static int k_word(int t, int c) { return VEC ? KC * t + c : t + 4 * c; }
    // word of output row g, block k
    __device__ static int v_word(int g, int k) { return SWZ ? 2 * g + k : g + 8 * k; }
};

template <int W, int NT>
__global__ void __launch_bounds__(ATT4_WARPS * 32, ATT4_PER_SM) attn_kv4_kernel(AttnParams p) {
    using A = Attn4<W, NT>;
    constexpr int KC = A::KC, NBK = A::NBK, ROWS = A::ROWS;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint4 s_q[NT][KC][32];  // query operands, in the order of the matrix instruction
    __shared__ float s_fr[ROWS], s_qs[ROWS];
    __shared__ float s_m[ATT4_WARPS][ROWS], s_l[ATT4_WARPS][ROWS];
    __shared__ long long s_row[ROWS];  // index of the tile's rows in q and out
    __shared__ int s_off[ROWS];        // positions behind the sequence's end that a row does not see
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rep = p.rep, hd = p.hd;
    pdl_release_and_wait();
    AttnWork work;
    if (!find_attn_work(p, work)) return;
    const int b = work.b, kvh = work.unit / p.row_tiles, len = work.len;
    const int r0 = (work.unit - kvh * p.row_tiles) * ROWS, rows = min(ROWS, p.t * rep - r0);  // rows: query token * rep + head of the group
    // index of a row in q and out, and the positions behind the sequence's end that it does not see
    auto row_of = [&](int r, int &off) {
        const int i = (r0 + r) / rep;
        off = p.t - 1 - i;
        return ((long long)b * p.t + i) * p.n_heads + kvh * rep + (r0 + r - i * rep);
    };
    // a warp takes NT query rows; their loads are under way first
    float x[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = warp + n * ATT4_WARPS;
        int off;
        const long long row = row_of(min(r, rows - 1), off);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = r < rows && lane + 32 * i < hd ? p.q[row * hd + lane + 32 * i] : 0.0f;
        if (lane == 0) {
            s_row[r] = row;
            s_off[r] = off;
        }
    }
    int last_off;
    row_of(rows - 1, last_off);
    const int last = len - last_off;  // positions the tile's last row sees: no row sees more
    const int c0 = work.chunk * work.size * ATT4_GRAIN, c1 = min(last, c0 + work.size * ATT4_GRAIN);
    if (p.slots && work.chunk == 0 && threadIdx.x == 0) p.part_of[((size_t)b * p.n_kv + kvh) * p.row_tiles + r0 / ROWS] = make_int2(blockIdx.x, work.chunks);

    // ---- ring of this warp
    uint32_t *ring = reinterpret_cast<uint32_t *>(smem) + warp * ATT4_STAGES * A::STAGE;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    const size_t base = ((size_t)b * p.n_kv + kvh) * p.lmax;
    const uint32_t *kc = p.k_codes + base * W, *vc = p.v_codes + base * W, *pairs = ((lane & 8) ? p.v_steps : p.k_steps) + base;
    // 16-byte pieces: piece i = lane + 32 j of a plane's 8 W.  SWZ: K's go to row r ^ (r / 2) % 2, V's change places inside
    // their row by (r / 4) % 4
    const int kdst = A::SWZ ? 16 * (lane ^ ((lane >> 1) & 4)) : 16 * lane;
    const int vdst[2] = {A::SWZ ? 16 * ((lane & ~3) | ((lane & 3) ^ (lane >> 4))) : 16 * lane,
                         A::SWZ ? 16 * ((lane & ~3) | ((lane & 3) ^ (lane >> 4) ^ 2)) : 16 * lane};
    auto issue = [&](int tile0, int stage) {
        const uint32_t dst = ring_at + stage * (A::STAGE * 4);
        if (tile0 + ATT4_TILE <= c1) {
            const uint32_t *ks = kc + (size_t)tile0 * W + 4 * lane, *vs = vc + (size_t)tile0 * W + 4 * lane;
#pragma unroll
            for (int j = 0; j < (8 * W + 31) / 32; ++j)
                if (32 * j + 31 < 8 * W || lane + 32 * j < 8 * W) {
                    copy16(dst + kdst + 512 * j, ks + 128 * j);
                    copy16(dst + ATT4_TILE * W * 4 + vdst[j & 1] + 512 * j, vs + 128 * j);
                }
            if (lane < 16) copy16(dst + 2 * ATT4_TILE * W * 4 + 16 * lane, pairs + tile0 + 4 * (lane & 7));
        } else if (tile0 < c1) {
            // the sequence ends inside: rows up to the next multiple of 4 exist (lmax is one), the rest is filled with zeros
            const int have = ((c1 + 3) & ~3) - tile0;
#pragma unroll
            for (int j = 0; j < (8 * W + 31) / 32; ++j)
                if (lane + 32 * j < 8 * W) {
                    const bool ok = 4 * (lane + 32 * j) < have * W;
                    const size_t off = (size_t)tile0 * W + (ok ? 4 * (lane + 32 * j) : 0);
                    copy16_or_zero(dst + kdst + 512 * j, kc + off, ok);
                    copy16_or_zero(dst + ATT4_TILE * W * 4 + vdst[j & 1] + 512 * j, vc + off, ok);
                }
            if (lane < 16) {
                const bool ok = 4 * (lane & 7) < have;
                copy16_or_zero(dst + 2 * ATT4_TILE * W * 4 + 16 * lane, pairs + tile0 + (ok ? 4 * (lane & 7) : 0), ok);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const int first = c0 + warp * ATT4_TILE, stride = ATT4_WARPS * ATT4_TILE;
#pragma unroll
    for (int s = 0; s < ATT4_STAGES - 1; ++s) issue(first + s * stride, s);

    // ---- queries times scale log2(e), scaled by a power of two to [2^13, 2^14), split, laid out
    static_assert(ATT4_ROWS == ATT4_WARPS, "a warp takes one row of each set");
#pragma unroll
    for (int m = 0; m < NT; ++m) {
        const int r = warp + m * ATT4_WARPS;
        const float unit2 = p.scale * 1.4426950408889634f;  // scores in units of log 2
        float amax = 0.0f, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[m][i] *= unit2;
            amax = fmaxf(amax, fabsf(x[m][i]));
            sum += x[m][i];
        }
        amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));  // not negative: ordered as integers
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        // by exponent fields; below 2^-113 the scores are 0 to any accuracy, from 2^120 on the row is given up (NaN)
        const int e = max((int)(__float_as_uint(amax) >> 23), 14);
        const float up = __int_as_float((267 - e) << 23);
        if (lane == 0) {
            s_fr[r] = __int_as_float(min(e + 7, 254) << 23);  // 2^20 / up
            s_qs[r] = e > 247 ? __uint_as_float(0x7fffffffu) : sum;
        }
        __half *dst = reinterpret_cast<__half *>(s_q[m]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 32 * i, w = d >> 3, n = d & 7;
            if (w >= 4 * KC) continue;
            const int tt = A::VEC ? w / KC : w & 3, c = A::VEC ? w % KC : w >> 2;
            const uint32_t y = split_f16(x[m][i] * up);
            // step (n & 2) / 2 of word c, register n & 1, half n / 4; column 2 warp holds hi, the next one lo
            __half *at = dst + ((size_t)c * 32 + warp * 8 + tt) * 8 + ((n >> 1) & 1) * 4 + (n & 1) * 2 + (n >> 2);
            at[0] = __ushort_as_half((unsigned short)(y & 0xffffu));
            at[32] = __ushort_as_half((unsigned short)(y >> 16));
        }
    }
    __syncthreads();
    const int least = min(c1, len - s_off[0]);  // the smallest limit of the tile's rows
    uint4 qf[KC];  // held in registers where they fit
    if (NT == 1) {
#pragma unroll
        for (int c = 0; c < KC; ++c) qf[c] = s_q[0][c][lane];
    }
    int end[NT];  // positions of the chunk that this lane's row sees
    float fr[NT], qs[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = 4 * n + t;
        end[n] = r < rows ? min(c1, len - s_off[r]) : 0;
        fr[n] = s_fr[r];
        qs[n] = s_qs[r];
    }

    float acc[NT][NBK][4][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < NBK; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) acc[n][k][j][i] = 0.0f;
    // of row t of each set: reference, sums over this lane's positions, the largest |weight * step| at the last rescaling, and
    // what weights are held times: 2^6 / 2^floor(log2 wref)
    float mref[NT], l[NT], alo[NT], wref[NT], ws[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) mref[n] = -INFINITY, l[n] = alo[n] = 0.0f, wref[n] = 0x1p-100f, ws[n] = 0x1p106f;
    // every second position counts down from its largest value, lo + 15 step - (15 - c) step: the sums of the products and of
    // the constant parts then change sign as the values do.  With codes alone they only grow, and the instruction's truncated
    // adds pull all of it one way (2.8e-4 of the result at 32768 positions).  Odd lanes g count down in block 0, even ones in
    // block 1, so that every lane does both
    const float down[2] = {g & 1 ? 15.0f : 0.0f, g & 1 ? 0.0f : 15.0f}, sign = g & 1 ? -1.0f : 1.0f;

    int stage = 0;
    for (int tile0 = first; tile0 < c1; tile0 += stride) {
        asm volatile("cp.async.wait_group %0;" ::"n"(ATT4_STAGES - 2) : "memory");
        __syncwarp();  // this tile has landed for every lane, and every lane is done with the stage that is filled next
        issue(tile0 + (ATT4_STAGES - 1) * stride, stage == 0 ? ATT4_STAGES - 1 : stage - 1);
        const uint32_t *sk = ring + stage * A::STAGE, *sv = sk + ATT4_TILE * W, *sp = sv + ATT4_TILE * W;
        stage = stage + 1 == ATT4_STAGES ? 0 : stage + 1;

        // ---- scores: block h holds positions 16 h + 2 g (rows g of its tile) and 16 h + 2 g + 1 (rows g + 8)
        float s[NT][2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t kw[2][KC];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t *row = sk + (16 * h + (A::SWZ ? (2 * g + i) ^ (g & 1) : 2 * g + i)) * W + A::k_word(t, 0);
                if (A::VEC && KC == 4) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(row);
                    kw[i][0] = v.x; kw[i][1 % KC] = v.y; kw[i][2 % KC] = v.z; kw[i][3 % KC] = v.w;
                } else if (A::VEC && KC == 2) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(row);
                    kw[i][0] = v.x; kw[i][1 % KC] = v.y;
                } else {
#pragma unroll
                    for (int c = 0; c < KC; ++c) kw[i][c] = A::VEC || 4 * c + 3 < W || t + 4 * c < W ? row[A::VEC ? c : 4 * c] : 0u;
                }
            }
            float sc[NT][4];
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const uint32_t x = kw[0][c], y = kw[1][c];
                const uint32_t a[4] = {(x << 4) & 0x00f000f0u, (y << 4) & 0x00f000f0u, x & 0x00f000f0u, y & 0x00f000f0u};
                const uint32_t x8 = x >> 8, y8 = y >> 8;
                const uint32_t a8[4] = {(x8 << 4) & 0x00f000f0u, (y8 << 4) & 0x00f000f0u, x8 & 0x00f000f0u, y8 & 0x00f000f0u};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint4 q = NT == 1 ? qf[c] : s_q[n][c][lane];
                    if (c == 0) mma_f16_first(sc[n], a[0], a[1], a[2], a[3], q.x, q.y);
                    else mma_f16(sc[n], a[0], a[1], a[2], a[3], q.x, q.y);
                    mma_f16(sc[n], a8[0], a8[1], a8[2], a8[3], q.z, q.w);
                }
            }
            const uint2 kp = *reinterpret_cast<const uint2 *>(sp + 16 * h + 2 * g);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s[n][h][0] = fmaf(sc[n][0] + sc[n][1], kv4_step(kp.x) * fr[n], kv4_lo(kp.x) * qs[n]);
                s[n][h][1] = fmaf(sc[n][2] + sc[n][3], kv4_step(kp.y) * fr[n], kv4_lo(kp.y) * qs[n]);
            }
        }
        const bool tail = tile0 + ATT4_TILE > least;  // some row does not see all of the tile
        if (tail) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (tile0 + 16 * h + 2 * g + i >= end[n]) s[n][h][i] = -INFINITY;
        }
        // ---- softmax weights
        float top[NT], corr[NT];
        bool rise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            top[n] = fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][1][0], s[n][1][1]));
            rise |= top[n] > mref[n] + ATT4_SLACK;
            corr[n] = 1.0f;
        }
        const bool fresh = __any_sync(0xffffffffu, rise);
        if (fresh) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float m = fmaxf(mref[n], max_over_g(top[n]));
                corr[n] = m == -INFINITY ? 1.0f : exp2_fast(mref[n] - m);
                mref[n] = m;
                l[n] *= corr[n];
                alo[n] *= corr[n];
                wref[n] = fmaxf(wref[n] * corr[n], 0x1p-100f);
            }
        }
        uint2 vp[2];
        vp[0] = *reinterpret_cast<const uint2 *>(sp + ATT4_TILE + 2 * g);
        vp[1] = *reinterpret_cast<const uint2 *>(sp + ATT4_TILE + 16 + 2 * g);
        float wmax[NT];
        bool large = fresh;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float ref = mref[n] == -INFINITY ? 0.0f : mref[n];  // nothing seen yet: every weight is 0
            wmax[n] = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t pr = i ? vp[h].y : vp[h].x;
                    if (tail) pr = s[n][h][i] == -INFINITY ? 0u : pr;  // what is not seen may hold anything, NaN too
                    const float pj = exp2_fast(s[n][h][i] - ref), step = kv4_step(pr);
                    l[n] += pj;
                    alo[n] = fmaf(pj, fmaf(down[h], step, kv4_lo(pr)), alo[n]);
                    s[n][h][i] = pj * step;
                    wmax[n] = fmaxf(wmax[n], s[n][h][i]);
                }
            large |= wmax[n] * ws[n] > 0x1p15f;
        }
        if (__any_sync(0xffffffffu, large)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                wref[n] = fminf(fmaxf(wref[n], max_over_g(wmax[n])), 0x1p127f);
                const float ws_new = __uint_as_float(0x82000000u - (__float_as_uint(wref[n]) & 0x7f800000u));  // by exponent fields
                const float adj = corr[n] * fminf(__fdividef(ws_new, ws[n]), 0x1p127f);  // a ratio of powers of two; corr may be 0
                ws[n] = ws_new;
#pragma unroll
                for (int k = 0; k < NBK; ++k)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) acc[n][k][j][i] *= adj;
            }
        }
        // ---- weighted sum of the codes
        const uint32_t *vrow = sv + 4 * t * W + (A::SWZ ? 4 * ((g >> 1) ^ t) + 2 * (g & 1) : g);
        uint32_t vw[2][NBK][4], b0[2][NT], b1[2][NT];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t *row = vrow + (16 * h + i) * W;
                if (A::SWZ) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(row);
                    vw[h][0][i] = v.x;
                    vw[h][NBK - 1][i] = v.y;
                } else {
#pragma unroll
                    for (int k = 0; k < NBK; ++k) vw[h][k][i] = 8 * k + 7 < W || g + 8 * k < W ? row[8 * k] : 0u;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float f = h == 0 ? ws[n] * sign : -(ws[n] * sign);
                b0[h][n] = transpose_8x8(split_f16(s[n][h][0] * f));  // positions 4t and 4t + 2 of column g
                b1[h][n] = transpose_8x8(split_f16(s[n][h][1] * f));  // positions 4t + 1 and 4t + 3
            }
        }
        // a tile's sums start from zero and are added by rounding: left in the instruction's accumulators they would shrink
        // by up to 2^-23 with every step
#pragma unroll
        for (int k = 0; k < NBK; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // byte j of the words: dims 2j (rows g) and 2j + 1 (rows g + 8)
                const uint32_t sel = 0x4400u + 0x1111u * j;
                float part[NT][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    auto code = [&](uint32_t x) {  // of two positions, one counted down: (x & mask) ^ half of it in one instruction
                        uint32_t y;
                        asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(y) : "r"(x), "r"(0x00f000f0u), "r"(h == 0 ? 0x00f00000u : 0x000000f0u));
                        return y;
                    };
                    const uint32_t x = __byte_perm(vw[h][k][0], vw[h][k][2], sel), y = __byte_perm(vw[h][k][1], vw[h][k][3], sel);
                    const uint32_t a0 = code(x << 4), a1 = code(x), a2 = code(y << 4), a3 = code(y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (h == 0) mma_f16_first(part[n], a0, a1, a2, a3, b0[h][n], b1[h][n]);
                        else mma_f16(part[n], a0, a1, a2, a3, b0[h][n], b1[h][n]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) acc[n][k][j][i] += part[n][2 * i] + part[n][2 * i + 1];
            }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    // ---- join the warps: sums of a row over its eight lanes, then rows over the warps through shared memory
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l[n] = sum_over_g(l[n]);
        alo[n] = sum_over_g(alo[n]);
        if (g == 0) {
            s_m[warp][4 * n + t] = mref[n];
            s_l[warp][4 * n + t] = l[n];
        }
    }
    __syncthreads();  // every warp is done with its ring
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float *so = reinterpret_cast<float *>(smem) + (warp * ROWS + 4 * n + t) * A::OLD;
        // 2^20 / ws in two factors: from weights times steps of 2^114 on their product leaves f32 where the sums do not
        const float back = __uint_as_float(0x82000000u - __float_as_uint(ws[n]));  // 2^6 / ws
#pragma unroll
        for (int k = 0; k < NBK; ++k) {
            float4 *dst = reinterpret_cast<float4 *>(so + 8 * A::v_word(g, k));
#pragma unroll
            for (int j = 0; j < 4; j += 2)
                dst[j / 2] = make_float4(fmaf(acc[n][k][j][0] * 0x1p14f, back, alo[n]), fmaf(acc[n][k][j][1] * 0x1p14f, back, alo[n]),
                                         fmaf(acc[n][k][j + 1][0] * 0x1p14f, back, alo[n]), fmaf(acc[n][k][j + 1][1] * 0x1p14f, back, alo[n]));
        }
    }
    __syncthreads();
    static_assert(KV4_MAX_HD <= ATT4_WARPS * 32, "a thread takes one dim");
    const int d = threadIdx.x;
    if (d >= hd) return;
    for (int r = 0; r < rows; ++r) {
        float m = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < ATT4_WARPS; ++w) m = fmaxf(m, s_m[w][r]);
#pragma unroll
        for (int w = 0; w < ATT4_WARPS; ++w) {
            const float f = s_l[w][r] == 0.0f ? 0.0f : exp2_fast(s_m[w][r] - m);  // a warp that saw nothing of the row
            sum = fmaf(s_l[w][r], f, sum);
            o = fmaf(reinterpret_cast<const float *>(smem)[(w * ROWS + r) * A::OLD + d], f, o);
        }
        if (work.chunks == 1) {
            p.out[s_row[r] * hd + d] = sum == 0.0f ? 0.0f : __fdiv_rn(o, sum);
        } else {
            const size_t at = (size_t)blockIdx.x * ROWS + r;
            p.part[at * hd + d] = o;
            if (d == 0) p.part_ml[at] = make_float2(m, sum);
        }
    }
}

template <int W>
static int launch_attn_kv4(const AttnParams &p, unsigned ctas, int dev, cudaStream_t stream) {
    if (p.words != W) {
        if constexpr (W > 1) return launch_attn_kv4<W - 1>(p, ctas, dev, stream);
        return fail(KB_ERR_UNSUPPORTED, "attention: rows of %d words", p.words);
    }
    const bool one = p.tile_rows == ATT4_ROWS;
    void (*kern)(AttnParams) = one ? attn_kv4_kernel<W, 1> : attn_kv4_kernel<W, 2>;
    const size_t smem = one ? Attn4<W, 1>::SMEM : Attn4<W, 2>::SMEM;
    if (int rc = set_dyn_smem_once(reinterpret_cast<const void *>(kern), dev, (int)smem, "kv4 attention smem attribute")) return rc;
    const cudaError_t e = launch_pdl(kern, dim3(ctas), dim3(ATT4_WARPS * 32), smem, stream, p);
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "kv4 attention launch");
}

// One CTA per query row: the weighted mean of its chunks where there are several, a thread per dim.  A round takes 32 chunks,
// a lane's factor each; the first sums are on their way while the factors are worked out.
__global__ void __launch_bounds__(KV4_MAX_HD) attn_kv4_join_kernel(AttnParams p) {
    const unsigned row = blockIdx.x, tok = row / p.n_heads;
    const int lane = threadIdx.x & 31, d = threadIdx.x, h = row - tok * p.n_heads, b = tok / p.t, i = tok - b * p.t;
    const int kvh = h / p.rep, r = i * p.rep + h - kvh * p.rep, tile = r / p.tile_rows;
    pdl_release_and_wait();
    const int2 of = p.part_of[((size_t)b * p.n_kv + kvh) * p.row_tiles + tile];
    const int n = of.y;
    if (n == 1) return;  // the first kernel wrote it
    const size_t stride = p.tile_rows, at = (size_t)of.x * stride + (r - tile * p.tile_rows);
    const float2 *ml = p.part_ml + at;
    const float *src = p.part + at * p.hd + (d < p.hd ? d : 0);
    constexpr int FIRST = 16;
    float x[FIRST];
    float2 v = lane < n ? ml[lane * stride] : make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int k = 0; k < FIRST; ++k) x[k] = k < n ? src[k * stride * p.hd] : 0.0f;
    float top = v.x, sum = 0.0f, o = 0.0f;
    for (int s = 32 + lane; s < n; s += 32) top = fmaxf(top, ml[s * stride].x);
    top = warp_reduce_max(top);
    for (int s0 = 0; s0 < n; s0 += 32) {
        if (s0) v = s0 + lane < n ? ml[(s0 + lane) * stride] : make_float2(0.0f, 0.0f);
        const float mine = v.y == 0.0f ? 0.0f : exp2_fast(v.x - top);
        sum = fmaf(v.y, mine, sum);
        const int m = min(32, n - s0);
        for (int s = 0; s < m; s += FIRST) {
            if (s0 + s) {
#pragma unroll
                for (int k = 0; k < FIRST; ++k) x[k] = s + k < m ? src[(s0 + s + k) * stride * p.hd] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < FIRST; ++k) o = fmaf(x[k], __shfl_sync(0xffffffffu, mine, s + k), o);
        }
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (d < p.hd) p.out[(size_t)row * p.hd + d] = sum == 0.0f ? 0.0f : __fdiv_rn(o, sum);
}

static int check_kv4(int n_heads, int n_kv, int hd, int lmax) {
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv) return fail(KB_ERR_INVALID, "kv4: %d heads over %d KV heads", n_heads, n_kv);
    if (hd < 4 || hd > KV4_MAX_HD || hd % 4) return fail(KB_ERR_UNSUPPORTED, "kv4: head_dim %d must be a multiple of 4 up to %d", hd, KV4_MAX_HD);
    if (lmax < 4 || lmax % 4 || lmax > KV4_MAX_LEN) return fail(KB_ERR_UNSUPPORTED, "kv4: cache length %d must be a multiple of 4 up to %d", lmax, KV4_MAX_LEN);
    return KB_OK;
}

// query rows of a CTA: one set of columns where it holds them all
static int attn_tile_rows(int t, int n_heads, int n_kv) { return (size_t)t * (n_heads / n_kv) <= ATT4_ROWS ? ATT4_ROWS : 2 * ATT4_ROWS; }

// How a call is launched: CTAs, and the workspace of its chunks.  The lengths are on the device; a cache that could not make
// two chunks of a sequence is not split, nor a call of so many units that a long one among short ones hardly shows.
struct AttnPlan {
    int tile_rows, row_tiles, slots;
    size_t units, ctas;
    size_t of_bytes, ml_bytes, part_bytes;
    size_t bytes() const { return of_bytes + ml_bytes + part_bytes; }
};
static AttnPlan attn_plan(size_t batch, int t, int n_heads, int n_kv, int hd, int lmax, int sms) {
    AttnPlan a = {};
    a.tile_rows = attn_tile_rows(t, n_heads, n_kv);
    a.row_tiles = (int)(((size_t)t * (n_heads / n_kv) + a.tile_rows - 1) / a.tile_rows);
    a.units = batch * n_kv * a.row_tiles;
    a.slots = sms * ATT4_PER_SM;
    if (lmax <= (a.units < ATT4_MANY ? ATT4_WHOLE : ATT4_WHOLE + 2) * ATT4_GRAIN || a.units > (size_t)16 * a.slots) a.slots = 0;
    a.ctas = a.slots == 0 ? a.units : a.units * 2 < (size_t)a.slots ? (size_t)a.slots : a.units + a.slots;  // see find_attn_work
    if (a.slots) {
        auto up = [](size_t v) { return (v + 255) / 256 * 256; };
        a.of_bytes = up(a.units * sizeof(int2));
        a.ml_bytes = up(a.ctas * a.tile_rows * sizeof(float2));
        a.part_bytes = a.ctas * a.tile_rows * (size_t)hd * sizeof(float);
    }
    return a;
}

static bool aligned16(const void *a, const void *b = nullptr, const void *c = nullptr, const void *d = nullptr) {
    return !((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15);
}

// blocks of 8 warps for `rows * groups` warps
static int warp_grid(size_t rows, size_t groups, unsigned *tasks, unsigned *grid) {
    if (rows > 0x7fffffffu || groups > 0x7fffffffu || rows * groups > 0x7fffffffu) return fail(KB_ERR_UNSUPPORTED, "%zu rows of %zu head groups in one call", rows, groups);
    *tasks = (unsigned)(rows * groups);
    *grid = (*tasks + 7) / 8;
    return KB_OK;
}

static int append(AppendParams &p, bool q4, size_t n, size_t max_pos, size_t n_seqs, kb_stream stream) {
    const size_t heads = (size_t)p.n_heads + 2 * (size_t)p.n_kv;
    if (p.ld == 0) p.ld = heads * p.hd;
    if (p.ld < heads * p.hd) return fail(KB_ERR_INVALID, "append: row stride %zu below %zu", p.ld, heads * p.hd);
    if (!(p.eps >= 0.0f)) return fail(KB_ERR_INVALID, "append: eps must not be negative");
    if (n == 0) return KB_OK;
    if (n > 0x7fffffffu || heads > 0xffffffu || max_pos > 0x7fffffffu || n_seqs > 0x7fffffffu)
        return fail(KB_ERR_UNSUPPORTED, "append: %zu tokens of %zu heads, %zu sequences", n, heads, n_seqs);
    p.max_pos = (int)max_pos;
    p.cache_len = (long long)n_seqs * p.lmax;
    p.per_dim = 1.0 / p.hd;
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.qkv) | reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t) |
                          reinterpret_cast<uintptr_t>(p.q_gamma) | reinterpret_cast<uintptr_t>(p.k_gamma) | reinterpret_cast<uintptr_t>(p.q_out) |
                          reinterpret_cast<uintptr_t>(p.k_cache) | reinterpret_cast<uintptr_t>(p.v_cache);
    const bool pairs = p.hd % 4 == 0 && p.ld % 2 == 0 && all % 8 == 0;
    // one head per warp while that leaves warps to spare (16 per SM), four for many tokens
    int dev = 0;
    KB_CUDA(cudaGetDevice(&dev));
    const bool many = n * heads > (size_t)sm_count(dev) * 16;
    p.groups = (unsigned)(many ? (heads + 3) / 4 : heads);
    unsigned grid = 0;
    if (int rc = warp_grid(n, p.groups, &p.tasks, &grid)) return rc;
    void (*kern)(AppendParams) =
        q4 ? (many ? (pairs ? (p.hd == 128 ? append_kernel<true, 4, true, true> : append_kernel<true, 4, true>) : append_kernel<true, 4, false>) : (pairs ? append_kernel<true, 1, true> : append_kernel<true, 1, false>))
           : (many ? (pairs ? (p.hd == 128 ? append_kernel<false, 4, true, true> : append_kernel<false, 4, true>) : append_kernel<false, 4, false>) : (pairs ? append_kernel<false, 1, true> : append_kernel<false, 1, false>));
    const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream), p);
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "append launch");
}

}  // namespace kb

using namespace kb;

extern "C" {

size_t kb_kv4_row_words(int head_dim) { return head_dim < 1 ? 0 : (size_t)kv4_words(head_dim); }

int kb_qknorm_rope_kv(const float *qkv, size_t ld, const int *positions, const long long *cache_rows, const float *cos_table,
                      const float *sin_table, size_t max_pos, const float *q_gamma, const float *k_gamma, float eps, size_t n,
                      int n_heads, int n_kv_heads, int head_dim, size_t n_seqs, int lmax, float *q_out, float *k_cache,
                      float *v_cache, kb_stream stream) {
    if (!qkv || !positions || !cache_rows || !cos_table || !sin_table || !q_out || !k_cache || !v_cache)
        return fail(KB_ERR_INVALID, "null pointer");
    if (n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads) return fail(KB_ERR_INVALID, "append: %d heads over %d KV heads", n_heads, n_kv_heads);
    if (head_dim < 2 || head_dim > KV4_MAX_HD || head_dim % 2)
        return fail(KB_ERR_UNSUPPORTED, "append: head_dim %d must be even, up to %d", head_dim, KV4_MAX_HD);
    if (lmax < 1) return fail(KB_ERR_INVALID, "append: cache length %d", lmax);
    AppendParams p = {};
    p.qkv = qkv; p.ld = ld; p.positions = positions; p.cache_rows = cache_rows; p.cos_t = cos_table; p.sin_t = sin_table;
    p.q_gamma = q_gamma; p.k_gamma = k_gamma; p.eps = eps; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.hd = head_dim; p.lmax = lmax;
    p.q_out = q_out; p.k_cache = k_cache; p.v_cache = v_cache;
    return append(p, false, n, max_pos, n_seqs, stream);
}

int kb_qknorm_rope_kv4(const float *qkv, size_t ld, const int *positions, const long long *cache_rows, const float *cos_table,
                       const float *sin_table, size_t max_pos, const float *q_gamma, const float *k_gamma, float eps, size_t n,
                       int n_heads, int n_kv_heads, int head_dim, size_t n_seqs, int lmax, float *q_out, uint32_t *k_codes,
                       uint32_t *k_steps, uint32_t *v_codes, uint32_t *v_steps, kb_stream stream) {
    if (!qkv || !positions || !cache_rows || !cos_table || !sin_table || !q_out || !k_codes || !k_steps || !v_codes || !v_steps)
        return fail(KB_ERR_INVALID, "null pointer");
    if (int rc = check_kv4(n_heads, n_kv_heads, head_dim, lmax)) return rc;
    if (!aligned16(k_codes, k_steps, v_codes, v_steps)) return fail(KB_ERR_INVALID, "kv4: planes must be 16-byte aligned");
    AppendParams p = {};
    p.qkv = qkv; p.ld = ld; p.positions = positions; p.cache_rows = cache_rows; p.cos_t = cos_table; p.sin_t = sin_table;
    p.q_gamma = q_gamma; p.k_gamma = k_gamma; p.eps = eps; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.hd = head_dim; p.lmax = lmax;
    p.q_out = q_out; p.k_codes = k_codes; p.k_steps = k_steps; p.v_codes = v_codes; p.v_steps = v_steps;
    return append(p, true, n, max_pos, n_seqs, stream);
}

int kb_kv4_read(const uint32_t *k_codes, const uint32_t *k_steps, const uint32_t *v_codes, const uint32_t *v_steps,
                const long long *cache_rows, size_t n, int n_kv_heads, int head_dim, size_t n_seqs, int lmax, float *k_out,
                float *v_out, kb_stream stream) {
    if (!cache_rows || (!k_out && !v_out) || (k_out && (!k_codes || !k_steps)) || (v_out && (!v_codes || !v_steps)))
        return fail(KB_ERR_INVALID, "null pointer");
    if (int rc = check_kv4(n_kv_heads, n_kv_heads, head_dim, lmax)) return rc;
    if (!aligned16(k_codes, k_steps, v_codes, v_steps) || !aligned16(k_out, v_out))
        return fail(KB_ERR_INVALID, "kv4: planes and outputs must be 16-byte aligned");
    if (n == 0) return KB_OK;
    if (n_seqs > 0x7fffffffu) return fail(KB_ERR_UNSUPPORTED, "kv4: %zu sequences", n_seqs);
    unsigned tasks = 0, grid = 0;
    const unsigned groups = (unsigned)(n_kv_heads + READ_HEADS - 1) / READ_HEADS;
    if (int rc = warp_grid(n, groups, &tasks, &grid)) return rc;
    const cudaError_t e = launch_pdl(kv4_read_kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream), k_codes, k_steps, v_codes,
                                       v_steps, cache_rows, tasks, groups, n_kv_heads, head_dim, (long long)n_seqs * lmax, lmax, k_out, v_out);
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "kv4 read launch");
}

size_t kb_attn_kv4_workspace_bytes(size_t batch, int t, int n_heads, int n_kv_heads, int head_dim, int lmax) {
    int dev = 0;
    if (batch == 0 || t < 1 || check_kv4(n_heads, n_kv_heads, head_dim, lmax) != KB_OK || cudaGetDevice(&dev) != cudaSuccess) return 0;
    return attn_plan(batch, t, n_heads, n_kv_heads, head_dim, lmax, sm_count(dev)).bytes();
}

int kb_attn_kv4(const float *q, const uint32_t *k_codes, const uint32_t *k_steps, const uint32_t *v_codes, const uint32_t *v_steps,
                const int *lens, size_t batch, int t, int n_heads, int n_kv_heads, int head_dim, int lmax, float scale, float *out,
                void *workspace, size_t workspace_bytes, kb_stream stream) {
    if (!q || !k_codes || !k_steps || !v_codes || !v_steps || !lens || !out) return fail(KB_ERR_INVALID, "null pointer");
    if (int rc = check_kv4(n_heads, n_kv_heads, head_dim, lmax)) return rc;
    if (t < 0) return fail(KB_ERR_INVALID, "attention: %d query tokens", t);
    if (!(fabsf(scale) < INFINITY)) return fail(KB_ERR_INVALID, "attention: scale must be finite");
    if (!aligned16(k_codes, k_steps, v_codes, v_steps) || !aligned16(workspace))
        return fail(KB_ERR_INVALID, "kv4: planes and workspace must be 16-byte aligned");
    if (batch == 0 || t == 0) return KB_OK;
    if (batch > 0x7fffffffu || batch * (size_t)t * n_heads > 0x7fffffffu || (size_t)t * n_heads > 0x7fffffffu)
        return fail(KB_ERR_UNSUPPORTED, "attention: %zu sequences of %d tokens", batch, t);
    int dev = 0;
    KB_CUDA(cudaGetDevice(&dev));
    const AttnPlan plan = attn_plan(batch, t, n_heads, n_kv_heads, head_dim, lmax, sm_count(dev));
    if (plan.ctas > 0x7fffffffu) return fail(KB_ERR_UNSUPPORTED, "attention: %zu sequences of %d tokens", batch, t);
    const size_t rows = batch * (size_t)t * n_heads;
    AttnParams p = {};
    p.q = q; p.k_codes = k_codes; p.k_steps = k_steps; p.v_codes = v_codes; p.v_steps = v_steps; p.lens = lens;
    p.t = t; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.rep = n_heads / n_kv_heads; p.hd = head_dim; p.lmax = lmax; p.words = kv4_words(head_dim); p.out = out;
    p.scale = scale != 0.0f ? scale : 1.0f / sqrtf((float)head_dim);
    p.least_ctas = plan.units < (size_t)plan.slots ? (int)plan.units : plan.slots;
    p.batch = (int)batch; p.row_tiles = plan.row_tiles; p.tile_rows = plan.tile_rows; p.slots = plan.slots;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    void *own = nullptr;
    if (plan.slots) {
        if (workspace && workspace_bytes < plan.bytes())
            return fail(KB_ERR_STORAGE, "workspace too small: need %zu bytes, got %zu", plan.bytes(), workspace_bytes);
        if (!workspace) {
            KB_CUDA(cudaMallocAsync(&own, plan.bytes(), st));
            workspace = own;
        }
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        p.part_of = reinterpret_cast<int2 *>(ws);
        p.part_ml = reinterpret_cast<float2 *>(ws + plan.of_bytes);
        p.part = reinterpret_cast<float *>(ws + plan.of_bytes + plan.ml_bytes);
    }
    int rc = launch_attn_kv4<KV4_MAX_HD / 8>(p, (unsigned)plan.ctas, dev, st);
    if (rc == KB_OK && plan.slots) {
        const cudaError_t e = launch_pdl(attn_kv4_join_kernel, dim3((unsigned)rows), dim3(KV4_MAX_HD), 0, st, p);
        if (e != cudaSuccess) rc = cuda_fail(e, "kv4 attention join launch");
    }
    if (own) {
        const cudaError_t e = cudaFreeAsync(own, st);
        if (rc == KB_OK && e != cudaSuccess) rc = cuda_fail(e, "cudaFreeAsync");
    }
    return rc;
}

}  // extern "C"
