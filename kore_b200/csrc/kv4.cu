// A KV cache held in 4 bits: append (with the norms of queries and keys and the rotation), read-back, attention (sm_100a).
//
// Layout and arithmetic are those of include/kore_b200.h: one row per (sequence, KV head, position), 4-bit codes in
// natural dim order (dim 8w + i in bits 4i .. 4i+3 of word w) and one word (bfloat16 step | bfloat16 lo << 16); a code c
// stands for lo + c * step.  One pair per row keeps the unpacking out of the products: a score is
//     step_j * sum_d(q_d c_jd) + lo_j * sum_d(q_d)      and an output      sum_j (p_j step_j) c_jd + sum_j p_j lo_j,
// so both contractions run on bare codes and the pair touches one number per (query, position).
#include <stdlib.h>

#include "common.cuh"
#include "device_utils.cuh"

namespace kb {

constexpr int KV4_MAX_HD = 128;

__host__ __device__ inline int kv4_words(int hd) { return (hd + 7) / 8; }

__device__ __forceinline__ float kv4_step(uint32_t s) { return __uint_as_float(s << 16); }
__device__ __forceinline__ float kv4_lo(uint32_t s) { return __uint_as_float(s & 0xffff0000u); }

template <typename... KArgs, typename... Args>
static cudaError_t launch_after(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    static const bool pdl = [] {
        const char *v = getenv("KB_GEMV_PDL");
        return !(v && *v == '0');
    }();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, KArgs(args)...);
}

// as in decoder_ops.cu: inputs that an earlier kernel of the step writes are plain pointers, read after this
__device__ __forceinline__ void release_and_wait() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- norm + rotation + append ------------------------------------------------------------------
struct AppendParams {
    const float *qkv;
    size_t ld;
    const int *positions;
    const long long *cache_rows;
    const float *cos_t, *sin_t;
    long long max_pos;
    const float *q_gamma, *k_gamma;
    float eps;
    long long tasks;  // tokens * (n_heads + 2 n_kv)
    int n_heads, n_kv, hd;
    long long cache_len;  // n_seqs * lmax
    int lmax;
    float *q_out, *k_cache, *v_cache;
    uint32_t *k_codes, *k_steps, *v_codes, *v_steps;
};

// x >= 0 or x < 0, finite: the bfloat16 at or below x, and (x >= 0) the one at or above it
__device__ __forceinline__ float bf16_below(float x) {
    const uint32_t i = __float_as_uint(x), cut = i & 0xffff0000u;
    return __uint_as_float(x < 0.0f && i != cut ? cut + 0x10000u : cut);
}
__device__ __forceinline__ float bf16_above_nonneg(float x) {
    const uint32_t i = __float_as_uint(x), cut = i & 0xffff0000u;
    return __uint_as_float(i != cut ? cut + 0x10000u : cut);
}

// A warp takes one head of one token.  Lane l owns the rotation pairs 2l and 2l + 1, dims {2l, 2l + 1} of each half:
// its codes are then whole bytes of the row, and a row needs no shared memory.
template <bool Q4>
__global__ void __launch_bounds__(256) append_kernel(AppendParams p) {
    const int lane = threadIdx.x & 31;
    const long long task = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    release_and_wait();
    if (task >= p.tasks) return;
    const int heads = p.n_heads + 2 * p.n_kv, hd = p.hd, half = hd / 2;
    const long long t = task / heads;
    const int head = (int)(task - t * heads);
    const bool is_q = head < p.n_heads, is_v = head >= p.n_heads + p.n_kv;
    const long long pos = p.positions[t];
    const bool pos_ok = pos >= 0 && pos < p.max_pos;
    const long long crow = p.cache_rows[t];
    if (!is_q && (!pos_ok || crow < 0 || crow >= p.cache_len)) return;  // not appended
    const float *row = p.qkv + (size_t)t * p.ld + (size_t)head * hd;
    const int i0 = 2 * lane;
    const bool own0 = i0 < half, own1 = i0 + 1 < half;
    float a[2] = {own0 ? row[i0] : 0.0f, own1 ? row[i0 + 1] : 0.0f};
    float b[2] = {own0 ? row[half + i0] : 0.0f, own1 ? row[half + i0 + 1] : 0.0f};
    const float *gamma = is_q ? p.q_gamma : p.k_gamma;
    if (!is_v && gamma) {
        double ss = 0.0;  // f64: the order of the sum then cannot move a rounding of inv, so codes do not depend on it
#pragma unroll
        for (int i = 0; i < 2; ++i) ss += (double)a[i] * a[i] + (double)b[i] * b[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = (float)(1.0 / sqrt(ss / hd + (double)p.eps));
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i0 + i < half) {
                a[i] = __fmul_rn(__fmul_rn(a[i], inv), gamma[i0 + i]);
                b[i] = __fmul_rn(__fmul_rn(b[i], inv), gamma[half + i0 + i]);
            }
    }
    if (!is_v && pos_ok) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i0 + i < half) {
                const float c = p.cos_t[(size_t)pos * half + i0 + i], s = p.sin_t[(size_t)pos * half + i0 + i];
                const float x = a[i], y = b[i];
                a[i] = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
                b[i] = __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c));
            }
    }
    if (is_q) {
        float *q = p.q_out + ((size_t)t * p.n_heads + head) * hd;
        const float bad = __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i0 + i < half) {
                q[i0 + i] = pos_ok ? a[i] : bad;
                q[half + i0 + i] = pos_ok ? b[i] : bad;
            }
        return;
    }
    const int kvh = is_v ? head - p.n_heads - p.n_kv : head - p.n_heads;
    const size_t crow_head = ((size_t)(crow / p.lmax) * p.n_kv + kvh) * p.lmax + (size_t)(crow % p.lmax);
    if (!Q4) {
        float *dst = (is_v ? p.v_cache : p.k_cache) + crow_head * hd;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i0 + i < half) {
                dst[i0 + i] = a[i];
                dst[half + i0 + i] = b[i];
            }
        return;
    }
    // hd is a multiple of 4 here, so a lane owns both of its pairs or none
    float mn = own0 ? fminf(fminf(a[0], a[1]), fminf(b[0], b[1])) : INFINITY;
    float mx = own0 ? fmaxf(fmaxf(a[0], a[1]), fmaxf(b[0], b[1])) : -INFINITY;
    const float big = fmaxf(fmaxf(fabsf(a[0]), fabsf(a[1])), fmaxf(fabsf(b[0]), fabsf(b[1])));
    const bool nan = a[0] != a[0] || a[1] != a[1] || b[0] != b[0] || b[1] != b[1];  // fmaxf passes over them
    const bool broken = __any_sync(0xffffffffu, own0 && (nan || big == INFINITY));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    const float lo = bf16_below(mn);
    const float step = bf16_above_nonneg(fmaxf(__fdiv_rn(__fsub_rn(mx, lo), 15.0f), 0x1p-100f));
    const bool ok = !broken && fabsf(lo) < INFINITY && step < INFINITY;
    const float inv = __frcp_rn(step);
    auto code = [&](float x) {
        const int c = ok ? __float2int_rn(__fmul_rn(__fsub_rn(x, lo), inv)) : 0;
        return (uint32_t)max(0, min(15, c));
    };
    const int words = kv4_words(hd);
    uint8_t *bytes = reinterpret_cast<uint8_t *>((is_v ? p.v_codes : p.k_codes) + crow_head * words);
    if (own0) {
        bytes[lane] = (uint8_t)(code(a[0]) | code(a[1]) << 4);
        bytes[half / 2 + lane] = (uint8_t)(code(b[0]) | code(b[1]) << 4);
    }
    if (lane < 4 * words - half) bytes[half + lane] = 0;  // tail of the last word
    if (lane == 0)
        (is_v ? p.v_steps : p.k_steps)[crow_head] = ok ? (__float_as_uint(lo) | __float_as_uint(step) >> 16) : 0x7fc07fc0u;
}

// ---- read-back ---------------------------------------------------------------------------------
// A warp takes one head of one row: lanes 0..15 the words of K, lanes 16..31 those of V, eight values (32 bytes) a lane.
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint32_t *k_codes, const uint32_t *k_steps, const uint32_t *v_codes,
                                                       const uint32_t *v_steps, const long long *cache_rows, long long tasks, int n_kv,
                                                       int hd, long long cache_len, int lmax, float *k_out, float *v_out) {
    const int lane = threadIdx.x & 31, w = lane & 15;
    const long long task = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    release_and_wait();
    if (task >= tasks) return;
    const bool is_v = lane >= 16;
    const int words = kv4_words(hd);
    float *out = is_v ? v_out : k_out;
    if (!out || w >= words) return;
    const long long i = task / n_kv;
    const int head = (int)(task - i * n_kv);
    const long long crow = cache_rows[i];
    float v[8] = {};
    if (crow >= 0 && crow < cache_len) {
        const size_t at = ((size_t)(crow / lmax) * n_kv + head) * lmax + (size_t)(crow % lmax);
        const uint32_t c = (is_v ? v_codes : k_codes)[at * words + w], s = (is_v ? v_steps : k_steps)[at];
        const float step = kv4_step(s), lo = kv4_lo(s);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fmaf((float)((c >> (4 * j)) & 15u), step, lo);
    }
    float4 *dst = reinterpret_cast<float4 *>(out + (size_t)task * hd + 8 * w);
    dst[0] = make_float4(v[0], v[1], v[2], v[3]);
    if (8 * w + 4 < hd) dst[1] = make_float4(v[4], v[5], v[6], v[7]);
}

// ---- attention ---------------------------------------------------------------------------------
struct AttnParams {
    const float *q;
    const uint32_t *k_codes, *k_steps, *v_codes, *v_steps;
    const int *lens;
    int t, n_heads, n_kv, hd, lmax;
    float scale;
    float *out;
};

// One CTA per (sequence, query token, head); a half-warp takes one position at a time, a lane one word of its row.
__global__ void __launch_bounds__(256) attn_kv4_kernel(AttnParams p) {
    __shared__ float s_m[16], s_l[16], s_acc[16][KV4_MAX_HD];
    const int lane = threadIdx.x & 31, w = lane & 15, group = threadIdx.x >> 4;
    const long long row = blockIdx.x;
    const int h = (int)(row % p.n_heads), i = (int)(row / p.n_heads % p.t);
    const long long b = row / p.n_heads / p.t;
    release_and_wait();
    const int words = kv4_words(p.hd), len = min(max(p.lens[b], 0), p.lmax) - (p.t - 1 - i);
    const size_t base = ((size_t)b * p.n_kv + h / (p.n_heads / p.n_kv)) * p.lmax;
    float q[8], qs = 0.0f, acc[8] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        q[j] = 8 * w + j < p.hd ? p.q[(size_t)row * p.hd + 8 * w + j] * p.scale : 0.0f;
        qs += q[j];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) qs += __shfl_xor_sync(0xffffffffu, qs, o);
    for (int j0 = 0; j0 < len; j0 += 16) {
        const int j = j0 + group;
        const bool ok = j < len;
        const size_t at = base + (ok ? j : j0);
        const uint32_t kc = w < words ? p.k_codes[at * words + w] : 0u, vc = w < words ? p.v_codes[at * words + w] : 0u;
        const uint32_t ks = p.k_steps[at], vs = p.v_steps[at];
        float dot = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf(q[e], (float)((kc >> (4 * e)) & 15u), dot);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (!ok) continue;  // uniform over the half-warp; the shuffles above are done
        dot = dot * kv4_step(ks) + qs * kv4_lo(ks);
        const float m_new = fmaxf(m, dot), corr = expf(m - m_new), pj = expf(dot - m_new);
        l = l * corr + pj;
        const float step = pj * kv4_step(vs), lo = pj * kv4_lo(vs);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(acc[e], corr, fmaf(step, (float)((vc >> (4 * e)) & 15u), lo));
        m = m_new;
    }
    if (w == 0) { s_m[group] = m; s_l[group] = l; }
#pragma unroll
    for (int e = 0; e < 8; ++e) s_acc[group][8 * w + e] = acc[e];
    __syncthreads();
    if ((int)threadIdx.x < p.hd) {
        float top = -INFINITY, cl = 0.0f, ca = 0.0f;
        for (int g = 0; g < 16; ++g) top = fmaxf(top, s_m[g]);
        for (int g = 0; g < 16; ++g) {
            const float f = s_l[g] == 0.0f ? 0.0f : expf(s_m[g] - top);  // a group without positions has l = 0
            cl += s_l[g] * f;
            ca += s_acc[g][threadIdx.x] * f;
        }
        p.out[(size_t)row * p.hd + threadIdx.x] = cl == 0.0f ? 0.0f : ca / cl;
    }
}

static int check_kv4(int n_heads, int n_kv, int hd, int lmax) {
    if (n_heads < 1 || n_kv < 1 || n_heads % n_kv) return fail(KB_ERR_INVALID, "kv4: %d heads over %d KV heads", n_heads, n_kv);
    if (hd < 4 || hd > KV4_MAX_HD || hd % 4) return fail(KB_ERR_UNSUPPORTED, "kv4: head_dim %d must be a multiple of 4 up to %d", hd, KV4_MAX_HD);
    if (lmax < 4 || lmax % 4) return fail(KB_ERR_UNSUPPORTED, "kv4: cache length %d must be a multiple of 4", lmax);
    return KB_OK;
}

static bool aligned16(const void *a, const void *b = nullptr, const void *c = nullptr, const void *d = nullptr) {
    return !((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(d)) & 15);
}

// blocks of 8 warps for `tasks` warps
static int warp_grid(long long tasks, unsigned *grid) {
    const long long g = (tasks + 7) / 8;
    if (g > 0x7fffffffLL) return fail(KB_ERR_UNSUPPORTED, "%lld rows in one call", tasks);
    *grid = (unsigned)g;
    return KB_OK;
}

static int append(AppendParams &p, bool q4, size_t n, size_t max_pos, size_t n_seqs, kb_stream stream) {
    const size_t heads = (size_t)p.n_heads + 2 * (size_t)p.n_kv;
    if (p.ld == 0) p.ld = heads * p.hd;
    if (p.ld < heads * p.hd) return fail(KB_ERR_INVALID, "append: row stride %zu below %zu", p.ld, heads * p.hd);
    if (!(p.eps >= 0.0f)) return fail(KB_ERR_INVALID, "append: eps must not be negative");
    if (n == 0) return KB_OK;
    if (n > 0x7fffffffu || heads > 0xffffffu || max_pos > 0x7fffffffu || n_seqs > 0x7fffffffu) return fail(KB_ERR_UNSUPPORTED, "append: %zu tokens of %zu heads", n, heads);
    p.tasks = (long long)n * (long long)heads;
    p.max_pos = (long long)max_pos;
    p.cache_len = (long long)n_seqs * p.lmax;
    unsigned grid = 0;
    if (int rc = warp_grid(p.tasks, &grid)) return rc;
    const cudaError_t e = launch_after(q4 ? append_kernel<true> : append_kernel<false>, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream), p);
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
    if (n > 0x7fffffffu || n_seqs > 0x7fffffffu) return fail(KB_ERR_UNSUPPORTED, "kv4: %zu rows of %zu sequences", n, n_seqs);
    const long long tasks = (long long)n * n_kv_heads;
    unsigned grid = 0;
    if (int rc = warp_grid(tasks, &grid)) return rc;
    const cudaError_t e = launch_after(kv4_read_kernel, dim3(grid), dim3(256), 0, static_cast<cudaStream_t>(stream), k_codes, k_steps, v_codes,
                                       v_steps, cache_rows, tasks, n_kv_heads, head_dim, (long long)n_seqs * lmax, lmax, k_out, v_out);
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "kv4 read launch");
}

size_t kb_attn_kv4_workspace_bytes(size_t, int, int, int, int, int) { return 0; }

int kb_attn_kv4(const float *q, const uint32_t *k_codes, const uint32_t *k_steps, const uint32_t *v_codes, const uint32_t *v_steps,
                const int *lens, size_t batch, int t, int n_heads, int n_kv_heads, int head_dim, int lmax, float scale, float *out,
                void *workspace, size_t workspace_bytes, kb_stream stream) {
    (void)workspace; (void)workspace_bytes;
    if (!q || !k_codes || !k_steps || !v_codes || !v_steps || !lens || !out) return fail(KB_ERR_INVALID, "null pointer");
    if (int rc = check_kv4(n_heads, n_kv_heads, head_dim, lmax)) return rc;
    if (t < 0) return fail(KB_ERR_INVALID, "attention: %d query tokens", t);
    if (!(fabsf(scale) < INFINITY)) return fail(KB_ERR_INVALID, "attention: scale must be finite");
    if (!aligned16(k_codes, k_steps, v_codes, v_steps) || !aligned16(q, out)) return fail(KB_ERR_INVALID, "kv4: planes, queries and outputs must be 16-byte aligned");
    if (batch == 0 || t == 0) return KB_OK;
    const size_t rows = batch * (size_t)t * n_heads;
    if (batch > 0x7fffffffu || rows > 0x7fffffffu) return fail(KB_ERR_UNSUPPORTED, "attention: %zu sequences of %d tokens", batch, t);
    AttnParams p = {};
    p.q = q; p.k_codes = k_codes; p.k_steps = k_steps; p.v_codes = v_codes; p.v_steps = v_steps; p.lens = lens;
    p.t = t; p.n_heads = n_heads; p.n_kv = n_kv_heads; p.hd = head_dim; p.lmax = lmax; p.out = out;
    p.scale = scale != 0.0f ? scale : 1.0f / sqrtf((float)head_dim);
    const cudaError_t e = launch_after(attn_kv4_kernel, dim3((unsigned)rows), dim3(256), 0, static_cast<cudaStream_t>(stream), p);
    return e == cudaSuccess ? KB_OK : cuda_fail(e, "kv4 attention launch");
}

}  // extern "C"
