// What the kernels of attention over the paged nvfp4 cache share.
#pragma once
#include "kv_cache.cuh"

namespace qcc {

constexpr unsigned int QCC_DEVERR_QUERIES = 22u;    // query offsets that are not ascending within the rows of q
constexpr int KV_MAX_SEQS = 4096;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Probabilities are kept against a reference that is P_LIFT below a row's maximum, in fp16: a row's largest is 2^7 when the reference
// is set and, as that moves only once a score is P_MOST above it, at most 2^15.  So the upper end of fp16's range is used, and a key's rounding is half a step,
// 2^-11, down to 2^-21 of the largest; below, half of 2^-24, 2^-32 of the largest.  (All in log2 units; lse has the reference added back.)
constexpr float P_LIFT = 7.0f, P_MOST = 15.0f;
// the reference for a row's largest score; scores beyond 2^28 are multiples of 32, and one whose reference was rounded down that far would leave
// fp16's range: there the next number up
__device__ __forceinline__ float reference_of(float score, float factor)
{
    const float r = fmaf(score, factor, -P_LIFT);
    return fmaf(score, factor, -r) > P_MOST ? u2f(f2u(r) + (r > 0.0f ? 1u : 0xFFFFFFFFu)) : r;
}

struct AttnArgs {
    const uint16_t *q;
    const uint8_t *cache;
    const int32_t *table, *kv_lens, *cu_q;
    const float *k_outer, *v_outer;
    uint16_t *out;
    float *lse, *part;      // part: 2 slots per CTA, each the sums of its rows (rows, D), then their maxima and denominators
    int4 *seams;            // 2 per CTA
    int64_t q_token, q_head, table_stride, num_pages, rows;
    float scale_log2;
    int seqs, width, q_heads, kv_heads, group, page, max_q;
    int whole;              // kv_attention.cu: units are dealt out whole, none spans CTAs
    int wide;               // kv_prompt.cu: rows of q (1), of out (2), of part (4) lie on 32-byte boundaries
};

__device__ __forceinline__ float ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t lds_u8(uint32_t addr)
{
    uint32_t r;
    asm volatile("{\n.reg .u16 t;\nld.shared.u8 t, [%1];\ncvt.u32.u16 %0, t;\n}\n" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr)
{
    uint16_t r;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t addr)
{
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a)
{
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void bulk_load_at(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// queries and cached tokens of sequence b, checked against what the caller's tensors hold
__device__ __forceinline__ void seq_of(const AttnArgs &g, int b, int &q0, int &n, int &L)
{
    if (g.cu_q) {
        q0 = ld_i32(g.cu_q + b);
        const int64_t end = ld_i32(g.cu_q + b + 1), count = end - q0;      // (64 bits: the offsets may be anything)
        n = (int)count;
        if (q0 < 0 || count < 0 || count > g.max_q || end > g.rows) {
            atomicMax(&g_qcc_error, QCC_DEVERR_QUERIES);
            q0 = 0;
            n = 0;
        }
    } else {
        q0 = b;
        n = 1;
    }
    L = max(ld_i32(g.kv_lens + b), 0);
    if (L > (int64_t)g.width * g.page) {
        atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
        L = g.width * g.page;
    }
}

// The power of two that brings a row of q to fp16, its largest magnitude (fp32 bits) to [2^7, 2^8), and its inverse; 1 for a row
// with an infinity.  Infinities and NaN stay what they are.  2^70 at most: rows that are smaller still score 0 to all 24 bits of exp.
__device__ __forceinline__ void q_power(uint32_t largest, float &mult, float &back)
{
    uint32_t e = largest >> 23;
    e = e == 255u ? 134u : max(e, 64u);
    mult = u2f((261u - e) << 23);
    back = u2f((e - 7u) << 23);
}

// Zeros, and lse -inf: all heads of `n` rows of q from row `first` on, by CTA `cta` of `ctas`.
template <int D>
__device__ __forceinline__ void fill_rows(const AttnArgs &g, int64_t first, int64_t n, int cta, int ctas)
{
    uint4 *o = reinterpret_cast<uint4 *>(g.out + first * g.q_heads * D);
    const int64_t step = (int64_t)ctas * blockDim.x, at = (int64_t)cta * blockDim.x + threadIdx.x;
    for (int64_t i = at; i < n * g.q_heads * (D / 8); i += step) o[i] = make_uint4(0, 0, 0, 0);
    if (g.lse)
        for (int64_t i = at; i < n * g.q_heads; i += step) g.lse[first * g.q_heads + i] = -INFINITY;
}

// ---- joining what the CTAs of one kernel left of the units (rows of a sequence and kv head) that span them
//
// CTA i works on the flat tiles [total * i / ctas, total * (i + 1) / ctas).  Where its first tile is not the first of its unit it
// notes the seam: {unit's first tile, tile behind its last, total, number of the sequence's rows}, {q0, head, the unit's first row, 0}.
__device__ __forceinline__ void note_seam(const AttnArgs &g, int unit_first, int unit_last, int total, int rows, int q0, int head, int row0)
{
    g.seams[2 * blockIdx.x] = make_int4(unit_first, unit_last, total, rows);
    g.seams[2 * blockIdx.x + 1] = make_int4(q0, head, row0, 0);
}
__device__ __forceinline__ int owner_of(int tile, int ctas, int total) { return (int)((((int64_t)tile + 1) * ctas - 1) / total); }

// CTA (c, y): rows y * ROWS ... of the unit whose first seam is CTA c's.  D / 4 threads take a row at a time; PG groups of threads
// share the parts of a row.  A thread loads four parts, maxima and sums, before it needs any of them.  Everything is added in
// a fixed order.
template <int D, int PG, int ROWS, int THREADS>
__global__ void __launch_bounds__(THREADS) kv_join_kernel(const AttnArgs g, int grid, int slot_rows)
{
    constexpr int TPR = D / 4, STEP = THREADS / TPR / PG;
    static_assert(PG == 1 || STEP == ROWS, "with groups a CTA takes its rows at once");
    __shared__ float4 acc[PG > 1 ? THREADS : 1];
    __shared__ float2 stat[PG > 1 ? THREADS / TPR : 1];
    pdl_wait();
    const int c = blockIdx.x;
    const int4 s0 = g.seams[2 * c], s1 = g.seams[2 * c + 1];
    const float v_outer = *g.v_outer;
    if (s0.x < 0) return;
    const int total = s0.z, ctas = min(grid, total), i0 = owner_of(s0.x, ctas, total);
    if (i0 != c - 1) return;
    const int parts = owner_of(s0.y - 1, ctas, total) - i0 + 1;
    const int second = (int)((int64_t)total * i0 / ctas) < s0.x ? 1 : 0;      // the unit is not the first of its first CTA
    const size_t slot = (size_t)slot_rows * (D + 2);
    const float *base = g.part + 2 * i0 * slot;
    const int in = threadIdx.x % TPR, d = in * 4, pg = threadIdx.x / TPR % PG;
#pragma unroll 2
    for (int k = threadIdx.x / TPR / PG; k < ROWS; k += STEP) {
        const int row = blockIdx.y * ROWS + k, r = s1.z + row;
        float top = -INFINITY, den = 0.0f;
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int j0 = pg; j0 < parts; j0 += 4 * PG) {
            float2 w[4];
            float4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int j = j0 + u * PG;
                w[u] = make_float2(-INFINITY, 0.0f);
                v[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (j < parts) {
                    const float *p = base + (2 * j + (j ? 0 : second)) * slot;
                    w[u] = reinterpret_cast<const float2 *>(p + slot_rows * D)[row];
                    v[u] = *reinterpret_cast<const float4 *>(p + row * D + d);
                }
            }
            const float up = fmaxf(fmaxf(fmaxf(top, w[0].x), fmaxf(w[1].x, w[2].x)), w[3].x);
            const float old = top == -INFINITY ? 1.0f : ex2(top - up);       // a part that saw nothing holds zeros (or NaN, which stays)
            top = up;
            den *= old; sum.x *= old; sum.y *= old; sum.z *= old; sum.w *= old;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float a = w[u].x == -INFINITY ? 1.0f : ex2(w[u].x - top);
                den = fmaf(w[u].y, a, den);
                sum.x = fmaf(v[u].x, a, sum.x); sum.y = fmaf(v[u].y, a, sum.y); sum.z = fmaf(v[u].z, a, sum.z); sum.w = fmaf(v[u].w, a, sum.w);
            }
        }
        if (PG > 1) {
            acc[threadIdx.x] = sum;
            if (in == 0) stat[threadIdx.x / TPR] = make_float2(top, den);
            __syncthreads();
            if (pg) return;
            const int g0 = threadIdx.x / TPR;
            for (int i = 0; i < PG; i++) top = fmaxf(top, stat[g0 + i].x);
            den = 0.0f;
            sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int i = 0; i < PG; i++) {
                const float2 w = stat[g0 + i];
                const float4 v = acc[threadIdx.x + i * TPR];
                const float a = w.x == -INFINITY ? 1.0f : ex2(w.x - top);
                den = fmaf(w.y, a, den);
                sum.x = fmaf(v.x, a, sum.x); sum.y = fmaf(v.y, a, sum.y); sum.z = fmaf(v.z, a, sum.z); sum.w = fmaf(v.w, a, sum.w);
            }
        }
        if (r >= s0.w) continue;
        const int i = r / g.group;
        const int64_t at = (int64_t)(s1.x + i) * g.q_heads + s1.y * g.group + r - i * g.group;
        const bool none = den == 0.0f;
        const float inv = none ? 0.0f : __fdividef(v_outer, den);
        const __nv_bfloat162 y0 = __floats2bfloat162_rn(none ? 0.0f : sum.x * inv, none ? 0.0f : sum.y * inv);
        const __nv_bfloat162 y1 = __floats2bfloat162_rn(none ? 0.0f : sum.z * inv, none ? 0.0f : sum.w * inv);
        *reinterpret_cast<uint2 *>(g.out + at * D + d) = make_uint2(*reinterpret_cast<const uint32_t *>(&y0), *reinterpret_cast<const uint32_t *>(&y1));
        if (in == 0 && g.lse) g.lse[at] = none ? -INFINITY : (top + log2f(den)) * LN2;
    }
}

// kv_prompt.cu: many queries a sequence
bool prompt_fits(int64_t rows, int group, int seqs, int kv_heads, int64_t cached);      // whether its tiles can be numbered in 31 bits
size_t prompt_workspace_bytes(int64_t rows, int group, int seqs, int head_dim);
int prompt_launch(const AttnArgs &g, int head_dim, void *workspace, cudaStream_t st);

}  // namespace qcc
