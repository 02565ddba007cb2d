// What the kernels of attention over the paged nvfp4 cache share.
#pragma once
#include "kv_cache.cuh"

namespace qcc {

constexpr unsigned int QCC_DEVERR_QUERIES = 22u;    // query offsets that are not ascending within the rows of q
constexpr int KV_MAX_SEQS = 4096;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct AttnArgs {
    const uint16_t *q;
    const uint8_t *cache;
    const int32_t *table, *kv_lens, *cu_q;
    const float *k_outer, *v_outer;
    uint16_t *out;
    float *lse, *part;      // part: 2 slots per CTA, each the sums of its rows, then their maxima and denominators
    int32_t *prefix;        // few queries: tiles before each sequence, seqs + 1
    int64_t q_token, q_head, table_stride, num_pages, rows;
    float scale_log2;
    int seqs, width, q_heads, kv_heads, group, page, max_q;
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
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// queries and cached tokens of sequence b, checked against what the caller's tensors hold
__device__ __forceinline__ void seq_of(const AttnArgs &g, int b, int &q0, int &n, int &L)
{
    if (g.cu_q) {
        q0 = __ldg(g.cu_q + b);
        n = __ldg(g.cu_q + b + 1) - q0;
        if (q0 < 0 || n < 0 || n > g.max_q || (int64_t)q0 + n > g.rows) {
            atomicMax(&g_qcc_error, QCC_DEVERR_QUERIES);
            q0 = 0;
            n = 0;
        }
    } else {
        q0 = b;
        n = 1;
    }
    L = max(__ldg(g.kv_lens + b), 0);
    if (L > (int64_t)g.width * g.page) {
        atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
        L = g.width * g.page;
    }
}

// The power of two that brings a row of q to fp16, its largest magnitude (fp32 bits) to [2^7, 2^8), and its inverse; 1 for a row
// with an infinity or a NaN, which stay what they are.  2^70 at most: rows that are smaller still score 0 to all 24 bits of exp.
__device__ __forceinline__ void q_power(uint32_t largest, float &mult, float &back)
{
    uint32_t e = largest >> 23;
    e = e == 255u ? 134u : max(e, 64u);
    mult = u2f((261u - e) << 23);
    back = u2f((e - 7u) << 23);
}

// kv_prompt.cu: many queries a sequence
bool prompt_fits(int64_t rows, int group, int seqs, int kv_heads, int64_t cached);      // whether its tiles can be numbered in 31 bits
size_t prompt_workspace_bytes(int64_t rows, int group, int seqs, int head_dim);
int prompt_launch(const AttnArgs &g, int head_dim, void *workspace, cudaStream_t st);

}  // namespace qcc
