// Writing and reading the paged nvfp4 key/value cache, sm_100a: append (position rotation of queries and keys, nvfp4 cast of
// keys and values into their slots) and read-back (a ragged batch of sequences as bf16).
//
// Both move a few bytes an element and compute little: they are bound by HBM for prompts and by launch latency for single
// tokens.  The nvfp4 cast is the recipe of nvfp4_gs_f (G:1494-1517) with a given outer scale.
#include "kv_cache.cuh"

#include "host_util.h"

namespace qcc {

constexpr int KV_THREADS = 128;
constexpr int KV_ROWS = 4;      // rows (heads) of a token that one group of threads takes, with one load of its angles

struct AppendArgs {
    const uint16_t *k, *v, *q;
    uint16_t *q_out;
    uint8_t *cache;
    const int64_t *slots, *positions;
    const float *cos_sin, *k_outer, *v_outer;
    int64_t tokens, max_pos, num_slots;
    int64_t k_token, k_head, v_token, v_head, q_token, q_head;   // strides, elements
    int kv_heads, q_heads, page, rot, interleaved, recip_div;
};

// max(a, b), NaN if either is: a block with a NaN gets a NaN scale, and all its values read back as NaN
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// D / 16 threads share a row of D elements; each holds two 8-element chunks, `ca` and `cb`.  With rotation in halves they are
// partners (element i of one turns with element i of the other), so no thread needs another's data; chunks 2i and 2i + 1, one
// nvfp4 block, are in neighbouring threads.
template <int D>
__global__ void __launch_bounds__(KV_THREADS) kv_append_kernel(const AppendArgs g)
{
    constexpr int TPR = D / 16, GROUPS = KV_THREADS / TPR;
    pdl_trigger();
    pdl_wait();
    const int t = threadIdx.x % TPR;
    const int rows = g.q_heads + 2 * g.kv_heads, per_token = (rows + KV_ROWS - 1) / KV_ROWS;
    const int64_t item = (int64_t)blockIdx.x * GROUPS + threadIdx.x / TPR;
    const int64_t token = item / per_token;
    const int part = (int)(item - token * per_token);
    const bool live = token < g.tokens;
    int ca, cb;
    if (g.interleaved || t < g.rot / 16) {
        ca = t;
        cb = t + (g.interleaved ? TPR : g.rot / 16);
    } else {
        ca = g.rot / 16 + t;
        cb = ca + (D - g.rot) / 16;
    }

    uint4 xa[KV_ROWS], xb[KV_ROWS];
#pragma unroll
    for (int i = 0; i < KV_ROWS; i++) {
        const int r = part * KV_ROWS + i;        // queries first, then keys, then values
        const uint16_t *p = nullptr;
        if (live && r < rows) {
            if (r < g.q_heads) p = g.q + token * g.q_token + r * g.q_head;
            else if (r < g.q_heads + g.kv_heads) p = g.k + token * g.k_token + (r - g.q_heads) * g.k_head;
            else p = g.v + token * g.v_token + (r - g.q_heads - g.kv_heads) * g.v_head;
        }
        xa[i] = p ? ld_nc_v4(p + 8 * ca) : make_uint4(0, 0, 0, 0);
        xb[i] = p ? ld_nc_v4(p + 8 * cb) : make_uint4(0, 0, 0, 0);
    }

    const int64_t slot = live ? g.slots[token] : -1;
    bool keep = slot >= 0, placed = true;
    if (slot >= g.num_slots) {
        atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
        keep = false;
    }
    // halves: 8 cosines and sines of this thread's pairs; interleaved: 4 for chunk ca, 4 for chunk cb
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) { c[i] = 1.0f; s[i] = 0.0f; }
    if (live && g.rot > 0) {
        const int64_t pos = g.positions[token];
        placed = pos >= 0 && pos < g.max_pos;
        if (!placed && keep) atomicMax(&g_qcc_error, QCC_DEVERR_POSITION);
        keep = keep && placed;
        const float *cs = g.cos_sin + (placed ? pos : 0) * g.rot;
        const int half = g.rot / 2;
        if (!g.interleaved) {
            if (t < g.rot / 16) {
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 a = *reinterpret_cast<const float4 *>(cs + 8 * t + i), b = *reinterpret_cast<const float4 *>(cs + half + 8 * t + i);
                    c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
                    s[i] = b.x; s[i + 1] = b.y; s[i + 2] = b.z; s[i + 3] = b.w;
                }
            }
        } else {
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const int ch = w ? cb : ca;
                if (8 * ch < g.rot) {
                    const float4 a = *reinterpret_cast<const float4 *>(cs + 4 * ch), b = *reinterpret_cast<const float4 *>(cs + half + 4 * ch);
                    c[4 * w] = a.x; c[4 * w + 1] = a.y; c[4 * w + 2] = a.z; c[4 * w + 3] = a.w;
                    s[4 * w] = b.x; s[4 * w + 1] = b.y; s[4 * w + 2] = b.z; s[4 * w + 3] = b.w;
                }
            }
        }
    }
    const float k_outer = __ldg(g.k_outer), v_outer = __ldg(g.v_outer), k_inv = __fdiv_rn(1.0f, k_outer), v_inv = __fdiv_rn(1.0f, v_outer);
    // the page, and the place in it, of this token
    const int shift = 31 - __clz(g.page), off = (int)(slot & (g.page - 1));
    uint8_t *const page = g.cache + (slot >> shift) * ((int64_t)g.kv_heads * 2 * g.page * kv_row_bytes<D>());
    const bool turn_halves = !g.interleaved && t < g.rot / 16;

#pragma unroll
    for (int i = 0; i < KV_ROWS; i++) {
        const int r = part * KV_ROWS + i;
        const bool is_q = r < g.q_heads, is_v = r >= g.q_heads + g.kv_heads;
        float a[8], b[8];
        const uint32_t wa[4] = {xa[i].x, xa[i].y, xa[i].z, xa[i].w}, wb[4] = {xb[i].x, xb[i].y, xb[i].z, xb[i].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            a[2 * j] = bf16lo(wa[j]); a[2 * j + 1] = bf16hi(wa[j]);
            b[2 * j] = bf16lo(wb[j]); b[2 * j + 1] = bf16hi(wb[j]);
        }
        // products and differences are rounded one by one (no fused multiply-add): the same bits as the formula in fp32
        if (!is_v && turn_halves) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = a[j], y = b[j];
                a[j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
                b[j] = __fadd_rn(__fmul_rn(y, c[j]), __fmul_rn(x, s[j]));
            }
        } else if (!is_v && g.interleaved) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (8 * ca < g.rot) {
                    const float x = a[2 * j], y = a[2 * j + 1];
                    a[2 * j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
                    a[2 * j + 1] = __fadd_rn(__fmul_rn(y, c[j]), __fmul_rn(x, s[j]));
                }
                if (8 * cb < g.rot) {
                    const float x = b[2 * j], y = b[2 * j + 1];
                    b[2 * j] = __fsub_rn(__fmul_rn(x, c[4 + j]), __fmul_rn(y, s[4 + j]));
                    b[2 * j + 1] = __fadd_rn(__fmul_rn(y, c[4 + j]), __fmul_rn(x, s[4 + j]));
                }
            }
        }
        // Block maxima and scales, where the warp has a key or a value at all.  A block is half in this thread and half in its neighbour,
        // so are two blocks: the even thread works out the scale of `ca`'s, the odd one that of `cb`'s (three divisions each).
        float ra = 0.0f, rb = 0.0f;
        uint32_t scale = 0;
        const float outer = is_v ? v_outer : k_outer;
        if (__any_sync(0xFFFFFFFFu, keep && r < rows && !is_q)) {
            float ma = 0.0f, mb = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                ma = max_nan(ma, fabsf(a[j]));
                mb = max_nan(mb, fabsf(b[j]));
            }
            const bool odd = t & 1;
            const float mine = max_nan(odd ? mb : ma, __shfl_xor_sync(0xFFFFFFFFu, odd ? ma : mb, 1));
            float rec;
            scale = nvfp4_inner(mine, outer, is_v ? v_inv : k_inv, rec, g.recip_div != 0);
            if (mine != mine) scale = 0x7Fu;     // e4m3 NaN
            const float other = __shfl_xor_sync(0xFFFFFFFFu, rec, 1);
            ra = odd ? other : rec;
            rb = odd ? rec : other;
        }
        if (!live || r >= rows) continue;
        if (is_q) {
            uint4 oa = make_uint4(0, 0, 0, 0), ob = oa;
            if (placed) {
                __nv_bfloat162 p;
#define QCC_PACK(dst, lo, hi) p = __floats2bfloat162_rn(lo, hi), dst = *reinterpret_cast<uint32_t *>(&p)
                QCC_PACK(oa.x, a[0], a[1]); QCC_PACK(oa.y, a[2], a[3]); QCC_PACK(oa.z, a[4], a[5]); QCC_PACK(oa.w, a[6], a[7]);
                QCC_PACK(ob.x, b[0], b[1]); QCC_PACK(ob.y, b[2], b[3]); QCC_PACK(ob.z, b[4], b[5]); QCC_PACK(ob.w, b[6], b[7]);
#undef QCC_PACK
            }
            uint4 *o = reinterpret_cast<uint4 *>(g.q_out + (token * g.q_heads + r) * D);
            o[ca] = oa;
            o[cb] = ob;
        } else if (keep) {
            const int head = is_v ? r - g.q_heads - g.kv_heads : r - g.q_heads;
            uint8_t *base = page + (head * 2 + (is_v ? 1 : 0)) * (g.page * kv_row_bytes<D>());
            uint32_t *codes = reinterpret_cast<uint32_t *>(base + off * kv_row_codes<D>());
            uint8_t *scales = base + g.page * kv_row_codes<D>() + off * kv_row_scales<D>();
#pragma unroll
            for (int j = 0; j < 8; j++) {
                a[j] = __fmul_rn(a[j], ra);
                b[j] = __fmul_rn(b[j], rb);
            }
            codes[ca] = cvt_e2m1x8(a);
            codes[cb] = cvt_e2m1x8(b);
            scales[(t & 1 ? cb : ca) >> 1] = (uint8_t)scale;
        }
    }
}

struct GatherArgs {
    const uint8_t *cache;
    const int32_t *table, *cu;
    const float *k_outer, *v_outer;
    uint16_t *k, *v;
    int64_t total, table_stride, num_pages;
    int seqs, width, kv_heads, page;
};

// D / 16 threads take one token and head, each a 16-element block of the key and one of the value: neighbouring threads read
// neighbouring bytes of a page and write whole 32-byte sectors
template <int D>
__global__ void __launch_bounds__(KV_THREADS) kv_gather_kernel(const GatherArgs g)
{
    constexpr int TPR = D / 16, TOKENS = KV_THREADS / TPR;
    pdl_trigger();
    pdl_wait();
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * TOKENS + threadIdx.x / TPR;
    const int head = blockIdx.y;
    if (row >= g.total) return;
    // sequence of the row: the last b with cu[b] <= row
    int lo = 0, hi = g.seqs;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(g.cu + mid) <= row) lo = mid; else hi = mid - 1;
    }
    uint4 out[2][2] = {};
    if (lo < g.seqs && row >= __ldg(g.cu)) {
        const int64_t i = row - __ldg(g.cu + lo), pi = i / g.page;
        const int off = (int)(i - pi * g.page);
        const int64_t pg = pi < g.width ? __ldg(g.table + lo * g.table_stride + pi) : -1;
        if (pg < 0 || pg >= g.num_pages) {
            atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
        } else {
            const uint8_t *base = g.cache + (pg * g.kv_heads + head) * (int64_t)(2 * g.page * kv_row_bytes<D>());
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const uint2 codes = __ldg(reinterpret_cast<const uint2 *>(base + off * kv_row_codes<D>()) + t);
                const uint32_t sc = e4m3_to_half2(__ldg(base + g.page * kv_row_codes<D>() + off * kv_row_scales<D>() + t));
                const float outer = __ldg(w ? g.v_outer : g.k_outer);
                uint32_t h[8], o[8];
                e2m1x8_to_half(codes.x, *reinterpret_cast<uint32_t(*)[4]>(h));
                e2m1x8_to_half(codes.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const uint32_t p = hmul2_bits(h[j], sc);       // exact: 2 + 4 significant bits
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&p));
                    const __nv_bfloat162 b = __floats2bfloat162_rn(__fmul_rn(f.x, outer), __fmul_rn(f.y, outer));
                    o[j] = *reinterpret_cast<const uint32_t *>(&b);
                }
                out[w][0] = make_uint4(o[0], o[1], o[2], o[3]);
                out[w][1] = make_uint4(o[4], o[5], o[6], o[7]);
                base += g.page * kv_row_bytes<D>();
            }
        }
    }
    const size_t at = ((size_t)row * g.kv_heads + head) * D + t * 16;
    reinterpret_cast<uint4 *>(g.k + at)[0] = out[0][0];
    reinterpret_cast<uint4 *>(g.k + at)[1] = out[0][1];
    reinterpret_cast<uint4 *>(g.v + at)[0] = out[1][0];
    reinterpret_cast<uint4 *>(g.v + at)[1] = out[1][1];
}

static bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

}  // namespace qcc

using namespace qcc;

extern "C" int qcc_kv_cache_device_error(unsigned int *out) { return read_clear_device_error(out); }

extern "C" size_t qcc_nvfp4_kv_page_bytes(int kv_heads, int page, int head_dim)
{
    if (kv_heads < 1 || !page_ok(page) || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)kv_heads * 2 * page * (head_dim / 2 + head_dim / 16);
}

extern "C" int qcc_nvfp4_kv_append(const qcc_kv_append_args *p, void *stream)
{
    if (!p) return QCC_ERR_ARG;
    int flags = p->flags;
    const int recip = take_recip_div(flags);
    if ((flags & ~QCC_ROPE_INTERLEAVED) != 0) return QCC_ERR_ARG;
    if (p->head_dim != 64 && p->head_dim != 128) return QCC_ERR_SHAPE;
    if (p->kv_heads < 1 || p->kv_heads > 4096 || p->q_heads < 0 || p->q_heads > 4096 || !page_ok(p->page) || p->tokens < 0 || p->num_pages < 0) return QCC_ERR_SHAPE;
    if (p->rot < 0 || p->rot > p->head_dim || p->rot % 32 != 0 || p->max_pos < 0) return QCC_ERR_SHAPE;
    if (p->tokens == 0) return 0;
    if (!p->k || !p->v || !p->cache || !p->slots || !p->k_outer || !p->v_outer) return QCC_ERR_ARG;
    if (p->rot > 0 && (!p->positions || !p->cos_sin || p->max_pos < 1)) return QCC_ERR_ARG;
    if (p->q_heads > 0 && (!p->q || !p->q_out)) return QCC_ERR_ARG;
    if (!aligned16(p->k) || !aligned16(p->v) || !aligned16(p->cache) || (p->rot > 0 && !aligned16(p->cos_sin))) return QCC_ERR_ALIGN;
    if ((p->k_stride[0] | p->k_stride[1] | p->v_stride[0] | p->v_stride[1]) % 8 != 0) return QCC_ERR_ALIGN;
    if (p->q_heads > 0 && (!aligned16(p->q) || !aligned16(p->q_out) || (p->q_stride[0] | p->q_stride[1]) % 8 != 0)) return QCC_ERR_ALIGN;
    AppendArgs g;
    g.k = static_cast<const uint16_t *>(p->k); g.v = static_cast<const uint16_t *>(p->v); g.q = static_cast<const uint16_t *>(p->q);
    g.q_out = static_cast<uint16_t *>(p->q_out);
    g.cache = static_cast<uint8_t *>(p->cache);
    g.slots = p->slots; g.positions = p->positions;
    g.cos_sin = p->cos_sin; g.k_outer = p->k_outer; g.v_outer = p->v_outer;
    g.tokens = p->tokens; g.max_pos = p->max_pos; g.num_slots = p->num_pages * p->page;
    g.k_token = p->k_stride[0]; g.k_head = p->k_stride[1];
    g.v_token = p->v_stride[0]; g.v_head = p->v_stride[1];
    g.q_token = p->q_stride[0]; g.q_head = p->q_stride[1];
    g.kv_heads = p->kv_heads; g.q_heads = p->q_heads; g.page = p->page;
    g.rot = p->rot; g.interleaved = (flags & QCC_ROPE_INTERLEAVED) != 0 && p->rot > 0; g.recip_div = recip;
    const int per_token = (g.q_heads + 2 * g.kv_heads + KV_ROWS - 1) / KV_ROWS, groups = KV_THREADS / (p->head_dim / 16);
    const int64_t blocks = (p->tokens * per_token + groups - 1) / groups;
    if (blocks > 0x7FFFFFFF) return QCC_ERR_SHAPE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return (int)(p->head_dim == 128 ? launch_maybe_pdl(kv_append_kernel<128>, dim3((unsigned)blocks), dim3(KV_THREADS), 0, st, true, g)
                                    : launch_maybe_pdl(kv_append_kernel<64>, dim3((unsigned)blocks), dim3(KV_THREADS), 0, st, true, g));
}

extern "C" int qcc_nvfp4_kv_gather(const void *cache, int64_t num_pages, int kv_heads, int page, int head_dim, const int32_t *table,
                                   int64_t table_stride, int table_width, const int32_t *cu_kv, int seqs, int64_t total, const float *k_outer,
                                   const float *v_outer, void *k, void *v, void *stream)
{
    if ((head_dim != 64 && head_dim != 128) || kv_heads < 1 || kv_heads > 4096 || !page_ok(page) || num_pages < 0 || seqs < 0 || total < 0 ||
        table_width < 0 || table_stride < 0)
        return QCC_ERR_SHAPE;
    if (total == 0) return 0;
    if (!cache || !cu_kv || !k_outer || !v_outer || !k || !v || (!table && table_width > 0)) return QCC_ERR_ARG;
    if (!aligned16(cache) || !aligned16(k) || !aligned16(v)) return QCC_ERR_ALIGN;
    const GatherArgs g = {static_cast<const uint8_t *>(cache), table, cu_kv, k_outer, v_outer, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v),
                          total, table_stride, num_pages, seqs, table_width, kv_heads, page};
    const int tokens = KV_THREADS / (head_dim / 16);
    const int64_t blocks = (total + tokens - 1) / tokens;
    if (blocks > 0x7FFFFFFF) return QCC_ERR_SHAPE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)blocks, (unsigned)kv_heads);
    return (int)(head_dim == 128 ? launch_maybe_pdl(kv_gather_kernel<128>, grid, dim3(KV_THREADS), 0, st, true, g)
                                 : launch_maybe_pdl(kv_gather_kernel<64>, grid, dim3(KV_THREADS), 0, st, true, g));
}
