// Writing and reading the paged nvfp4 key/value cache, sm_100a: append (position rotation of queries and keys, nvfp4 cast of
// keys and values into their slots) and read-back (a ragged batch of sequences as bf16).
//
// Both move a few bytes an element and compute little: they are bound by HBM for prompts and by launch latency for single
// tokens.  The nvfp4 cast is the recipe of nvfp4_gs_f (G:1494-1517) with a given outer scale.
#include "kv_cache.cuh"

#include "host_util.h"

namespace qcc {

constexpr int KV_THREADS = 128;
constexpr int KVB = 5;          // blocks of the append on an SM (96 registers a thread; 4 and 6 took 58 and 56 us against 54)

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

// max(|a|, |b|, |c|), NaN if one is
__device__ __forceinline__ float absmax3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
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
//
// An item is two rows of a token with one load of its angles: two heads of q (KV false), or the key and the value of a kv head (KV
// true); the blocks of a launch do one or the other, so a warp carries no instruction of the other kind (60 -> 52 us at 12000 tokens of 48
// heads).  Items are dealt out to the groups of threads in turn, and the rows, the slot and the position of the next one are on
// their way while one is worked on (67 -> 60 us).
__device__ __forceinline__ void rotate_halves(float (&a)[8], float (&b)[8], const float (&c)[8], const float (&s)[8])
{
    // products and differences are rounded one by one (no fused multiply-add): the same bits as the formula in fp32.  (Packed
    // mul.rn.f32x2 and sub.rn.f32x2 gave fused results in one of 10^5 roundings to bf16.)
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float x = a[j], y = b[j];
        a[j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
        b[j] = __fadd_rn(__fmul_rn(y, c[j]), __fmul_rn(x, s[j]));
    }
}
// pairs (2j, 2j + 1) of a chunk
__device__ __forceinline__ void rotate_pairs(float (&a)[8], const float *c, const float *s)
{
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float x = a[2 * j], y = a[2 * j + 1];
        a[2 * j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
        a[2 * j + 1] = __fadd_rn(__fmul_rn(y, c[j]), __fmul_rn(x, s[j]));
    }
}
__device__ __forceinline__ void widen8(uint4 x, float (&a)[8])
{
    a[0] = bf16lo(x.x); a[1] = bf16hi(x.x); a[2] = bf16lo(x.y); a[3] = bf16hi(x.y);
    a[4] = bf16lo(x.z); a[5] = bf16hi(x.z); a[6] = bf16lo(x.w); a[7] = bf16hi(x.w);
}
__device__ __forceinline__ uint4 narrow8(const float (&a)[8])
{
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(a[2 * j], a[2 * j + 1]);
        o[j] = *reinterpret_cast<const uint32_t *>(&p);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int D, bool KV>
__device__ __forceinline__ void append_rows(const AppendArgs &g, float *lut, int block, int blocks)
{
    constexpr int TPR = D / 16, GROUPS = KV_THREADS / TPR;
    const int t = threadIdx.x % TPR, per_token = KV ? g.kv_heads : (g.q_heads + 1) / 2;
    int ca, cb;
    if (g.interleaved || t < g.rot / 16) {
        ca = t;
        cb = t + (g.interleaved ? TPR : g.rot / 16);
    } else {
        ca = g.rot / 16 + t;
        cb = ca + (D - g.rot) / 16;
    }
    const bool turn_halves = !g.interleaved && t < g.rot / 16, turn_a = g.interleaved && 8 * ca < g.rot, turn_b = g.interleaved && 8 * cb < g.rot;

    struct Item {
        int64_t token, slot, pos;
        int part;
        uint4 x[2][2];
    } cur, next;
    const auto load = [&](Item &it) {
        const bool live = it.token < g.tokens;
        const uint16_t *p0, *p1;
        if (KV) {
            p0 = g.k + it.token * g.k_token + it.part * g.k_head;
            p1 = g.v + it.token * g.v_token + it.part * g.v_head;
        } else {
            p0 = g.q + it.token * g.q_token + 2 * it.part * g.q_head;
            p1 = p0 + g.q_head;
        }
        const bool second = live && (KV || 2 * it.part + 1 < g.q_heads);
        const uint4 none = make_uint4(0, 0, 0, 0);
        it.x[0][0] = live ? ld_once_v4(p0 + 8 * ca) : none;
        it.x[0][1] = live ? ld_once_v4(p0 + 8 * cb) : none;
        it.x[1][0] = second ? ld_once_v4(p1 + 8 * ca) : none;
        it.x[1][1] = second ? ld_once_v4(p1 + 8 * cb) : none;
        it.slot = live ? g.slots[it.token] : -1;
        it.pos = live && g.rot > 0 ? g.positions[it.token] : 0;
    };
    const int64_t stride = (int64_t)blocks * GROUPS, first = (int64_t)block * GROUPS + threadIdx.x / TPR, d_token = stride / per_token;
    const int d_part = (int)(stride - d_token * per_token);
    next.token = first / per_token;
    next.part = (int)(first - next.token * per_token);
    load(next);
    float k_outer = 1.0f, v_outer = 1.0f;
    if (KV) {
        k_outer = *g.k_outer;
        v_outer = *g.v_outer;
        nvfp4_fill_recip_lut(lut, __fdiv_rn(1.0f, k_outer));
        nvfp4_fill_recip_lut(lut + 128, __fdiv_rn(1.0f, v_outer));
        __syncthreads();
    }
    const int shift = 31 - __clz(g.page), side = g.page * kv_row_bytes<D>();      // side: bytes of the keys, or values, of a page and head
    // (a warp goes on while one of its groups has an item: the exchanges below need all lanes)
    while (__any_sync(0xFFFFFFFFu, next.token < g.tokens)) {
        cur = next;
        next.token += d_token;
        if ((next.part += d_part) >= per_token) {
            next.part -= per_token;
            next.token++;
        }
        load(next);
        const bool live = cur.token < g.tokens, placed = g.rot == 0 || (cur.pos >= 0 && cur.pos < g.max_pos);
        // halves: 8 cosines and sines of this thread's pairs; interleaved: 4 for chunk ca, 4 for chunk cb
        float c[8], s[8];
        if (turn_halves || turn_a) {
            const float *cs = g.cos_sin + (live && placed ? cur.pos : 0) * g.rot;
            const int half = g.rot / 2, at = turn_halves ? 8 * t : 4 * ca, more = turn_halves ? 4 : 4 * (cb - ca);
            const bool both = turn_halves || turn_b;
            const float4 c0 = *reinterpret_cast<const float4 *>(cs + at), s0 = *reinterpret_cast<const float4 *>(cs + half + at);
            const float4 c1 = both ? *reinterpret_cast<const float4 *>(cs + at + more) : c0, s1 = both ? *reinterpret_cast<const float4 *>(cs + half + at + more) : s0;
            c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
            s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
        }
        bool keep = live && cur.slot >= 0;
        if (KV) {
            if (keep && cur.slot >= g.num_slots) {
                atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
                keep = false;
            }
            if (keep && !placed) {
                atomicMax(&g_qcc_error, QCC_DEVERR_POSITION);
                keep = false;
            }
        }
        uint8_t *base = nullptr;
        const int off = (int)(cur.slot & (g.page - 1));
        if (KV) base = g.cache + ((cur.slot >> shift) * g.kv_heads + cur.part) * (int64_t)(2 * side);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float a[8], b[8];
            widen8(cur.x[i][0], a);
            widen8(cur.x[i][1], b);
            if (!KV || i == 0) {
                if (turn_halves) rotate_halves(a, b, c, s);
                if (turn_a) rotate_pairs(a, c, s);
                if (turn_b) rotate_pairs(b, c + 4, s + 4);
            }
            if (!KV) {
                const int r = 2 * cur.part + i;
                if (live && r < g.q_heads) {
                    uint4 *o = reinterpret_cast<uint4 *>(g.q_out + (cur.token * g.q_heads + r) * D);
                    o[ca] = placed ? narrow8(a) : make_uint4(0, 0, 0, 0);
                    o[cb] = placed ? narrow8(b) : make_uint4(0, 0, 0, 0);
                }
                continue;
            }
            // A block is half in this thread and half in its neighbour, so are two blocks: the even thread works out the scale of `ca`'s,
            // the odd one that of `cb`'s.
            float ma = 0.0f, mb = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                ma = absmax3_nan(ma, a[j], a[j + 1]);
                mb = absmax3_nan(mb, b[j], b[j + 1]);
            }
            const bool odd = t & 1;
            const float mine = max_nan(odd ? mb : ma, __shfl_xor_sync(0xFFFFFFFFu, odd ? ma : mb, 1));
            float rec;
            uint32_t scale = nvfp4_inner_lut(mine, i ? v_outer : k_outer, lut + 128 * i, rec, g.recip_div != 0);
            if (mine != mine) scale = 0x7Fu;     // e4m3 NaN
            const float other = __shfl_xor_sync(0xFFFFFFFFu, rec, 1);
            const float ra = odd ? other : rec, rb = odd ? rec : other;
            if (keep) {
                uint32_t *codes = reinterpret_cast<uint32_t *>(base + i * side + off * kv_row_codes<D>());
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    a[j] = __fmul_rn(a[j], ra);
                    b[j] = __fmul_rn(b[j], rb);
                }
                codes[ca] = cvt_e2m1x8(a);
                codes[cb] = cvt_e2m1x8(b);
                base[i * side + g.page * kv_row_codes<D>() + off * kv_row_scales<D>() + ((odd ? cb : ca) >> 1)] = (uint8_t)scale;
            }
        }
    }
}

template <int D>
__global__ void __launch_bounds__(KV_THREADS, KVB) kv_append_kernel(const AppendArgs g, int kv_blocks)
{
    __shared__ float lut[256];      // of each block scale, the multiplier of the data: keys, values
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x < kv_blocks) append_rows<D, true>(g, lut, blockIdx.x, kv_blocks);
    else append_rows<D, false>(g, lut, blockIdx.x - kv_blocks, gridDim.x - kv_blocks);
}

struct GatherArgs {
    const uint8_t *cache;
    const int32_t *table, *cu;
    const float *k_outer, *v_outer;
    uint16_t *k, *v;
    int64_t total, table_stride, num_pages;
    int seqs, width, kv_heads, page;
};

// D / 16 threads take one token and head, each two 8-element chunks, D / 2 apart, of the key and of the value: neighbouring threads read
// neighbouring bytes of a page, and each of their stores fills whole sectors
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
    const float outer[2] = {*g.k_outer, *g.v_outer};
    // sequence of the row: the last b with cu[b] <= row
    int lo = 0, hi = g.seqs;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (g.cu[mid] <= row) lo = mid; else hi = mid - 1;
    }
    const int side = g.page * kv_row_bytes<D>();
    const uint8_t *base = nullptr;
    int off = 0;
    if (lo < g.seqs && row >= *g.cu) {
        const int shift = 31 - __clz(g.page);
        const int64_t i = row - g.cu[lo], pi = i >> shift;
        const int64_t pg = pi < g.width ? g.table[lo * g.table_stride + pi] : -1;
        off = (int)(i & (g.page - 1));
        if (pg < 0 || pg >= g.num_pages) atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
        else base = g.cache + (pg * g.kv_heads + head) * (int64_t)(2 * side);
    }
    uint32_t codes[2][2] = {}, scales[2][2] = {};
    if (base) {
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const uint8_t *p = base + w * side;
                codes[w][c] = reinterpret_cast<const uint32_t *>(p + off * kv_row_codes<D>())[t + c * TPR];
                scales[w][c] = p[g.page * kv_row_codes<D>() + off * kv_row_scales<D>() + ((t + c * TPR) >> 1)];
            }
    }
    const size_t at = ((size_t)row * g.kv_heads + head) * D;
#pragma unroll
    for (int w = 0; w < 2; w++) {
        uint4 *dst = reinterpret_cast<uint4 *>((w ? g.v : g.k) + at) + t;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const uint32_t sc = e4m3_to_half2(scales[w][c]);
            uint32_t v[4], o[4];
            e2m1x8_to_half(codes[w][c], v);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t p = hmul2_bits(v[j], sc);       // exact: 2 + 4 significant bits
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&p));
                const __nv_bfloat162 b = __floats2bfloat162_rn(__fmul_rn(f.x, outer[w]), __fmul_rn(f.y, outer[w]));
                o[j] = base ? *reinterpret_cast<const uint32_t *>(&b) : 0;
            }
            dst[c * TPR] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
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
    if (!p->k || !p->v || (!p->cache && p->num_pages > 0) || !p->slots || !p->k_outer || !p->v_outer) return QCC_ERR_ARG;
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
    // blocks for keys and values, and for queries: as many as the items fill, at most as many as are resident, in proportion to the work (an
    // item of keys and values, which are cast, takes about half as long again: with shares of 1, 1.25, 1.5, 2 and 3 to one 12000 tokens of 48
    // heads took 62, 56, 52, 55 and 60 us)
    const int groups = KV_THREADS / (p->head_dim / 16), q_pairs = (g.q_heads + 1) / 2;
    const int64_t kv_all = (p->tokens * g.kv_heads + groups - 1) / groups, q_all = (p->tokens * q_pairs + groups - 1) / groups, most = (int64_t)sm_count() * KVB;
    int64_t kv_blocks = kv_all, q_blocks = q_all;
    if (kv_all + q_all > most) {
        kv_blocks = most * 3 * g.kv_heads / (3 * g.kv_heads + 2 * q_pairs);
        kv_blocks = kv_blocks < 1 ? 1 : kv_blocks > kv_all ? kv_all : kv_blocks;
        q_blocks = q_all == 0 ? 0 : most - kv_blocks < 1 ? 1 : most - kv_blocks < q_all ? most - kv_blocks : q_all;
    }
    const unsigned blocks = (unsigned)(kv_blocks + q_blocks);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return (int)(p->head_dim == 128 ? launch_maybe_pdl(kv_append_kernel<128>, dim3(blocks), dim3(KV_THREADS), 0, st, true, g, (int)kv_blocks)
                                    : launch_maybe_pdl(kv_append_kernel<64>, dim3(blocks), dim3(KV_THREADS), 0, st, true, g, (int)kv_blocks));
}

extern "C" int qcc_nvfp4_kv_gather(const void *cache, int64_t num_pages, int kv_heads, int page, int head_dim, const int32_t *table,
                                   int64_t table_stride, int table_width, const int32_t *cu_kv, int seqs, int64_t total, const float *k_outer,
                                   const float *v_outer, void *k, void *v, void *stream)
{
    if ((head_dim != 64 && head_dim != 128) || kv_heads < 1 || kv_heads > 4096 || !page_ok(page) || num_pages < 0 || seqs < 0 || total < 0 ||
        table_width < 0 || table_stride < 0)
        return QCC_ERR_SHAPE;
    if (total == 0) return 0;
    if ((!cache && num_pages > 0) || !cu_kv || !k_outer || !v_outer || !k || !v || (!table && table_width > 0 && seqs > 0)) return QCC_ERR_ARG;
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
