// Attention over the paged nvfp4 key/value cache, sm_100a.
//
//   o = sum_j softmax_j(scale * q . k_j) v_j,   lse = log sum_j exp(scale * q . k_j)
//
// over the keys j that a query sees: query i of the n of a sequence with L cached tokens sees j <= L - n + i.  A query that
// sees none gets o = 0 and lse = -inf.  One pass over the cache with the running maximum and sum of the softmax in fp32.
#include "kv_attention.cuh"
#include "tcgen05.cuh"      // settle()

#include <type_traits>

#include "host_util.h"

namespace qcc {

constexpr unsigned int KV_ATTN_ERR = 8u;            // a wait for a bulk copy ran out

// -------------------------------------------------------------------------------------------------------------------
// Few queries: work split over the cached tokens
//
// The rows of a sequence and kv head (its queries times the heads of the group) are at most a few, so the time is that of
// reading the cache: 9/16 byte an element, and every element has to be widened before a matrix instruction takes it.  That
// widening is what competes with HBM (41 elements a clock and SM at full bandwidth), so codes go from shared memory straight
// into the registers that mma.sync m16n8k16 wants, with no second trip through shared memory:
//   S^T = K Q^T    A: 16 tokens x 16 elements.  A thread's fragment rows are tokens, and the order of the contracted elements
//                  is free as long as Q has the same, so a thread reads 16 contiguous bytes (32 elements) of a token.
//   O^T = V^T P^T  A: 16 elements x 16 tokens.  A thread reads one 16-element block of four tokens; the nibbles of two tokens
//                  are brought side by side before they are widened, which gives the token pairs of the fragment.
// The queries are on the N side, 8 at a time: no row of the instruction is spent on padding when a group has 8 heads.
// Codes times block scales are exact in fp16 (2 + 4 significant bits); q is brought to fp16 by a power of two for its row,
// exact for all elements above 2^-22 of the row's largest; P is rounded to fp16 (see P_LIFT).  The tensor cores are
// far from busy (tcgen05 would need the widened tiles in shared memory, whose bandwidth that alone would use up).
//
// A tile is 128 tokens of one sequence and head, 32 for each warp.  A warp fetches its own tokens by bulk copies into a ring of
// its own, so the warps of a CTA meet only where a unit ends.  All tiles of the batch are numbered and dealt out evenly,
// whatever the lengths; a unit (sequence, head, row tile) that spans CTAs leaves partial sums which a second kernel joins in a
// fixed order.  Short units are dealt out whole instead, where there are many.
//
// Measured, 32 heads over 8 of 128 elements: 64 sequences of up to 16384 tokens 132.5 us, 4.4 TB/s of the cache, 56 % of the issue slots and of the
// ALU pipe; 2 of 131072 with 64 heads 72.3 us.  647 warp instructions for 32 tokens, of which the conversions, scalings and nibble merges are
// 372 and the matrix instructions 32.
// -------------------------------------------------------------------------------------------------------------------
constexpr int SP_WARPS = 4, SP_THREADS = SP_WARPS * 32, SP_WTOK = 32, SP_TOK = SP_WTOK * SP_WARPS;

// CTAs on an SM, as the registers allow: the grid, and with it the workspace, is that many for each SM
constexpr int split_ctas(int D, int NT) { return NT == 1 ? 4 : NT == 2 ? (D == 64 ? 4 : 3) : 2; }

template <int D, int NT> struct SplitCfg {
    static constexpr int TILE = SP_WTOK * 2 * (D / 2 + D / 16);     // bytes of one warp's tokens, keys and values
    static constexpr int CTAS = split_ctas(D, NT);
    static constexpr int STAGES = (NT == 4 ? 4 : 2) * (D == 64 ? 2 : 1);
    // Q in shared memory: it would not fit the registers beside O (NT 1 and 128 elements: it would just, 138 against 133 us for 64 sequences)
    static constexpr bool QS = NT * D > 256 || (NT == 1 && D == 128);
    static constexpr int QBYTES = QS ? NT * (D / 32) * 32 * 16 : 0;
    static constexpr int RED = SP_WARPS * NT * 8 * (D / 4) * 4;
    static constexpr int ML = SP_WARPS * NT * 8 * 2 * 4;
    static constexpr int FIXED = SP_WARPS * (TILE * STAGES + STAGES * 8) + RED + ML + QBYTES;
};

template <int D, int NT> __host__ __device__ constexpr int part_floats() { return NT * 8 * (D + 2); }   // sums (NT * 8, D), then (maximum, denominator) of each row

struct Segment {
    int b, q0, n, L, head, first, last, unit_last;   // first, last: tiles of the unit; unit_last: flat number of the tile behind it
};

// Whether the copies of phase `parity` have come within `polls` polls.  (No look at an abort word, as elsewhere: that alone took 3 % of a
// long decode.)
__device__ __forceinline__ bool copied(uint32_t bar, uint32_t parity, uint32_t polls)
{
    for (uint32_t it = 0; it < polls; it++) {
        uint32_t done;
        asm volatile(
            "{\n.reg .pred p;\n"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

// the segment that starts at flat tile t: its unit's tiles [first, last) within hi
__device__ __forceinline__ void find_segment(const AttnArgs &g, const int32_t *prefix, int t, int hi, Segment &s)
{
    int lo = 0, up = g.seqs - 1;      // last b with prefix[b] <= t (t < total, so it has tiles)
    while (lo < up) {
        const int mid = (lo + up + 1) >> 1;
        if (prefix[mid] <= t) lo = mid; else up = mid - 1;
    }
    s.b = lo;
    seq_of(g, lo, s.q0, s.n, s.L);
    const int kvt = (s.L + SP_TOK - 1) / SP_TOK, local = t - prefix[lo];
    s.head = local / kvt;
    s.first = local - s.head * kvt;
    s.last = min(kvt, s.first + hi - t);
    s.unit_last = prefix[lo] + (s.head + 1) * kvt;
}

template <int D, int NT>
__global__ void __launch_bounds__(SP_THREADS, (SplitCfg<D, NT>::CTAS)) kv_attn_split_kernel(const AttnArgs g)
{
    using C = SplitCfg<D, NT>;
    constexpr int KW = D / 32, VW = D / 64, MT = D / 16, RB = D / 2 + D / 16;    // words of a thread per token: keys, values; m tiles
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t *ring = smem + warp * (C::TILE * C::STAGES);
    float *red = reinterpret_cast<float *>(smem + SP_WARPS * C::TILE * C::STAGES);
    uint4 *s_q = reinterpret_cast<uint4 *>(red + C::RED / 4);
    float2 *ml = reinterpret_cast<float2 *>(s_q + C::QBYTES / 16);
    uint64_t *full = reinterpret_cast<uint64_t *>(ml + C::ML / 8) + warp * C::STAGES;
    int32_t *prefix = reinterpret_cast<int32_t *>(reinterpret_cast<uint64_t *>(ml + C::ML / 8) + SP_WARPS * C::STAGES);
    __shared__ int32_t wsum[SP_WARPS];
    __shared__ uint32_t out_of_time;      // a wait for a copy has run out

    if (lane == 0)
        for (int i = 0; i < C::STAGES; i++) mbar_init(full + i, 1);
    if (threadIdx.x == 0) {
        prefix[0] = 0;
        out_of_time = 0;
    }
    fence_barrier_init();
    pdl_trigger();
    pdl_wait();
    // tiles of each sequence, summed up
    int carry = 0;
    bool gap = false;
    for (int b0 = 0; b0 < g.seqs; b0 += SP_THREADS) {
        const int b = b0 + threadIdx.x;
        int v = 0;
        if (b < g.seqs) {
            int q0, n, L;
            seq_of(g, b, q0, n, L);
            gap |= n && !L;
            v = n ? g.kv_heads * ((L + SP_TOK - 1) / SP_TOK) : 0;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) wsum[warp] = v;
        __syncthreads();
        int before = carry, all = carry;
        for (int w = 0; w < SP_WARPS; w++) {
            if (w < warp) before += wsum[w];
            all += wsum[w];
        }
        if (b < g.seqs) prefix[b + 1] = before + v;
        carry = all;
        __syncthreads();
    }
    const bool empty = __syncthreads_or(gap);      // some sequence has queries and no tokens
    const int total = carry, ctas = min((int)gridDim.x, total);
    if (empty) {
        for (int b = blockIdx.x; b < g.seqs; b += gridDim.x) {
            if (prefix[b + 1] != prefix[b]) continue;
            int q0, n, L;
            seq_of(g, b, q0, n, L);
            fill_rows<D>(g, q0, n, 0, 1);
        }
    }
    if (g.cu_q) {
        const int64_t first = max(g.cu_q[g.seqs], 0);
        fill_rows<D>(g, first, g.rows - first, blockIdx.x, gridDim.x);
    }
    if ((int)blockIdx.x >= ctas) {
        if (threadIdx.x == 0) g.seams[2 * blockIdx.x].x = -1;
        return;
    }
    int lo = (int)((int64_t)total * blockIdx.x / ctas), hi = (int)((int64_t)total * (blockIdx.x + 1) / ctas);
    if (g.whole) {      // up to the next unit's first tile, each
        Segment s;
        find_segment(g, prefix, lo, hi, s);
        if (s.first) lo = s.unit_last;
        if (hi < total) {
            find_segment(g, prefix, hi, total, s);
            if (s.first) hi = s.unit_last;
        }
        if (lo >= hi) return;
    }

    // ---- fetching: the warp's tokens of tile after tile, C::STAGES ahead of their use.  The pages of the next fetch are looked up
    // one fetch early.  Pages of 32 tokens and more: four copies (codes and scales, keys and values), by a lane each; pages of 16:
    // two of a whole (page, head) block.  What a lane copies, and to where, is the same for every tile.
    //
    // A lane whose wait has run out (SP_LATE in its f_stage) copies, arms and waits no more: arming a barrier whose phase is incomplete is
    // undefined.  It goes on through the instructions of its warp, with whatever the stages hold; the host reads the error.
    const int shift = 31 - __clz(g.page), copies = shift == 4 ? 2 : 4;
    const uint32_t block_bytes = (uint32_t)g.page * 2 * RB, page_bytes = block_bytes * g.kv_heads, num_pages = (uint32_t)min(g.num_pages, (int64_t)0x7FFFFFFF);
    const uint32_t in_page = (warp * SP_WTOK) & (g.page - 1), scales_of = lane & 1;
    const uint32_t lane_src = shift == 4 ? 0 : (lane >> 1 & 1) * (g.page * RB) + (scales_of ? g.page * (D / 2) + in_page * (D / 16) : in_page * (D / 2));
    const uint32_t lane_dst = smem_u32(ring) + (shift == 4 ? lane * (C::TILE / 2) : (lane >> 1) * (C::TILE / 2) + scales_of * (SP_WTOK * D / 2));
    const uint32_t lane_bytes = shift == 4 ? C::TILE / 2 : scales_of ? SP_WTOK * D / 16 : SP_WTOK * D / 2;
    const uint32_t bar0 = smem_u32(full);
    int f_t = lo, f_left = 0, f_tok = 0, f_L = 0, f_page = -1;      // next segment; tiles left of this one; this lane's first token, and its page
    constexpr uint32_t SP_LATE = 1u << 31;
    uint32_t f_stage = 0;
    const int32_t *f_row = nullptr;
    const uint8_t *f_base = nullptr;
    const auto seek = [&]() {
        if (--f_left > 0) {
            f_tok += SP_TOK;
            f_row += SP_TOK >> shift;
        } else if (f_t < hi) {
            Segment s;
            find_segment(g, prefix, f_t, hi, s);
            f_left = s.last - s.first;
            f_t += f_left;
            f_L = s.L;
            f_tok = s.first * SP_TOK + warp * SP_WTOK + (shift == 4 ? lane * 16 : 0);
            f_row = g.table + s.b * g.table_stride + (f_tok >> shift);
            f_base = g.cache + s.head * (int64_t)block_bytes + lane_src;
        }
        f_page = f_left > 0 && lane < copies && f_tok < f_L ? ld_i32(f_row) : -1;
    };
    const auto fetch = [&]() {
        if (f_left <= 0) return;
        const bool on_time = !(f_stage & SP_LATE), ok = (uint32_t)f_page < num_pages && on_time;
        if ((uint32_t)f_page >= num_pages && lane < copies && f_tok < f_L) atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
        const uint32_t bytes = __popc(__ballot_sync(0xFFFFFFFFu, ok)) * (shift == 4 ? C::TILE / 2 : C::TILE / 4), bar = bar0 + f_stage * 8;
        if (lane == 0 && on_time) mbar_expect_at(bar, bytes);
        __syncwarp();
        if (ok) bulk_load_at(lane_dst + f_stage * C::TILE, f_base + (uint64_t)(uint32_t)f_page * page_bytes, lane_bytes, bar);
        f_stage = f_stage + 1 == C::STAGES ? 0 : f_stage + 1;
        seek();
    };
    // where a stage has codes and scales of keys and values, and the distance from the first 16 tokens to the second
    const uint32_t k_scales = shift == 4 ? 8 * D : SP_WTOK * D / 2, v_codes = shift == 4 ? 16 * RB : C::TILE / 2, v_scales = v_codes + k_scales;
    const uint32_t next_codes = shift == 4 ? C::TILE / 2 : 8 * D, next_scales = shift == 4 ? C::TILE / 2 : D;
    pdl_copies_fence();
    seek();
#pragma unroll 1
    for (int i = 0; i < C::STAGES; i++) fetch();

    // ---- 32 tokens of every tile each
    const int gr = lane >> 2, c = lane & 3;
    const float k_outer = ld_cg_f32(g.k_outer), v_outer = ld_cg_f32(g.v_outer);
    uint32_t stage = 0, phase = 0;
    for (int t = lo; t < hi;) {
        Segment s;
        find_segment(g, prefix, t, hi, s);
        const int end = s.last;
        const int rows = s.n * g.group;
        if (t == lo && threadIdx.x == 0) note_seam(g, s.first ? t - s.first : -1, s.unit_last, total, rows, s.q0, s.head, 0);

        uint32_t qf[C::QS ? 1 : NT][2 * KW * 2];    // row gr of each n tile, elements of this thread
        float factor[NT][2];            // score -> log2 units, columns 2c and 2c + 1
        int limit[NT][2];               // keys that the column sees
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 8 + gr;
            const int i = r / g.group, h = s.head * g.group + r - i * g.group;
            uint4 w[KW];
            uint32_t acc = 0;
#pragma unroll
            for (int j = 0; j < KW; j++) {
                w[j] = r < rows ? ld_v4(g.q + (int64_t)(s.q0 + i) * g.q_token + h * g.q_head + c * (D / 4) + j * 8) : make_uint4(0, 0, 0, 0);
                acc = absmax2_acc(absmax2_acc(absmax2_acc(absmax2_acc(acc, w[j].x), w[j].y), w[j].z), w[j].w);
            }
            uint32_t m = f2u(hmax_halves_f32(acc));
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
            m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
            float mult, back;
            q_power(m, mult, back);
#pragma unroll
            for (int j = 0; j < KW; j++) {
                uint32_t *f4 = qf[C::QS ? 0 : nt] + 4 * j;
                f4[0] = pack_half2(bf16lo(w[j].x) * mult, bf16hi(w[j].x) * mult);
                f4[1] = pack_half2(bf16lo(w[j].y) * mult, bf16hi(w[j].y) * mult);
                f4[2] = pack_half2(bf16lo(w[j].z) * mult, bf16hi(w[j].z) * mult);
                f4[3] = pack_half2(bf16lo(w[j].w) * mult, bf16hi(w[j].w) * mult);
                if (C::QS && warp == nt % SP_WARPS) s_q[(nt * KW + j) * 32 + lane] = make_uint4(f4[0], f4[1], f4[2], f4[3]);
            }
#pragma unroll
            for (int x = 0; x < 2; x++) {
                factor[nt][x] = __shfl_sync(0xFFFFFFFFu, back, (2 * c + x) * 4) * (g.scale_log2 * k_outer);
                const int rc = nt * 8 + 2 * c + x;
                limit[nt][x] = rc < rows ? s.L - s.n + rc / g.group + 1 : 0;
            }
        }

        if (C::QS) named_barrier(1, SP_WARPS * 32);
        float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < MT; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
        }
        // one warp's 32 tokens from `tok` on; MASKED: some of them are behind the last token, or hidden from some row
        const auto step = [&](auto masked, int tok) {
            constexpr bool MASKED = decltype(masked)::value;
            const uint32_t base = smem_u32(ring + stage * C::TILE);
            constexpr int HB = NT == 1 ? 2 : 1, UH = NT == 4 ? 1 : 2;      // 16-token blocks taken together, as registers allow
#pragma unroll UH
            for (int h0 = 0; h0 < 2; h0 += HB) {
                float sc[HB][NT][4];
#pragma unroll
                for (int h = 0; h < HB; h++) {
                    const uint32_t kc = base + (h0 + h) * next_codes, ks = base + k_scales + (h0 + h) * next_scales;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) sc[h][nt][0] = sc[h][nt][1] = sc[h][nt][2] = sc[h][nt][3] = 0.0f;
                    uint32_t wa[KW], wb[KW], sa[2], sb[2];     // tokens gr and gr + 8
                    if (D == 128) {
                        const uint4 a = lds_v4(kc + gr * 64 + c * 16), b = lds_v4(kc + (gr + 8) * 64 + c * 16);
                        wa[0] = a.x; wa[1] = a.y; wa[2 % KW] = a.z; wa[3 % KW] = a.w;
                        wb[0] = b.x; wb[1] = b.y; wb[2 % KW] = b.z; wb[3 % KW] = b.w;
                        const uint32_t u = e4m3x2_to_half2(lds_u16(ks + gr * 8 + 2 * c)), v = e4m3x2_to_half2(lds_u16(ks + (gr + 8) * 8 + 2 * c));
                        sa[0] = __byte_perm(u, u, 0x1010); sa[1] = __byte_perm(u, u, 0x3232);
                        sb[0] = __byte_perm(v, v, 0x1010); sb[1] = __byte_perm(v, v, 0x3232);
                    } else {
                        const uint2 a = lds_v2(kc + gr * 32 + c * 8), b = lds_v2(kc + (gr + 8) * 32 + c * 8);
                        wa[0] = a.x; wa[1] = a.y;
                        wb[0] = b.x; wb[1] = b.y;
                        sa[0] = sa[1] = e4m3_to_half2(lds_u8(ks + gr * 4 + c));
                        sb[0] = sb[1] = e4m3_to_half2(lds_u8(ks + (gr + 8) * 4 + c));
                    }
#pragma unroll
                    for (int j = 0; j < KW; j++) {
                        uint32_t ha[4], hb[4];
                        e2m1x8_to_half(wa[j], ha);
                        e2m1x8_to_half(wb[j], hb);
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            ha[u] = hmul2_bits(ha[u], sa[j * 2 / KW]);
                            hb[u] = hmul2_bits(hb[u], sb[j * 2 / KW]);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const uint32_t *r4 = qf[C::QS ? 0 : nt] + 4 * j;
                            const uint4 q4 = C::QS ? lds_v4(smem_u32(s_q + (nt * KW + j) * 32 + lane)) : make_uint4(r4[0], r4[1], r4[2], r4[3]);
                            mma16816(sc[h][nt], ha[0], hb[0], ha[1], hb[1], q4.x, q4.y);
                            mma16816(sc[h][nt], ha[2], hb[2], ha[3], hb[3], q4.z, q4.w);
                        }
                    }
                }
                // exponents of the probabilities, against the running reference
                const auto seen = [&](int h, int nt, int x) { return !MASKED || tok + (h0 + h) * 16 + gr + (x >> 1) * 8 < limit[nt][x & 1]; };
                float e[HB][NT][4], most = -INFINITY;
#pragma unroll
                for (int h = 0; h < HB; h++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            e[h][nt][x] = seen(h, nt, x) ? fmaf(sc[h][nt][x], factor[nt][x & 1], -m[nt][x & 1]) : -INFINITY;
                            most = fmaxf(most, e[h][nt][x]);
                        }
                if (__any_sync(0xFFFFFFFFu, most > P_MOST)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            float top = -INFINITY;
#pragma unroll
                            for (int h = 0; h < HB; h++)
#pragma unroll
                                for (int y = x; y < 4; y += 2) top = fmaxf(top, seen(h, nt, y) ? sc[h][nt][y] : -INFINITY);
#pragma unroll
                            for (int sh = 4; sh < 32; sh <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, sh));
                            const float v = fmaxf(m[nt][x], reference_of(top, factor[nt][x])), a = v == -INFINITY ? 1.0f : ex2(m[nt][x] - v);
                            m[nt][x] = v;
                            l[nt][x] *= a;
#pragma unroll
                            for (int i = 0; i < MT; i++) {
                                o[nt][i][x] *= a;
                                o[nt][i][x + 2] *= a;
                            }
#pragma unroll
                            for (int h = 0; h < HB; h++)
#pragma unroll
                                for (int y = x; y < 4; y += 2) e[h][nt][y] = seen(h, nt, y) ? fmaf(sc[h][nt][y], factor[nt][x], -v) : -INFINITY;
                        }
                }
#pragma unroll
                for (int h = 0; h < HB; h++) {
                    uint32_t pb[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const float p0 = ex2(e[h][nt][0]), p1 = ex2(e[h][nt][1]), p2 = ex2(e[h][nt][2]), p3 = ex2(e[h][nt][3]);
                        l[nt][0] += p0 + p2;
                        l[nt][1] += p1 + p3;
                        pb[nt][0] = transpose8x8(pack_half2(p0, p1));
                        pb[nt][1] = transpose8x8(pack_half2(p2, p3));
                    }
                    // values of tokens 2c, 2c + 1 and 2c + 8, 2c + 9
                    const uint32_t vc = base + v_codes + (h0 + h) * next_codes, vs = base + v_scales + (h0 + h) * next_scales;
                    uint32_t vs2[2], vw[4][VW], nan = 0;      // nan: tokens whose block of this thread's elements is NaN
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const int t0 = 2 * c + 8 * x;
                        uint32_t s0 = D == 128 ? lds_u8(vs + t0 * 8 + gr) : lds_u8(vs + t0 * 4 + (gr >> 1)), s1 = D == 128 ? lds_u8(vs + t0 * 8 + 8 + gr) : lds_u8(vs + t0 * 4 + 4 + (gr >> 1));
                        if (MASKED) {        // whatever the slots behind the last token hold, it counts as zero
                            if (tok + (h0 + h) * 16 + t0 >= s.L) s0 = 0;
                            if (tok + (h0 + h) * 16 + t0 + 1 >= s.L) s1 = 0;
                        }
                        if (MASKED) {        // a NaN reaches the columns that see its token: zero here, added to their sums below
                            if ((s0 & 0x7Fu) == 0x7Fu) { nan |= 1u << t0; s0 = 0; }
                            if ((s1 & 0x7Fu) == 0x7Fu) { nan |= 2u << t0; s1 = 0; }
                        }
                        vs2[x] = e4m3x2_to_half2(s0 | (s1 << 8));
                        if (D == 128) {
                            const uint2 a = lds_v2(vc + t0 * 64 + gr * 8), b = lds_v2(vc + t0 * 64 + 64 + gr * 8);
                            vw[2 * x][0] = a.x; vw[2 * x][1 % VW] = a.y;
                            vw[2 * x + 1][0] = b.x; vw[2 * x + 1][1 % VW] = b.y;
                        } else {
                            vw[2 * x][0] = lds_u32(vc + t0 * 32 + gr * 4);
                            vw[2 * x + 1][0] = lds_u32(vc + t0 * 32 + 32 + gr * 4);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < VW; j++) {
                        uint32_t ev[2][4], od[2][4];      // even and odd elements, token pairs
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const uint32_t w0 = vw[2 * x][j], w1 = vw[2 * x + 1][j];
                            e2m1x8_to_half((w0 & 0x0F0F0F0Fu) | ((w1 << 4) & 0xF0F0F0F0u), ev[x]);
                            e2m1x8_to_half(((w0 >> 4) & 0x0F0F0F0Fu) | (w1 & 0xF0F0F0F0u), od[x]);
#pragma unroll
                            for (int u = 0; u < 4; u++) {
                                ev[x][u] = hmul2_bits(ev[x][u], vs2[x]);
                                od[x][u] = hmul2_bits(od[x][u], vs2[x]);
                            }
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma16816(o[nt][4 * j + u], ev[0][u], od[0][u], ev[1][u], od[1][u], pb[nt][0], pb[nt][1]);
                    }
                    if (MASKED && __any_sync(0xFFFFFFFFu, nan)) {
                        nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 1);
                        nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 2);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int x = 0; x < 2; x++) {
                                const int sees = min(max(limit[nt][x] - tok - (h0 + h) * 16, 0), 16);
                                if (nan & ((1u << sees) - 1u)) {
#pragma unroll
                                    for (int i = 0; i < MT; i++) o[nt][i][x] = o[nt][i][x + 2] = u2f(0x7FFFFFFFu);
                                }
                            }
                    }
                }
            }
        };
        const int clear = s.L - s.n + 1;      // keys that every row sees

        for (int tile = s.first; tile < end; tile++) {
            if (!copied(bar0 + stage * 8, phase, f_stage & SP_LATE ? 0 : 1u << 24)) {
                f_stage |= SP_LATE;
                out_of_time = 1;
                atomicMax(&g_qcc_error, KV_ATTN_ERR);
            }
            const int tok = tile * SP_TOK + warp * SP_WTOK;
            if (tok + SP_WTOK <= clear) step(std::false_type(), tok);
            else if (tok < s.L) step(std::true_type(), tok);
            __syncwarp();      // all lanes have read the stage that the next fetch overwrites
            fetch();
            if (++stage == C::STAGES) {
                stage = 0;
                phase ^= 1;
            }
        }

        // ---- join the warps, then write the unit's result or this CTA's partial sums
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
#pragma unroll
                for (int sh = 4; sh < 32; sh <<= 1) l[nt][x] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][x], sh);
                if (gr == 0) ml[warp * NT * 8 + nt * 8 + 2 * c + x] = make_float2(m[nt][x], l[nt][x]);
            }
        named_barrier(1, SP_WARPS * 32);
        const bool whole = s.first == 0 && t + s.last - s.first == s.unit_last;
        float *slot = g.part + (size_t)(2 * blockIdx.x + (t == lo ? 0 : 1)) * part_floats<D, NT>();
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                float top = -INFINITY;
                for (int w = 0; w < SP_WARPS; w++) top = fmaxf(top, ml[w * NT * 8 + nt * 8 + 2 * c + x].x);
                const float a = m[nt][x] == -INFINITY ? 1.0f : ex2(m[nt][x] - top);      // an empty warp holds zeros (or NaN, which stays)
#pragma unroll
                for (int i = 0; i < MT; i++) {
                    o[nt][i][x] *= a;
                    o[nt][i][x + 2] *= a;
                }
            }
        constexpr int DQ = D / 4, PER = MT / 4;        // elements and m tiles of one round
#pragma unroll
        for (int round = 0; round < 4; round++) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < PER; i++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        red[(warp * NT * 8 + nt * 8 + 2 * c + (x & 1)) * DQ + gr * (2 * PER) + 2 * i + (x >> 1)] = o[nt][round * PER + i][x];
            named_barrier(1, SP_WARPS * 32);
            for (int e = threadIdx.x; e < NT * 8 * DQ; e += SP_WARPS * 32) {
                const int qi = e / DQ, x = e - qi * DQ;
                const int d = (x / (2 * PER)) * (4 * 2 * PER) + round * 2 * PER + x % (2 * PER);
                float sum = 0.0f, top = -INFINITY, den = 0.0f;
                for (int w = 0; w < SP_WARPS; w++) {
                    sum += red[(w * NT * 8 + qi) * DQ + x];
                    top = fmaxf(top, ml[w * NT * 8 + qi].x);
                }
                for (int w = 0; w < SP_WARPS; w++) {
                    const float2 v = ml[w * NT * 8 + qi];
                    den += v.y * (v.x == -INFINITY ? 1.0f : ex2(v.x - top));
                }
                if (whole) {
                    const int r = qi;
                    if (r < rows) {
                        const int i = r / g.group;
                        const int64_t at = (int64_t)(s.q0 + i) * g.q_heads + s.head * g.group + r - i * g.group;
                        const __nv_bfloat16 y = __float2bfloat16_rn(den == 0.0f ? 0.0f : __fdividef(sum * v_outer, den));
                        g.out[at * D + d] = *reinterpret_cast<const uint16_t *>(&y);
                        if (round == 0 && x == 0 && g.lse) g.lse[at] = den == 0.0f ? -INFINITY : (top + log2f(den)) * LN2;
                    }
                } else {
                    slot[qi * D + d] = sum;
                    if (round == 0 && x == 0) reinterpret_cast<float2 *>(slot + NT * 8 * D)[qi] = make_float2(top, den);
                }
            }
            named_barrier(1, SP_WARPS * 32);
        }
        t += s.last - s.first;
    }
    settle(smem_u32(&out_of_time));      // (the last unit ended with a barrier)
}

template <int D, int NT>
static int split_launch(const AttnArgs &g, cudaStream_t st)
{
    using C = SplitCfg<D, NT>;
    static PerDeviceFlag done;
    const int dev = current_device_slot();
    if (dev < 0) return QCC_ERR_ARG;
    if (!done.get(dev)) {
        cudaError_t e = cudaFuncSetAttribute(kv_attn_split_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::FIXED + (KV_MAX_SEQS + 1) * 4);
        if (e != cudaSuccess) return (int)e;
        done.set(dev);
    }
    const int grid = sm_count() * C::CTAS;
    cudaError_t e = launch_maybe_pdl(kv_attn_split_kernel<D, NT>, dim3(grid), dim3(SP_THREADS), C::FIXED + (g.seqs + 1) * 4, st, true, g);
    if (e != cudaSuccess) return (int)e;
    if (g.whole) return 0;
    return (int)launch_maybe_pdl(kv_join_kernel<D, 2, 4, 2 * D>, dim3(grid, 2 * NT), dim3(2 * D), 0, st, true, g, grid, NT * 8);
}

// how the rows of a sequence and kv head are tiled: 8 * nt rows
static int row_tiles_of(int64_t rows) { return rows <= 8 ? 1 : rows <= 16 ? 2 : 4; }
// More rows than 32: the tcgen05 kernel.  Below, the widening in registers is ahead or even: 18 rows over up to 2000 tokens of 64 sequences 66 against 77 us,
// 32 over 8000 247 against 246, with 64-element heads 57 against 81; 16 rows over 8000 tokens 79 against 144.  Only 32 rows over 100 tokens are
// behind (19 against 15).
static bool many_queries(int max_q, int group) { return (int64_t)max_q * group > 32; }
// Units are dealt out whole, with nothing to join and one launch less, where the longest that the table allows is short, or where it is not long (16 tiles of
// 8 rows) and there are enough of them for the GPU.  One sequence of 250 tokens 9.1 against 9.0 us and the launch, 64 of 1000 25.8 against 31.8, 150 of up to
// 2000 73 against 82, 300 of up to 1000 86 against 94; the worst met, 80 of 1000 (640 units for 592 CTAs), 41 against 37.
static bool dealt_out_whole(const qcc_kv_attention_args *p, int nt)
{
    const int64_t most = nt * (((int64_t)p->table_width * p->page + SP_TOK - 1) / SP_TOK);
    return most <= 2 || (most <= 16 && (int64_t)p->seqs * p->kv_heads * 4 >= 3 * sm_count() * split_ctas(p->head_dim, nt));
}

}  // namespace qcc

using namespace qcc;

extern "C" int qcc_kv_attention_device_error(unsigned int *out) { return read_clear_device_error(out); }

extern "C" size_t qcc_nvfp4_kv_attention_workspace_bytes(int64_t rows, int seqs, int max_q, int q_heads, int kv_heads, int head_dim)
{
    if (rows < 0 || seqs < 0 || max_q < 1 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    if (many_queries(max_q, q_heads / kv_heads)) return prompt_workspace_bytes(rows, q_heads / kv_heads, seqs, head_dim);
    const int nt = row_tiles_of((int64_t)max_q * (q_heads / kv_heads));
    return (size_t)sm_count() * split_ctas(head_dim, nt) * 2 * (16 + nt * 8 * (head_dim + 2) * 4);
}

extern "C" int qcc_nvfp4_kv_attention_launches(const qcc_kv_attention_args *p)
{
    if (!p || p->kv_heads < 1 || p->seqs <= 0 || p->rows <= 0) return 0;
    const int group = p->q_heads / p->kv_heads, max_q = p->cu_q ? p->max_q : 1;
    if (many_queries(max_q, group)) return 3;
    return dealt_out_whole(p, row_tiles_of((int64_t)max_q * group)) ? 1 : 2;
}

extern "C" int qcc_nvfp4_kv_attention(const qcc_kv_attention_args *p, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!p) return QCC_ERR_ARG;
    if ((p->head_dim != 64 && p->head_dim != 128) || p->kv_heads < 1 || p->q_heads < p->kv_heads || p->q_heads % p->kv_heads || p->q_heads > 4096)
        return QCC_ERR_SHAPE;
    if ((p->page != 16 && p->page != 32 && p->page != 64 && p->page != 128) || p->seqs < 0 || p->seqs > KV_MAX_SEQS || p->rows < 0 || p->max_q < 1 ||
        p->num_pages < 0 || p->table_width < 0 || p->table_stride < 0 || (int64_t)p->table_width * p->page > 0x40000000)
        return QCC_ERR_SHAPE;
    if (p->seqs == 0 || p->rows == 0) return 0;
    if (!p->cu_q && p->rows != p->seqs) return QCC_ERR_SHAPE;
    if (!(p->scale > 0.0f)) return QCC_ERR_ARG;
    if (!p->q || (!p->cache && p->num_pages > 0) || !p->kv_lens || !p->k_outer || !p->v_outer || !p->out || (!p->table && p->table_width > 0)) return QCC_ERR_ARG;
    if (!aligned16(p->q) || !aligned16(p->cache) || !aligned16(p->out) || (p->q_stride[0] | p->q_stride[1]) % 8 != 0) return QCC_ERR_ALIGN;
    const int group = p->q_heads / p->kv_heads, max_q = p->cu_q ? p->max_q : 1, nt = row_tiles_of((int64_t)max_q * group);
    const int64_t cached = (int64_t)p->table_width * p->page;
    if (many_queries(max_q, group) ? !prompt_fits(p->rows, group, p->seqs, p->kv_heads, cached)
                                   : (int64_t)p->seqs * p->kv_heads > 0x7FFFFF00 / ((cached + SP_TOK - 1) / SP_TOK + 1))
        return QCC_ERR_SHAPE;
    if (!workspace || workspace_bytes < qcc_nvfp4_kv_attention_workspace_bytes(p->rows, p->seqs, max_q, p->q_heads, p->kv_heads, p->head_dim)) return QCC_ERR_WORKSPACE;
    if (!aligned16(workspace)) return QCC_ERR_ALIGN;
    AttnArgs g;
    g.q = static_cast<const uint16_t *>(p->q);
    g.cache = static_cast<const uint8_t *>(p->cache);
    g.table = p->table; g.kv_lens = p->kv_lens; g.cu_q = p->cu_q;
    g.k_outer = p->k_outer; g.v_outer = p->v_outer;
    g.out = static_cast<uint16_t *>(p->out);
    g.lse = p->lse;
    g.seams = static_cast<int4 *>(workspace);
    g.part = reinterpret_cast<float *>(g.seams + 2 * sm_count() * split_ctas(p->head_dim, nt));
    g.q_token = p->q_stride[0]; g.q_head = p->q_stride[1];
    g.table_stride = p->table_stride; g.num_pages = p->num_pages; g.rows = p->rows;
    g.scale_log2 = p->scale * LOG2E;
    g.seqs = p->seqs; g.width = p->table_width; g.q_heads = p->q_heads; g.kv_heads = p->kv_heads; g.group = group; g.page = p->page; g.max_q = max_q;
    g.wide = 0;
    g.whole = dealt_out_whole(p, nt);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (many_queries(max_q, group)) return prompt_launch(g, p->head_dim, workspace, st);
    if (p->head_dim == 128)
        return nt == 1 ? split_launch<128, 1>(g, st) : nt == 2 ? split_launch<128, 2>(g, st) : split_launch<128, 4>(g, st);
    return nt == 1 ? split_launch<64, 1>(g, st) : nt == 2 ? split_launch<64, 2>(g, st) : split_launch<64, 4>(g, st);
}
