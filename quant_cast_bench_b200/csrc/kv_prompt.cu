// Attention of many queries (chunks of prompts) over the paged nvfp4 key/value cache, on the tcgen05 tensor cores of sm_100a.
#include "kv_attention.cuh"
#include "tcgen05.cuh"

#include "host_util.h"

namespace qcc {

// -------------------------------------------------------------------------------------------------------------------
// Many queries: bound by the tensor cores and by the exponentials
//
// A unit is 256 rows (queries times the heads of a group, token-major) of a sequence and kv head: two row tiles of 128, whose
// softmaxes take turns with the matrix instructions.  (Of up to 128 rows both softmaxes take the one row tile, and the tiles of
// tokens in turn.)  For each tile of 128 tokens
//   S = Q K^T   128 x 128 x D, Q and K in shared memory, S in tensor memory;
//   P = exp2(S * factor - m), one thread a row, written back over S as fp16;
//   O += P V    P from tensor memory, V in shared memory (its elements contiguous: the N-major form), O in tensor memory.
// The codes of a page come by bulk copies; four warps widen them to fp16 (codes times block scales: exact) straight into the
// 128-byte swizzled rows that the instructions read, the same layout for K and V.  That happens once for 256 rows.
// q is brought to fp16 by a power of two for its row, exact for all elements above 2^-22 of the row's largest; P is rounded to fp16 (see P_LIFT);
// sums and maxima stay in fp32.  O is only rescaled when a row's maximum has grown by more than 2^8.
//
// Roles: warp 0 copies, warp 1 issues the matrix instructions, warps 4-7 widen, warps 8-11 and 12-15 are the softmax of the two
// row tiles.  All (unit, tile) pairs are numbered, by a first small kernel, and dealt out evenly to one CTA per SM, whatever the lengths and however
// many tiles the causal mask leaves a unit; a unit that spans CTAs leaves partial sums, which a third kernel joins in a fixed order.
//
// Measured, 32 heads over 8 of 128 elements: 4096 queries over 12288 tokens 600 us, 1.15 PFLOP/s (tensor cores 56 % active, exponential unit 55 %; 651 us
// and 1.60 GHz under the profiler, 1 044 000 clocks both); 16 prompts of up to 700 tokens 114 us.  A pair of row tiles and a tile of tokens takes
// about 3750 clocks, in which the exponentials and the matrix instructions of both need 2048 each by their rates; those of one row tile
// follow one another, and the two row tiles do not overlap fully.  The warps' code is close to what the instruction cache holds: loops
// that run once a part or are not on the critical path are rolled up (145 -> 111 us for the prompts of 700 tokens, when it was done).
// -------------------------------------------------------------------------------------------------------------------
constexpr int PT_THREADS = 512, PT_TOK = 128, PT_ROWS = 256, PT_RAW = 3, PT_NOTES = 8;
constexpr uint32_t PT_LAST = 256u, PT_TWO = 512u, PT_MASK = 1024u;      // notes on a tile: the last of its part; both row tiles of its
                                                                                       // unit have rows; some row does not see all its tokens
constexpr unsigned int PT_ERR = 9u;    // a barrier wait of this kernel ran out

template <int D> struct PromptCfg {
    static constexpr int BLOCKS = D / 64;                       // 64-element blocks of a row: 128 bytes of fp16
    static constexpr int TILE = BLOCKS * 128 * 128;             // 128 rows of Q, K or V as fp16
    static constexpr int RAW = PT_TOK * kv_row_bytes<D>();      // codes and scales of 128 tokens, keys or values
    static constexpr int SMEM = 1024 + 6 * TILE + PT_RAW * RAW + 256 + 128 * 8 + PT_NOTES * (8 + 8 + 48);
};

// ---- numbering: prefix[p] = tiles of all (sequence, row tile) pairs before p, times the kv heads; pairs[p] = (sequence, row tile)
struct PromptPlan {
    int32_t *count;      // [0]: pairs, [1]: those without tiles
    int2 *pairs;
    int32_t *prefix;     // pairs + 1
    int32_t *empty;      // the pairs without tiles
};
__host__ __device__ __forceinline__ int64_t prompt_max_pairs(int64_t rows, int group, int seqs) { return rows * group / PT_ROWS + seqs; }
static size_t prompt_plan_bytes(int64_t max_pairs) { return 16 + (size_t)(max_pairs + 1) * (8 + 4 + 4); }
static PromptPlan prompt_plan(void *ws, int64_t max_pairs)
{
    PromptPlan p;
    p.count = static_cast<int32_t *>(ws);
    p.pairs = reinterpret_cast<int2 *>(p.count + 4);
    p.prefix = reinterpret_cast<int32_t *>(p.pairs + max_pairs + 1);
    p.empty = p.prefix + max_pairs + 1;
    return p;
}
// tiles of row tile qt of a sequence: up to the last key that its last row sees
__device__ __forceinline__ int prompt_tiles(int n, int L, int qt, int group)
{
    const int i = (int)min((int64_t)n - 1, ((int64_t)(qt + 1) * PT_ROWS - 1) / group);
    return (max(L - n + i + 1, 0) + PT_TOK - 1) / PT_TOK;
}

// the first of them that its first row does not see whole
__device__ __forceinline__ int prompt_clear(int n, int L, int qt, int group) { return max(L - n + (int)((int64_t)qt * PT_ROWS / group) + 1, 0) / PT_TOK; }

// Sums of numbers that are not negative, 2^31 - 1 at most.  (Offsets that overlap, an error of the caller, can claim more pairs than that.)
__device__ __forceinline__ int sum_limited(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, 0x7FFFFFFFu); }
__device__ __forceinline__ int block_scan(int v, int32_t *wsum, int &all)     // inclusive; 1024 threads
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v = sum_limited(v, u);
    }
    if (lane == 31) wsum[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int u = wsum[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xFFFFFFFFu, u, o);
            if (lane >= o) u = sum_limited(u, x);
        }
        wsum[lane] = u;
    }
    __syncthreads();
    all = wsum[31];
    const int r = sum_limited(v, warp ? wsum[warp - 1] : 0);
    __syncthreads();
    return r;
}

__global__ void __launch_bounds__(1024) kv_prompt_plan_kernel(const AttnArgs g, const PromptPlan plan)
{
    __shared__ int32_t start[KV_MAX_SEQS + 1], wsum[32];
    pdl_trigger();
    pdl_wait();
    int carry = 0;
    for (int b0 = 0; b0 < g.seqs; b0 += 1024) {
        const int b = b0 + threadIdx.x;
        int q0, n = 0, L, all;
        if (b < g.seqs) seq_of(g, b, q0, n, L);
        const int v = block_scan((int)min(((int64_t)n * g.group + PT_ROWS - 1) / PT_ROWS, (int64_t)0x7FFFFFFF), wsum, all);
        if (b < g.seqs) start[b + 1] = sum_limited(carry, v);
        carry = sum_limited(carry, all);
    }
    if (threadIdx.x == 0) start[0] = 0;
    __syncthreads();
    const int pairs = min((int64_t)carry, prompt_max_pairs(g.rows, g.group, g.seqs));     // (more only if offsets overlap)
    int tiles = 0, without = 0;
    for (int p0 = 0; p0 < pairs; p0 += 1024) {
        const int p = p0 + threadIdx.x;
        int v = 0, all;
        if (p < pairs) {
            int lo = 0, up = g.seqs - 1;
            while (lo < up) {
                const int mid = (lo + up + 1) >> 1;
                if (start[mid] <= p) lo = mid; else up = mid - 1;
            }
            int q0, n, L;
            seq_of(g, lo, q0, n, L);
            plan.pairs[p] = make_int2(lo, p - start[lo]);
            v = prompt_tiles(n, L, p - start[lo], g.group) * g.kv_heads;
        }
        const int s = block_scan(v, wsum, all);
        if (p < pairs) plan.prefix[p + 1] = tiles + s;
        tiles += all;
        const bool none = p < pairs && v == 0;
        if (__syncthreads_or(none)) {
            const int e = block_scan(none ? 1 : 0, wsum, all);
            if (none) plan.empty[without + e - 1] = p;
            without += all;
        }
    }
    if (threadIdx.x == 0) {
        plan.prefix[0] = 0;
        plan.count[0] = pairs;
        plan.count[1] = without;
    }
}

// ---- the work of a CTA: parts of units
struct Part {
    int b, q0, n, L, qt, head, tiles, first, last, unit_first;     // tiles: of the unit; first, last: of this part; unit_first: flat
    int pair;
};
__device__ __forceinline__ void read_pair(const AttnArgs &g, const PromptPlan &plan, Part &s)
{
    const int2 pr = plan.pairs[s.pair];
    s.b = pr.x;
    s.qt = pr.y;
    s.tiles = (plan.prefix[s.pair + 1] - plan.prefix[s.pair]) / g.kv_heads;
    seq_of(g, s.b, s.q0, s.n, s.L);
}
// the part that starts at flat tile t, by search
__device__ __forceinline__ void find_part(const AttnArgs &g, const PromptPlan &plan, int pairs, int t, int hi, Part &s)
{
    int lo = 0, up = pairs - 1;       // the last pair with prefix <= t, which has tiles
    while (lo < up) {
        const int mid = (lo + up + 1) >> 1;
        if (plan.prefix[mid] <= t) lo = mid; else up = mid - 1;
    }
    s.pair = lo;
    read_pair(g, plan, s);
    const int start = plan.prefix[lo];
    s.head = (t - start) / s.tiles;
    s.unit_first = start + s.head * s.tiles;
    s.first = t - s.unit_first;
    s.last = min(s.tiles, s.first + hi - t);
}
// the part behind it, at t < hi: the first of the next unit
__device__ __forceinline__ void next_part(const AttnArgs &g, const PromptPlan &plan, int t, int hi, Part &s)
{
    if (++s.head == g.kv_heads) {
        s.head = 0;
        do {
            s.pair++;
            read_pair(g, plan, s);
        } while (s.tiles == 0);
    }
    s.unit_first = t;
    s.first = 0;
    s.last = min(s.tiles, hi - t);
}
template <int D> __host__ __device__ constexpr int prompt_part_floats() { return PT_ROWS * (D + 2); }

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                 "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }

__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// byte of 16-byte chunk `ch` (0 .. D / 8 - 1) of row r in a swizzled tile of 128 rows
__device__ __forceinline__ uint32_t tile_at(int r, int ch) { return (uint32_t)((ch >> 3) * 16384 + r * 128 + (((ch & 7) ^ (r & 7)) << 4)); }

// blocks of 16 elements in which some value of tokens [from, to) is NaN
template <int D>
__device__ __noinline__ uint32_t nan_blocks(const AttnArgs &g, int b, int head, int from, int to)
{
    uint32_t bits = 0;
    for (int t = from; t < to; t++) {
        const int p = t / g.page, off = t - p * g.page;
        const int64_t pg = ld_i32(g.table + b * g.table_stride + p);
        if (pg < 0 || pg >= g.num_pages) continue;
        const uint8_t *sc = g.cache + ((pg * g.kv_heads + head) * 2 + 1) * ((int64_t)g.page * kv_row_bytes<D>()) + g.page * (D / 2) + off * (D / 16);
        for (int i = 0; i < D / 16; i++) bits |= (uint32_t)((sc[i] & 0x7Fu) == 0x7Fu) << i;
    }
    return bits;
}

// 32 bytes at once where `wide` (the address is a multiple of 32), else in two pieces.  A thread of the softmax has a row of its own, so
// each piece of a warp's access is in another line, and a line takes a clock.
__device__ __forceinline__ void ld_row32(const void *p, bool wide, uint4 &a, uint4 &b)
{
    if (wide) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                     : "l"(p));
    } else {
        a = ld_v4(p);
        b = ld_v4(static_cast<const uint8_t *>(p) + 16);
    }
}
__device__ __forceinline__ void st_row32(void *p, bool wide, uint4 a, uint4 b)
{
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                     : "memory");
    } else {
        static_cast<uint4 *>(p)[0] = a;
        static_cast<uint4 *>(p)[1] = b;
    }
}

template <int D>
__global__ void __launch_bounds__(PT_THREADS, 1) kv_prompt_kernel(const __grid_constant__ AttnArgs g, const PromptPlan plan)
{
    using C = PromptCfg<D>;
    constexpr int RB = kv_row_bytes<D>();
    extern __shared__ uint8_t raw_smem[];
    // shared memory: Q of both row tiles, K and V twice, copied codes, barriers (in pairs but for the codes' three), tile notes
    const uint32_t sm = (smem_u32(raw_smem) + 1023u) & ~1023u;
    const uint32_t s_q = sm, s_k = sm + 2 * C::TILE, s_v = sm + 4 * C::TILE, s_raw = sm + 6 * C::TILE, bars = s_raw + PT_RAW * C::RAW;
    const uint32_t raw_full = bars, raw_empty = bars + 24, k_full = bars + 48, k_empty = bars + 64, v_full = bars + 80, v_empty = bars + 96, q_full = bars + 112,
                   s_full = bars + 128, p_full = bars + 144, o_done = bars + 160;
    const uint32_t s_info = bars + 176, slot = bars + 208, abort = bars + 212, s_nan = bars + 216, meeting = bars + 224, s_ml = bars + 256,      // s_info: notes of the last 8 tiles, tokens that exist, PT_LAST, PT_TWO
                   part_full = s_ml + 128 * 8, part_empty = part_full + 8 * PT_NOTES, s_part = part_empty + 8 * PT_NOTES;      // notes on parts
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    pdl_wait();      // the numbering
    const int pairs = plan.count[0], total = plan.prefix[pairs], ctas = min((int)gridDim.x, total);

    // rows that see no key, and rows behind the last sequence
    for (int e = blockIdx.x; e < plan.count[1] * 8; e += gridDim.x) {
        const int2 pr = plan.pairs[plan.empty[e >> 3]];
        int q0, n, L;
        seq_of(g, pr.x, q0, n, L);
        const int r0 = pr.y * PT_ROWS + (e & 7) * (PT_ROWS / 8), count = (int)min((int64_t)(PT_ROWS / 8), (int64_t)n * g.group - r0) * g.kv_heads;
        for (int k = warp; k < count; k += PT_THREADS / 32) {
            const int r = r0 + k / g.kv_heads, i = r / g.group;
            const int64_t at = (int64_t)(q0 + i) * g.q_heads + k % g.kv_heads * g.group + r - i * g.group;
            if (lane < D / 8) reinterpret_cast<uint4 *>(g.out + at * D)[lane] = make_uint4(0, 0, 0, 0);
            if (lane == 0 && g.lse) g.lse[at] = -INFINITY;
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
    const int lo = (int)((int64_t)total * blockIdx.x / ctas), hi = (int)((int64_t)total * (blockIdx.x + 1) / ctas);

    if (threadIdx.x == 0) {
        for (int i = 0; i < PT_RAW; i++) { mbar_init_at(raw_full + 8 * i, 1); mbar_init_at(raw_empty + 8 * i, 4); }
        for (int i = 0; i < 2; i++) {
            mbar_init_at(k_full + 8 * i, 4); mbar_init_at(k_empty + 8 * i, 1);
            mbar_init_at(v_full + 8 * i, 4); mbar_init_at(v_empty + 8 * i, 1);
            mbar_init_at(q_full + 8 * i, 4); mbar_init_at(s_full + 8 * i, 1); mbar_init_at(p_full + 8 * i, 4); mbar_init_at(o_done + 8 * i, 1);
        }
        for (int i = 0; i < PT_NOTES; i++) { mbar_init_at(part_full + 8 * i, 1); mbar_init_at(part_empty + 8 * i, 8); }
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(abort), "r"(0u) : "memory");
        mbar_init_at(meeting, 8);
        sts_u32(s_nan, 0);
        fence_barrier_init();
    }
    if (warp == 2) tmem_alloc_at(slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = lds_u32(slot);      // S0, S1 at columns 0 and 128 (P over their first halves), O0, O1 at 256 and 384

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0) {
            // ---- copies: a tile's keys, then its values
            pdl_copies_fence();
            uint32_t st = 0, ph = 1, tiles = 0;
            const int pages = PT_TOK / g.page;
            const uint32_t half = (uint32_t)(g.page * RB);
            Part s;
            find_part(g, plan, pairs, lo, hi, s);
            bool go = true;
            for (uint32_t t = lo, k = 0; go && (int)t < hi; k++) {
                mbar_wait_at(part_empty + 8 * (k & (PT_NOTES - 1)), (k / PT_NOTES & 1) ^ 1, PT_ERR, abort);
                if (__any_sync(0xFFFFFFFFu, lds_volatile(abort))) break;      // (the notes that are being read stay)
                if (lane == 0) {
                    const uint32_t at = s_part + (k & (PT_NOTES - 1)) * 48;
                    sts_v4(at, make_uint4(s.b, s.q0, s.n, s.L));
                    sts_v4(at + 16, make_uint4(s.qt, s.head, s.tiles, s.first));
                    sts_u32(at + 32, s.last);
                    mbar_arrive_at(part_full + 8 * (k & (PT_NOTES - 1)));
                }
                if (k == 0 && lane == 0) note_seam(g, s.first ? s.unit_first : -1, s.unit_first + s.tiles, total, (int)((int64_t)s.n * g.group), s.q0, s.head, s.qt * PT_ROWS);
                const int have = (s.L + g.page - 1) / g.page;
                const int32_t *row = g.table + s.b * g.table_stride;
                const uint32_t two = (int64_t)s.n * g.group - (int64_t)s.qt * PT_ROWS > 128 ? PT_TWO : 0;
                const int clear = prompt_clear(s.n, s.L, s.qt, g.group);
                for (int tile = s.first; go && tile < s.last; tile++, tiles++) {
                    const int p = tile * pages + lane;
                    int64_t pg = -1;
                    if (lane < pages && p < have) {
                        pg = ld_i32(row + p);
                        if (pg < 0 || pg >= g.num_pages) {
                            atomicMax(&g_qcc_error, QCC_DEVERR_PAGE);
                            pg = -1;
                        }
                    }
                    const int n = __popc(__ballot_sync(0xFFFFFFFFu, pg >= 0));
                    const uint8_t *src = g.cache + (pg * g.kv_heads + s.head) * (int64_t)(2 * half);
#pragma unroll 1
                    for (int w = 0; w < 2; w++) {
                        if (!(go = __all_sync(0xFFFFFFFFu, mbar_reached(raw_empty + 8 * (st), ph, PT_ERR, abort)))) break;
                        if (lane == 0) {
                            if (w == 0)
                                sts_u32(s_info + 4 * (tiles & 7), (uint32_t)min(max(s.L - tile * PT_TOK, 0), PT_TOK) | (tile + 1 == s.last ? PT_LAST : 0) | (tile >= clear ? PT_MASK : 0) | two);
                            mbar_expect_at(raw_full + 8 * st, n * half);
                        }
                        __syncwarp();
                        if (pg >= 0) bulk_load_at(s_raw + st * C::RAW + lane * half, src + w * half, half, raw_full + 8 * st);
                        if (++st == PT_RAW) { st = 0; ph ^= 1; }
                    }
                }
                t += s.last - s.first;
                if ((int)t < hi) next_part(g, plan, t, hi, s);
            }
        } else if (warp == 1 && elect_one()) {
            // ---- matrix instructions
            constexpr uint32_t id_s = (1u << 4) | ((uint32_t)(PT_TOK >> 3) << 17) | (8u << 24);
            constexpr uint32_t id_o = (1u << 4) | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24);
            // descriptors: the high words are the same (8 rows are 1024 bytes, 128-byte swizzle); the low words hold the address and, for V, whose
            // rows are tokens, the contracted side, the 16384 bytes between 64-element blocks of a row
            constexpr uint32_t high = 64u | (1u << 14) | (2u << 29);
            const uint32_t dq = (s_q >> 4) | (1u << 16), dk = (s_k >> 4) | (1u << 16), dv = (s_v >> 4) | (1024u << 16);
            uint32_t kt = 0, vt = 0, qn = 0, pn = 0;      // tiles of K and V; bit x: phase of row tile x's units, probabilities
            const auto scores = [&](int x, uint32_t kb) {
                const uint32_t a = dq + x * (C::TILE >> 4), b = dk + kb * (C::TILE >> 4);
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    const uint32_t step = (uint32_t)((k >> 2) * 1024 + (k & 3) * 2);
                    asm volatile(
                        "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
                        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(tmem + x * 128),
                        "r"(a + step), "r"(b + step), "r"(id_s), "r"(k > 0 ? 1u : 0u), "r"(high)
                        : "memory");
                }
                tc_commit_at(s_full + 8 * (x));
            };
            const auto product = [&](int x, uint32_t vb, uint32_t add) {      // add: whether O holds anything
                const uint32_t b = dv + vb * (C::TILE >> 4);
#pragma unroll
                for (int k = 0; k < PT_TOK / 16; k++)
                    asm volatile(
                        "{\n.reg .pred p;\n.reg .b64 b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 b, {%2, %5};\n"
                        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(tmem + 256 + x * 128),
                        "r"(tmem + x * 128 + k * 8), "r"(b + k * 128), "r"(id_o), "r"(k > 0 ? 1u : add), "r"(high)
                        : "memory");
                tc_commit_at(o_done + 8 * (x));
            };
            const uint32_t count = hi - lo;
            while (kt < count) {
                // a part's first scores
                mbar_wait_at(k_full + 8 * (kt & 1), (kt >> 1) & 1, PT_ERR, abort);
                uint32_t info = lds_volatile(s_info + 4 * (kt & 7));
                if (!(info & PT_TWO)) {
                    // one row tile: both softmaxes have the same rows, and take the tiles of tokens in turn
                    const auto next = [&](int x) {
                        mbar_wait_at(k_full + 8 * (kt & 1), (kt >> 1) & 1, PT_ERR, abort);
                        info = lds_volatile(s_info + 4 * (kt & 7));
                        tc_fence_after();
                        scores(x, kt & 1);
                        tc_commit_at(k_empty + 8 * (kt & 1));
                        kt++;
                    };
                    mbar_wait_at(q_full, qn & 1, PT_ERR, abort);
                    qn ^= 1;
                    next(0);
                    if (!(info & PT_LAST)) {
                        mbar_wait_at(q_full + 8, qn >> 1 & 1, PT_ERR, abort);
                        qn ^= 2;
                        next(1);
                    }
                    for (uint32_t j = 0; vt != kt && !lds_volatile(abort); j++) {
                        const int x = j & 1;
                        mbar_wait_at(v_full + 8 * (vt & 1), (vt >> 1) & 1, PT_ERR, abort);
                        mbar_wait_at(p_full + 8 * x, pn >> x & 1, PT_ERR, abort);
                        pn ^= 1u << x;
                        tc_fence_after();
                        product(x, vt & 1, j > 1);
                        tc_commit_at(v_empty + 8 * (vt & 1));
                        vt++;
                        if (!(info & PT_LAST)) next(x);
                    }
                    if (lds_volatile(abort)) break;
                    continue;
                }
#pragma unroll 1
                for (int x = 0; x < 2; x++) {
                    mbar_wait_at(q_full + 8 * x, qn >> x & 1, PT_ERR, abort);
                    qn ^= 1u << x;
                    tc_fence_after();
                    scores(x, kt & 1);
                }
                tc_commit_at(k_empty + 8 * (kt & 1));
                kt++;
                for (uint32_t o = 0;; o = 1) {
                    const bool more = !(info & PT_LAST);
                    mbar_wait_at(v_full + 8 * (vt & 1), (vt >> 1) & 1, PT_ERR, abort);
                    if (more) mbar_wait_at(k_full + 8 * (kt & 1), (kt >> 1) & 1, PT_ERR, abort);
#pragma unroll 1
                    for (int x = 0; x < 2; x++) {
                        mbar_wait_at(p_full + 8 * x, pn >> x & 1, PT_ERR, abort);
                        pn ^= 1u << x;
                        tc_fence_after();
                        product(x, vt & 1, o);
                        if (more) scores(x, kt & 1);      // over P: instructions run in order, the product above has read it
                    }
                    tc_commit_at(v_empty + 8 * (vt & 1));
                    vt++;
                    if (!more || lds_volatile(abort)) break;
                    info = lds_volatile(s_info + 4 * (kt & 7));
                    tc_commit_at(k_empty + 8 * (kt & 1));
                    kt++;
                }
                if (lds_volatile(abort)) break;
            }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ---- widening, a tile's keys, then its values.  A warp takes 8 tokens at a time: 4 threads a token (2 for D = 64), 32 elements
        // each.  The order of the lanes keeps the stores free of bank conflicts and the loads at two to a bank.
        constexpr int PIECES = D / 32;
        const int w = warp & 3;
        const int r_in = D == 128 ? (lane & 3) + ((lane >> 4) << 2) : (lane & 3) + ((lane >> 3) << 2), ch = D == 128 ? ((lane >> 2) & 1) | (((lane >> 3) & 1) << 1) : (lane >> 2) & 1;
        constexpr int PER = 32 / PIECES;         // tokens of a warp at a time
        const int shift = 31 - __clz(g.page);
        uint32_t st = 0, ph = 0, tiles = 0;
        for (const uint32_t count = hi - lo; tiles < count; tiles++) {
            const uint32_t buf = tiles & 1;
#pragma unroll 1
            for (int v = 0; v < 2; v++) {
                {
                    const uint32_t out_full = v ? v_full : k_full, out_empty = v ? v_empty : k_empty, out = v ? s_v : s_k;
                    mbar_wait_at(out_empty + 8 * (buf), ((tiles >> 1) & 1) ^ 1, PT_ERR, abort);
                    mbar_wait_at(raw_full + 8 * (st), ph, PT_ERR, abort);
                    const uint32_t info = lds_volatile(s_info + 4 * (tiles & 7));
                    const int left = info & 255;      // tokens of the tile that exist
                    const uint32_t src = s_raw + st * C::RAW, dst = out + buf * C::TILE;
                    constexpr int STEPS = 128 / (4 * PER);
                    uint4 c[STEPS];
                    uint32_t two[STEPS];
#pragma unroll
                    for (int i = 0; i < STEPS; i++) {       // all loads first: a step's stores would hold the next one's loads back
                        const int r = (i * 4 + w) * PER + r_in, off = r & (g.page - 1);
                        const uint32_t base = src + (uint32_t)((r >> shift) << shift) * RB;
                        c[i] = lds_v4(base + off * (D / 2) + ch * 16);
                        two[i] = lds_u16(base + (D / 2 << shift) + off * (D / 16) + ch * 2);
                        if (r >= left) two[i] = 0;          // whatever the slots behind the last token hold, it counts as zero
                    }
                    if (v && (info & PT_MASK)) {
                        // a NaN reaches the rows that see its token: zero here, the end of the unit sets their sums
#pragma unroll
                        for (int i = 0; i < STEPS; i++) {
                            const bool a = (two[i] & 0x7Fu) == 0x7Fu, b = (two[i] & 0x7F00u) == 0x7F00u;
                            if (a || b) sts_u32(s_nan, 1);
                            if (a) two[i] &= 0xFF00u;
                            if (b) two[i] &= 0xFFu;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < STEPS; i++) {
                        const int r = (i * 4 + w) * PER + r_in;
                        const uint32_t sc = e4m3x2_to_half2(two[i]), s0 = __byte_perm(sc, sc, 0x1010), s1 = __byte_perm(sc, sc, 0x3232);
                        const uint32_t word[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            uint32_t h[4];
                            e2m1x8_to_half(word[j], h);
#pragma unroll
                            for (int u = 0; u < 4; u++) h[u] = hmul2_bits(h[u], j < 2 ? s0 : s1);
                            sts_v4(dst + tile_at(r, ch * 4 + j), make_uint4(h[0], h[1], h[2], h[3]));
                        }
                    }
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_at(raw_empty + 8 * st);
                        mbar_arrive_at(out_full + 8 * buf);
                    }
                    if (++st == PT_RAW) { st = 0; ph ^= 1; }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        // ---- softmax of row tile x, one thread a row
        const int x = (warp - 8) >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21, t_s = tmem + lanes + x * 128, t_o = tmem + lanes + 256 + x * 128;
        const float k_outer = *g.k_outer, v_outer = *g.v_outer;
        uint32_t sn = 0, on = 0;        // scores, products so far
        float factor = 0.0f;
        bool placed = false;            // q of the part is in place already
        // the note on part k; after the wait for it, that it is there (not so when some wait has run out)
        const auto noted = [&](uint32_t k) {
            mbar_wait_at(part_full + 8 * (k & (PT_NOTES - 1)), k / PT_NOTES & 1, PT_ERR, abort);
            return (bool)__all_sync(0xFFFFFFFFu, lds_volatile(abort) == 0);
        };
        const auto read_note = [&](uint32_t k) {
            Part s;
            const uint32_t note = s_part + (k & (PT_NOTES - 1)) * 48;
            const uint4 a = lds_v4(note), b = lds_v4(note + 16);
            s.b = a.x; s.q0 = a.y; s.n = a.z; s.L = a.w;
            s.qt = b.x; s.head = b.y; s.tiles = b.z; s.first = b.w;
            s.last = lds_volatile(note + 32);
            return s;
        };
        // both softmaxes meet (a wait with a limit, as all are)
        uint32_t met = 0;
        const auto meet = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive_at(meeting);
            mbar_wait_at(meeting, met++ & 1, PT_ERR, abort);
        };
        // This thread's row of a part.  Both row tiles have rows: one for each softmax; one has: both softmaxes take it, and the
        // tiles of tokens in turn.
        struct Rows {
            bool two, live;
            int first, i, h, limit;      // first tile; query, head, keys that the row sees
        };
        const auto rows_of = [&](const Part &s) {
            Rows a;
            const int64_t rows = (int64_t)s.n * g.group, r0 = (int64_t)s.qt * PT_ROWS;
            a.two = rows - r0 > 128;
            const int64_t r = r0 + (a.two ? x * 128 : 0) + row;
            a.first = a.two ? s.first : s.first + x;
            a.live = r < rows;
            a.i = a.live ? (int)r / g.group : 0;
            a.h = s.head * g.group + (a.live ? (int)r - a.i * g.group : 0);
            a.limit = a.live ? s.L - s.n + a.i + 1 : 0;
            return a;
        };
        // q of this thread's row, into shared memory; its factor score -> log2 units
        const auto place_q = [&](const Part &s, const Rows &at) {
            uint4 w[D / 8];
            uint32_t acc = 0;
            const uint16_t *src = g.q + (int64_t)(s.q0 + at.i) * g.q_token + at.h * g.q_head;
#pragma unroll
            for (int j = 0; j < D / 8; j++) w[j] = make_uint4(0, 0, 0, 0);
            if (at.live) {
#pragma unroll
                for (int j = 0; j < D / 8; j += 2) ld_row32(src + 8 * j, g.wide & 1, w[j], w[j + 1]);
            }
#pragma unroll
            for (int j = 0; j < D / 8; j++) {
                acc = absmax2_acc(absmax2_acc(absmax2_acc(absmax2_acc(acc, w[j].x), w[j].y), w[j].z), w[j].w);
            }
            float mult, back;
            q_power(f2u(hmax_halves_f32(acc)), mult, back);
            const uint32_t dst = s_q + x * C::TILE;
#pragma unroll
            for (int j = 0; j < D / 8; j++)
                sts_v4(dst + tile_at(row, j),
                       make_uint4(pack_half2(bf16lo(w[j].x) * mult, bf16hi(w[j].x) * mult), pack_half2(bf16lo(w[j].y) * mult, bf16hi(w[j].y) * mult),
                                  pack_half2(bf16lo(w[j].z) * mult, bf16hi(w[j].z) * mult), pack_half2(bf16lo(w[j].w) * mult, bf16hi(w[j].w) * mult)));
            proxy_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive_at(q_full + 8 * x);
            const float f = back * (g.scale_log2 * k_outer);
            return f < 1e-37f ? 1e-37f : f;       // not zero: -inf of a hidden key has to stay
        };
        for (int t = lo, k = 0; t < hi; k++) {
            if (!noted(k)) break;
            int tile, last, step, limit;
            {
                const Part s = read_note(k);
                const Rows at = rows_of(s);
                tile = at.first;
                last = s.last;
                step = at.two ? 1 : 2;
                limit = at.limit;
                if (tile < last && !placed) factor = place_q(s, at);
                t += s.last - s.first;
            }
            const bool idle = tile >= last;
            const float scale_in = factor;
            if (!idle) {
                placed = false;
                bool any = false;               // O holds products of this part
                float m = -INFINITY, l = 0.0f;
                for (; tile < last; tile += step) {
                    mbar_wait_at(s_full + 8 * (x), sn++ & 1, PT_ERR, abort);
                    tc_fence_after();
                    uint32_t v[4][32];
#pragma unroll
                    for (int c = 0; c < 4; c++) tmem_ld32(t_s + 32 * c, v[c]);
                    tmem_wait_ld();
                    const int see = limit - tile * PT_TOK;       // columns that the row sees
                    if (__any_sync(0xFFFFFFFFu, see < PT_TOK)) {
#pragma unroll
                        for (int c = 0; c < 4; c++)
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (32 * c + j >= see) v[c][j] = 0xFF800000u;
                    }
                    float top[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) top[c] = fmaxf(u2f(v[c][0]), u2f(v[c][1]));
#pragma unroll
                    for (int j = 2; j < 32; j += 2)
#pragma unroll
                        for (int c = 0; c < 4; c++) top[c] = max3(top[c], u2f(v[c][j]), u2f(v[c][j + 1]));
                    const float most = fmaxf(max3(top[0], top[1], top[2]), top[3]);
                    const bool grow = fmaf(most, scale_in, -m) > P_MOST;      // (from -inf: always, once the row sees a key; one rounding, as below)
                    if (__any_sync(0xFFFFFFFFu, grow)) {
                        const float up = grow ? reference_of(most, scale_in) : m, a = grow ? ex2(m - up) : 1.0f;
                        m = up;
                        l *= a;
                        if (any) {
                            mbar_wait_at(o_done + 8 * x, (on - 1) & 1, PT_ERR, abort);
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                tmem_ld16(t_o + c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int j = 0; j < 16; j++) o[j] = f2u(u2f(o[j]) * a);
                                tmem_st16(t_o + c, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    const uint64_t factor2 = pack2(scale_in, scale_in), base2 = pack2(-base, -base);
                    uint64_t sum[2] = {0, 0};
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        uint32_t p[16];
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            // (scale_in is finite and positive: -inf stays -inf and exp2 gives 0)
                            float e0, e1;
                            unpack2(fma2(pack2(u2f(v[c][2 * j]), u2f(v[c][2 * j + 1])), factor2, base2), e0, e1);
                            e0 = ex2(e0);
                            e1 = ex2(e1);
                            sum[j & 1] = add2(sum[j & 1], pack2(e0, e1));
                            p[j] = pack_half2(e0, e1);
                        }
                        tmem_st16(t_s + 16 * c, p);
                    }
                    {
                        float a, b;
                        unpack2(add2(sum[0], sum[1]), a, b);
                        l += a + b;
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_at(p_full + 8 * x);
                    on++;
                    any = true;
                }
                const Part s = read_note(k);      // (again: it would take up registers that the loop needs)
                const Rows at = rows_of(s);
                __syncwarp();
                if (lane == 0) mbar_arrive_at(part_empty + 8 * (k & (PT_NOTES - 1)));
                const bool whole = s.first == 0 && s.last == s.tiles, join = !at.two && s.last - s.first > 1;
                if (!join && t < hi && noted(k + 1)) {
                    // q of the next part, whose first scores are then worked out behind the end of this one (one that joins needs the
                    // space of q)
                    const Part n = read_note(k + 1);
                    const Rows to = rows_of(n);
                    if (to.first < n.last) {
                        factor = place_q(n, to);
                        placed = true;
                    }
                }
                mbar_wait_at(o_done + 8 * (x), (on - 1) & 1, PT_ERR, abort);
                tc_fence_after();
                float mine = 1.0f, others = 0.0f;         // weights of this softmax's sums and of the other's
                if (join) {
                    // the second softmax hands its sums over in Q's place, column by column
                    meet();                // (both are done with Q)
                    if (x) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(t_o + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; j++) sts_u32(s_q + ((c + j) * 128 + row) * 4, o[j]);
                        }
                        sts_u32(s_ml + row * 8, f2u(m));
                        sts_u32(s_ml + row * 8 + 4, f2u(l));
                        tc_fence_before();
                    }
                    meet();
                    if (x) {
                        meet();            // (the sums are read)
                        continue;
                    }
                    const float m1 = u2f(lds_volatile(s_ml + row * 8)), l1 = u2f(lds_volatile(s_ml + row * 8 + 4)), up = fmaxf(m, m1);
                    mine = m == -INFINITY ? 1.0f : ex2(m - up);
                    others = m1 == -INFINITY ? 1.0f : ex2(m1 - up);
                    m = up;
                    l = l * mine + l1 * others;
                }
                // 16-element blocks of the row that a NaN of a masked tile makes NaN (once this CTA has met one)
                uint32_t nan = 0;
                if (lds_volatile(s_nan)) nan = nan_blocks<D>(g, s.b, s.head, max(s.first, prompt_clear(s.n, s.L, s.qt, g.group)) * PT_TOK, min(limit, s.last * PT_TOK));
                const float scale = l == 0.0f ? 0.0f : __fdividef(v_outer, l);
                const int64_t to = (int64_t)(s.q0 + at.i) * g.q_heads + at.h;
                float *part = g.part + (size_t)(2 * blockIdx.x + (k ? 1 : 0)) * prompt_part_floats<D>();
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t o[16];
                    tmem_ld16(t_o + c, o);
                    tmem_wait_ld();
                    if (join) {
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = f2u(u2f(o[j]) * mine + u2f(lds_volatile(s_q + ((c + j) * 128 + row) * 4)) * others);
                    }
                    if (nan >> (c / 16) & 1u) {
#pragma unroll
                        for (int j = 0; j < 16; j++) o[j] = 0x7FFFFFFFu;
                    }
                    if (whole) {
                        uint32_t y[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(l == 0.0f ? 0.0f : u2f(o[2 * j]) * scale, l == 0.0f ? 0.0f : u2f(o[2 * j + 1]) * scale);
                            y[j] = *reinterpret_cast<const uint32_t *>(&b);
                        }
                        if (at.live) {
                            st_row32(g.out + to * D + c, g.wide & 2, make_uint4(y[0], y[1], y[2], y[3]), make_uint4(y[4], y[5], y[6], y[7]));
                        }
                    } else {
                        float *dst = part + (x * 128 + row) * D + c;
#pragma unroll
                        for (int j = 0; j < 16; j += 8)
                            st_row32(dst + j, g.wide & 4, make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]), make_uint4(o[j + 4], o[j + 5], o[j + 6], o[j + 7]));
                    }
                }
                if (!whole) reinterpret_cast<float2 *>(part + PT_ROWS * D)[x * 128 + row] = make_float2(m, l);
                else if (at.live && g.lse) g.lse[to] = l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2;
                tc_fence_before();       // the next unit's products write O
                if (join) meet();
            } else {
                __syncwarp();
                if (lane == 0) mbar_arrive_at(part_empty + 8 * (k & (PT_NOTES - 1)));
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    settle(abort);
    if (warp == 2) {
        tc_fence_after();
        tmem_free(tmem, 512);
    }
}

bool prompt_fits(int64_t rows, int group, int seqs, int kv_heads, int64_t cached)
{
    return prompt_max_pairs(rows, group, seqs) * kv_heads <= 0x7FFFFFFF / ((cached + PT_TOK - 1) / PT_TOK + 1);
}
size_t prompt_workspace_bytes(int64_t rows, int group, int seqs, int head_dim)
{
    return (prompt_plan_bytes(prompt_max_pairs(rows, group, seqs)) + 31) / 32 * 32 + (size_t)2 * sm_count() * (16 + PT_ROWS * (head_dim + 2) * 4);
}

template <int D>
static int launch(AttnArgs g, void *ws, cudaStream_t st)
{
    using C = PromptCfg<D>;
    static PerDeviceFlag done;
    const int dev = current_device_slot();
    if (dev < 0) return QCC_ERR_ARG;
    if (!done.get(dev)) {
        cudaError_t e = cudaFuncSetAttribute(kv_prompt_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        // the warps re-divide the registers of the launch, 256 threads with 72 and 256 with 184: it has to bring as many
        cudaFuncAttributes at;
        if ((e = cudaFuncGetAttributes(&at, kv_prompt_kernel<D>)) != cudaSuccess) return (int)e;
        if (at.numRegs * PT_THREADS < 256 * (72 + 184)) return (int)cudaErrorInvalidConfiguration;
        done.set(dev);
    }
    const int64_t max_pairs = prompt_max_pairs(g.rows, g.group, g.seqs);
    const PromptPlan plan = prompt_plan(ws, max_pairs);
    const int grid = sm_count();
    g.seams = reinterpret_cast<int4 *>(static_cast<uint8_t *>(ws) + (prompt_plan_bytes(max_pairs) + 31) / 32 * 32);
    g.part = reinterpret_cast<float *>(g.seams + 2 * grid);
    const auto by32 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; };
    g.wide = (by32(g.q) && g.q_token % 16 == 0 && g.q_head % 16 == 0 ? 1 : 0) | (by32(g.out) ? 2 : 0) | (by32(g.part) ? 4 : 0);
    cudaError_t e = launch_maybe_pdl(kv_prompt_plan_kernel, dim3(1), dim3(1024), 0, st, true, g, plan);
    if (e != cudaSuccess) return (int)e;
    e = launch_maybe_pdl(kv_prompt_kernel<D>, dim3(grid), dim3(PT_THREADS), C::SMEM, st, true, g, plan);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_maybe_pdl(kv_join_kernel<D, 1, 16, 256>, dim3(grid, PT_ROWS / 16), dim3(256), 0, st, true, g, grid, PT_ROWS);
}

int prompt_launch(const AttnArgs &g, int head_dim, void *ws, cudaStream_t st)
{
    return head_dim == 128 ? launch<128>(g, ws, st) : launch<64>(g, ws, st);
}

}  // namespace qcc

extern "C" int qcc_kv_prompt_device_error(unsigned int *out) { return qcc::read_clear_device_error(out); }
