// 8-bit integer linear layer, sm_100a: the int8 cast of activations with one scale per token, and the product of two int8
// matrices with a scale per token and per output channel.
//
//   cast:    scale_m = max(max_k |x_mk|, bf16(1e-12)) / 127,  q = rne(x * (1 / scale))          (the recipe of rowwise_fp8_f,
//            G:301-307, with 127 for the fp8 maximum)
//   product: y_mn = (sum_k a_mk b_nk) * sa_m * sb_n + bias_n, the sum exact in 32-bit integers
#include <cuda_fp16.h>

#include "tcgen05.cuh"

#include "host_util.h"

namespace qcc {

// ---------------------------------------------------------------------------------------------
// cast
// ---------------------------------------------------------------------------------------------
constexpr int I8_THREADS = 256;

// max(|a|, |b|) of packed bf16 pairs; a NaN wins, as it does in torch.amax: a row with a NaN gets a NaN scale, so the row
// of any product of it is NaN too (8-bit codes alone could not carry it)
__device__ __forceinline__ uint32_t absmax2_nan(uint32_t acc, uint32_t w)
{
    __nv_bfloat162 a = *reinterpret_cast<__nv_bfloat162 *>(&acc), b = *reinterpret_cast<__nv_bfloat162 *>(&w);
    __nv_bfloat162 r = __hmax2_nan(a, __habs2(b));
    return *reinterpret_cast<uint32_t *>(&r);
}
// non-negative floats and NaN (any payload, sign cleared) order like integers
__device__ __forceinline__ uint32_t halves_max_bits(uint32_t acc) { return max(acc << 16, acc & 0x7FFF0000u); }

__device__ __forceinline__ float int8_scale_from_amax(float amax, bool recip)
{
    const float a = amax < u2f(0x2B8D0000u) ? u2f(0x2B8D0000u) : amax;   // bf16(1e-12); a NaN stays
    return div_by_const(a, 127.0f, recip);
}
// |v| <= 127: adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low byte
__device__ __forceinline__ uint32_t int8_byte(float x, float inv) { return f2u(__fadd_rn(__fmul_rn(x, inv), 12582912.0f)); }
__device__ __forceinline__ uint32_t int8x4(uint32_t w0, uint32_t w1, float inv)
{
    const uint32_t a = __byte_perm(int8_byte(bf16lo(w0), inv), int8_byte(bf16hi(w0), inv), 0x0040);
    const uint32_t b = __byte_perm(int8_byte(bf16lo(w1), inv), int8_byte(bf16hi(w1), inv), 0x0040);
    return __byte_perm(a, b, 0x5410);
}

// One CTA per row.  The row stays in registers (CH 16-byte pieces a thread) between its maximum and the cast, so x is read
// once; CH = 0: rows too long for that, or not a multiple of 8 elements, are read twice (the second time from L2), an element at a time.
template <int CH>
__global__ void __launch_bounds__(I8_THREADS) int8_rowwise_kernel(const uint16_t *x, int64_t N, uint8_t *q,
                                                                  float *scale, int recip_div)
{
    pdl_trigger();
    pdl_wait();
    const int64_t row = blockIdx.x;
    const uint16_t *xr = x + row * N;
    uint8_t *qr = q + row * N;
    const int64_t nchunk = N >> 3;
    uint32_t acc = 0;
    uint4 v[CH > 0 ? CH : 1];
    if (CH > 0) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int64_t k = threadIdx.x + (int64_t)c * I8_THREADS;
            v[c] = k < nchunk ? ld_once_v4(reinterpret_cast<const uint4 *>(xr) + k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < CH; c++) acc = absmax2_nan(absmax2_nan(absmax2_nan(absmax2_nan(acc, v[c].x), v[c].y), v[c].z), v[c].w);
    } else {
        for (int64_t k = threadIdx.x; k < N; k += I8_THREADS) acc = absmax2_nan(acc, xr[k]);
    }
    uint32_t m = halves_max_bits(acc);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    __shared__ uint32_t sm[I8_THREADS / 32];
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = m;
    __syncthreads();
    m = 0;
#pragma unroll
    for (int w = 0; w < I8_THREADS / 32; w++) m = max(m, sm[w]);
    const float s = int8_scale_from_amax(u2f(m), recip_div != 0);
    if (threadIdx.x == 0) scale[row] = s;
    const float inv = __fdiv_rn(1.0f, s);
    if (CH > 0) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int64_t k = threadIdx.x + (int64_t)c * I8_THREADS;
            if (k < nchunk) reinterpret_cast<uint2 *>(qr)[k] = make_uint2(int8x4(v[c].x, v[c].y, inv), int8x4(v[c].z, v[c].w, inv));
        }
    } else {
        for (int64_t k = threadIdx.x; k < N; k += I8_THREADS) qr[k] = (uint8_t)int8_byte(u2f((uint32_t)xr[k] << 16), inv);
    }
}

// ---------------------------------------------------------------------------------------------
// product
// ---------------------------------------------------------------------------------------------
// tcgen05.mma kind::i8 on tiles of 128 output channels (the M side of the instruction) by BN tokens, K in blocks of 128 bytes
// staged by TMA.  The tokens are on the N side because it goes down to 16: a decode batch wastes little of the instruction.
// Where there are fewer tiles than SMs, the CTAs of a cluster share out K and add their sums up through each other's shared
// memory; whole numbers, so in any order the same.
//
// Measured: 8192^3 351 us, 3.13 POP/s, tensor cores 92 % active; 2000 x 4096 x 7168 39 us, 3.0 POP/s; 64 x 14336 x 4096 9.7 us, again and again on the
// same weights (59 MB, less than L2).  Rows of K that are no multiple of 128 bytes cost a second line a row: K = 2064 21 us where 2048 takes 14.
constexpr int MM_BM = 128, MM_BK = 128, MM_THREADS = 384;
constexpr unsigned int MM_ERR = 7;   // a barrier wait of the product ran out

template <int BN> struct MmCfg {
    static constexpr int STAGE = (MM_BM + BN) * MM_BK;
    static constexpr int STAGES = BN >= 224 ? 4 : BN >= 160 ? 5 : BN >= 96 ? 6 : 8;
    static constexpr int RED = MM_BM * BN * 4;                              // sums of one CTA (split form), in the stages' memory
    static constexpr int BODY = STAGE * STAGES > RED ? STAGE * STAGES : RED;
    static constexpr int PARTS = BN >= 64 ? 2 : 1;                          // epilogue warps per 32 channels, each with a share of the tokens
    static constexpr int TURN = 4 * PARTS * 16 * 32 * 4;                    // 16 tokens x 32 channels of each epilogue warp
    static constexpr int SMEM = 1024 + BODY + TURN + BN * 4 * 2 + 256;
};

struct MmArgs {
    const float *sa, *sb;
    const uint16_t *bias;
    void *out;
    int M, N, kblocks, tiles_n, tiles_m, splits, piece;      // piece: log2 of the bytes that every row of the output is aligned to, up to 16
};

template <int OUT> struct OutType;
template <> struct OutType<QCC_OUT_BF16> { using T = uint16_t; static __device__ __forceinline__ T of(float y) { return __bfloat16_as_ushort(__float2bfloat16_rn(y)); } };
template <> struct OutType<QCC_OUT_F16> { using T = uint16_t; static __device__ __forceinline__ T of(float y) { return __half_as_ushort(__float2half_rn(y)); } };
template <> struct OutType<QCC_OUT_F32> { using T = float; static __device__ __forceinline__ T of(float y) { return y; } };

// the scales in fp32, a multiplication each, then the bias
__device__ __forceinline__ float mm_scaled(int32_t sum, float sa, float sb, bool has_bias, float bias)
{
    const float y = __fmul_rn(__fmul_rn((float)sum, sa), sb);
    return has_bias ? __fadd_rn(y, bias) : y;
}

// groups of 8 token tiles share the weights that pass through L2
__device__ __forceinline__ void mm_tile(const MmArgs &g, int t, int &tn, int &tm)
{
    const int per = 8 * g.tiles_n, grp = t / per, first = grp * 8, rows = min(8, g.tiles_m - first), r = t - grp * per;
    tm = first + r % rows;
    tn = r / rows;
}

// 16 tokens x 32 channels from shared memory to the output, in pieces of 2^LOG bytes: neighbouring lanes have neighbouring pieces of a row
template <int LOG, typename T>
__device__ __forceinline__ void mm_write(const MmArgs &g, uint32_t turn, int64_t m0, int n0, int lane)
{
    constexpr int ROW = 32 * sizeof(T), PIECES = ROW >> LOG, EACH = 16 * PIECES / 32;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = i * 32 + lane, tok = e / PIECES, at = (e % PIECES) << LOG, n = n0 + at / (int)sizeof(T);
        if (m0 + tok >= g.M || n >= g.N) continue;
        uint8_t *dst = static_cast<uint8_t *>(g.out) + ((m0 + tok) * g.N + n) * (int64_t)sizeof(T);
        const uint32_t src = turn + tok * ROW + at;
        if (LOG == 4) *reinterpret_cast<uint4 *>(dst) = lds_v4(src);
        else if (LOG == 3) *reinterpret_cast<uint2 *>(dst) = lds_v2(src);
        else if (LOG == 2) {
            uint32_t v;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(src));
            *reinterpret_cast<uint32_t *>(dst) = v;
        } else {
            uint16_t v;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(src));
            *reinterpret_cast<uint16_t *>(dst) = v;
        }
    }
}

template <int BN, bool SPLIT, int OUT>
__global__ void __launch_bounds__(MM_THREADS, 1) int8_mm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                const MmArgs g)
{
    using C = MmCfg<BN>;
    using T = typename OutType<OUT>::T;
    extern __shared__ uint8_t raw[];
    const uint32_t stages = (smem_u32(raw) + 1023u) & ~1023u, turns = stages + C::BODY, s_sa = turns + C::TURN;       // s_sa: 2 x BN token scales
    const uint32_t full = s_sa + 2 * BN * 4, empty = full + 8 * C::STAGES, acc_full = empty + 8 * C::STAGES, acc_empty = acc_full + 16, slot = acc_empty + 16,
                   abort = slot + 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr uint32_t ACC_COLS = BN <= 32 ? 32 : BN <= 64 ? 64 : BN <= 128 ? 128 : 256, TMEM_COLS = SPLIT ? ACC_COLS : 2 * ACC_COLS;

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        for (int i = 0; i < C::STAGES; i++) { mbar_init_at(full + 8 * i, 1); mbar_init_at(empty + 8 * i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init_at(acc_full + 8 * i, 1); mbar_init_at(acc_empty + 8 * i, 4 * C::PARTS); }
        sts_u32(abort, 0);
        fence_barrier_init();
    }
    if (warp == 2) tmem_alloc_at(slot, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    pdl_wait();
    const uint32_t tmem = lds_volatile(slot);
    const int total = g.tiles_n * g.tiles_m;
    // SPLIT: the CTAs of a cluster take one tile together, each a share of the K blocks
    const int rank = SPLIT ? blockIdx.x % g.splits : 0;
    const int kb0 = SPLIT ? (int)((int64_t)g.kblocks * rank / g.splits) : 0, kb1 = SPLIT ? (int)((int64_t)g.kblocks * (rank + 1) / g.splits) : g.kblocks;
    const int t0 = SPLIT ? blockIdx.x / g.splits : blockIdx.x, step = SPLIT ? total : gridDim.x;

    if (warp == 0) {
        if (elect_one()) {
            pdl_copies_fence();
            uint32_t s = 0, ph = 1;
            bool go = true;
            for (int t = t0; go && t < total; t += step) {
                int tn, tm;
                mm_tile(g, t, tn, tm);
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!(go = mbar_reached(empty + 8 * s, ph, MM_ERR, abort))) break;
                    const uint32_t p = stages + s * C::STAGE, bar = full + 8 * s;
                    mbar_expect_at(bar, C::STAGE);
                    tma_load_2d_at(p, &map_w, bar, kb * MM_BK, tn * MM_BM);
                    tma_load_2d_at(p + MM_BM * MM_BK, &map_x, bar, kb * MM_BK, tm * BN);
                    if (++s == C::STAGES) { s = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(MM_BM >> 4) << 24);
            constexpr uint32_t high = 64u | (1u << 14) | (2u << 29);      // high words of the descriptors: 8 rows are 1024 bytes, 128-byte swizzle
            uint32_t s = 0, ph = 0, n = 0;
            bool go = true;
            for (int t = t0; go && t < total; t += step, n++) {
                const uint32_t acc = SPLIT ? 0 : n & 1, aph = SPLIT ? 0 : (n >> 1) & 1;
                if (!mbar_reached(acc_empty + 8 * acc, aph ^ 1, MM_ERR, abort)) break;
                tc_fence_after();
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!(go = mbar_reached(full + 8 * s, ph, MM_ERR, abort))) break;
                    tc_fence_after();
                    const uint32_t da = ((stages + s * C::STAGE) >> 4) | (1u << 16), db = da + (MM_BM * MM_BK >> 4);
#pragma unroll
                    for (int k = 0; k < MM_BK / 32; k++)
                        asm volatile(
                            "{\n.reg .pred p;\n.reg .b64 a, b;\nsetp.ne.b32 p, %4, 0;\nmov.b64 a, {%1, %5};\nmov.b64 b, {%2, %5};\n"
                            "tcgen05.mma.cta_group::1.kind::i8 [%0], a, b, %3, p;\n}\n" ::"r"(tmem + acc * ACC_COLS),
                            "r"(da + 2 * k), "r"(db + 2 * k), "r"(idesc), "r"((kb > kb0 || k > 0) ? 1u : 0u), "r"(high)
                            : "memory");
                    tc_commit_at(empty + 8 * s);
                    if (++s == C::STAGES) { s = 0; ph ^= 1; }
                }
                tc_commit_at(acc_full + 8 * acc);
            }
        }
    } else if (warp >= 4 && warp < 4 + 4 * C::PARTS) {
        constexpr int EPI = 128 * C::PARTS, SHARE = BN / C::PARTS;
        const int w = warp & 3, part = (warp - 4) >> 2, et = threadIdx.x - 128;
        const uint32_t turn = turns + (warp - 4) * (16 * 32 * 4);
        uint32_t n = 0;
        for (int t = t0; t < total; t += step, n++) {
            int tn, tm;
            mm_tile(g, t, tn, tm);
            const uint32_t acc = SPLIT ? 0 : n & 1, aph = SPLIT ? 0 : (n >> 1) & 1;
            const int n0 = tn * MM_BM + w * 32, ch = n0 + lane;
            const uint32_t sa = s_sa + acc * BN * 4;
            for (int i = et; i < BN; i += EPI) sts_u32(sa + 4 * i, tm * BN + i < g.M ? f2u(g.sa[(int64_t)tm * BN + i]) : 0);
            named_barrier(1, EPI);
            const bool has_bias = g.bias != nullptr;
            const float sb = ch < g.N ? g.sb[ch] : 0.0f, bias = has_bias && ch < g.N ? u2f((uint32_t)g.bias[ch] << 16) : 0.0f;
            mbar_wait_at(acc_full + 8 * acc, aph, MM_ERR, abort);
            tc_fence_after();
#pragma unroll 1
            for (int c = part * SHARE; c < (part + 1) * SHARE; c += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + ((uint32_t)w << 21) + acc * ACC_COLS + c, r);
                tmem_wait_ld();
                if (SPLIT) {
#pragma unroll
                    for (int j = 0; j < 16; j++) sts_u32(stages + (uint32_t)((c + j) * MM_BM + w * 32 + lane) * 4, r[j]);
                    continue;
                }
                if (c + 16 == (part + 1) * SHARE) {                 // the accumulator is in registers: the next tile may have it
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_at(acc_empty + 8 * acc);
                }
                const int64_t m0 = (int64_t)tm * BN + c;
                if (m0 >= g.M) continue;
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const uint4 q = lds_v4(sa + 4 * (c + j));
                    const float s4[4] = {u2f(q.x), u2f(q.y), u2f(q.z), u2f(q.w)};
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const T y = OutType<OUT>::of(mm_scaled((int32_t)r[j + u], s4[u], sb, has_bias, bias));
                        const uint32_t at = turn + ((j + u) * 32 + lane) * (uint32_t)sizeof(T);
                        if (sizeof(T) == 4) sts_u32(at, *reinterpret_cast<const uint32_t *>(&y));
                        else asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(*reinterpret_cast<const uint16_t *>(&y)) : "memory");
                    }
                }
                __syncwarp();
                if (g.piece == 4) mm_write<4, T>(g, turn, m0, n0, lane);
                else if (g.piece == 3) mm_write<3, T>(g, turn, m0, n0, lane);
                else if (g.piece == 2 || sizeof(T) == 4) mm_write<2, T>(g, turn, m0, n0, lane);
                else mm_write<sizeof(T) == 4 ? 2 : 1, T>(g, turn, m0, n0, lane);
                __syncwarp();
            }
        }
    }
    __syncwarp();
    if (SPLIT) {
        // every CTA of the cluster adds up its share of the tokens from all shares of K, four channels a thread
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        int tn, tm;
        mm_tile(g, t0, tn, tm);
        const int rows = min(BN, g.M - tm * BN), lo = rows * rank / g.splits, hi = rows * (rank + 1) / g.splits;
        const int n = tn * MM_BM + lane * 4;
        const bool has_bias = g.bias != nullptr;
        float sb[4], bias[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            sb[u] = n + u < g.N ? g.sb[n + u] : 0.0f;
            bias[u] = has_bias && n + u < g.N ? u2f((uint32_t)g.bias[n + u] << 16) : 0.0f;
        }
        for (int i = lo + warp; i < hi; i += MM_THREADS / 32) {
            int4 sum = make_int4(0, 0, 0, 0);
#pragma unroll 8
            for (int p = 0; p < g.splits; p++) {
                uint32_t addr;
                int4 v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(stages + (uint32_t)(i * MM_BM + lane * 4) * 4u), "r"(p));
                asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
            const int s4[4] = {sum.x, sum.y, sum.z, sum.w};
            const float sa = u2f(lds_volatile(s_sa + 4 * i));
            T *dst = static_cast<T *>(g.out) + ((int64_t)tm * BN + i) * g.N + n;
            T y[4];
#pragma unroll
            for (int u = 0; u < 4; u++) y[u] = OutType<OUT>::of(mm_scaled(s4[u], sa, sb[u], has_bias, bias[u]));
            if (n < g.N && (1 << g.piece) >= 4 * (int)sizeof(T)) {      // (then N is a multiple of 4)
                if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(y);
                else *reinterpret_cast<uint2 *>(dst) = make_uint2(reinterpret_cast<const uint32_t *>(y)[0], reinterpret_cast<const uint32_t *>(y)[1]);
            } else {
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (n + u < g.N) dst[u] = y[u];
            }
        }
        // no CTA leaves while another may still read its sums
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    settle(abort);
    if (warp == 2) {
        tc_fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
}

template <int BN, bool SPLIT, int OUT>
static int mm_launch(const CUtensorMap &mw, const CUtensorMap &mx, const MmArgs &g, cudaStream_t st)
{
    using C = MmCfg<BN>;
    static PerDeviceFlag done;
    const int dev = current_device_slot();
    if (dev < 0) return QCC_ERR_ARG;
    if (!done.get(dev)) {
        cudaError_t e = cudaFuncSetAttribute(int8_mm_kernel<BN, SPLIT, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        done.set(dev);
    }
    const int total = g.tiles_n * g.tiles_m;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = SPLIT ? total * g.splits : (total < sm_count() ? total : sm_count());
    cfg.blockDim = MM_THREADS;
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = SPLIT ? g.splits : 1;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = SPLIT ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, int8_mm_kernel<BN, SPLIT, OUT>, mw, mx, g);
}
template <int BN, bool CAN_SPLIT = true>
static int mm_dispatch(const CUtensorMap &mw, const CUtensorMap &mx, const MmArgs &g, int out, cudaStream_t st)
{
    if constexpr (CAN_SPLIT)
        if (g.splits > 1)
            return out == QCC_OUT_BF16 ? mm_launch<BN, true, QCC_OUT_BF16>(mw, mx, g, st)
                   : out == QCC_OUT_F16 ? mm_launch<BN, true, QCC_OUT_F16>(mw, mx, g, st) : mm_launch<BN, true, QCC_OUT_F32>(mw, mx, g, st);
    return out == QCC_OUT_BF16 ? mm_launch<BN, false, QCC_OUT_BF16>(mw, mx, g, st)
           : out == QCC_OUT_F16 ? mm_launch<BN, false, QCC_OUT_F16>(mw, mx, g, st) : mm_launch<BN, false, QCC_OUT_F32>(mw, mx, g, st);
}

// Tokens a tile and shares of K for a product: the pair with the least estimated time.  A block of K counts by its way from L2, 128 rows of the
// weights and b of the tokens at 64 bytes a clock and SM (the matrix instructions take less by this estimate, 2 clocks a token and 128 at
// least); a tile has a start and an end of about 2500 clocks, of which all but the first overlap with other tiles; adding up
// over a cluster costs about 1500.  It ranks the choices and is no forecast: wide tiles share what they read, 8192^3 is estimated at 710 000
// clocks and takes 501 000.  The widths between the powers of two are there for the last wave: 600 x 4096 x 4096 16.4 -> 12.6 us (160
// tokens), 2000 x 4096 x 7168 43.3 -> 38.9 (224); of 7 sizes tried the choice was the best width in each but for 2 %.
static void mm_choose(int64_t M, int64_t N, int kblocks, int &bn, int &splits)
{
    const int sms = sm_count();
    double best = 0;
    bn = 0;
    for (int b = 16, last = 0; b <= 256; last = b, b += b < 32 ? 16 : 32) {
        if (last >= M) break;
        const int64_t tiles = (N + MM_BM - 1) / MM_BM * ((M + b - 1) / b);
        const double block = (MM_BM + b) * 2;
        for (int s = 1; s <= 8; s *= 2) {
            if (s > 1 && ((b & (b - 1)) || kblocks < 2 * s || tiles * s > sms)) break;
            const int64_t waves = (tiles * s + sms - 1) / sms;
            const double t = waves * ((kblocks + s - 1) / s) * block + 2500 + (waves - 1) * (b * 6.0) + (s > 1 ? 1500 : 0);
            if (bn == 0 || t < best) {
                best = t;
                bn = b;
                splits = s;
            }
        }
    }
}

static int byte_map(CUtensorMap *map, const void *base, int64_t rows, int64_t cols, int box_rows)
{
    const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)cols};
    const uint32_t box[2] = {MM_BK, (uint32_t)box_rows};
    const int rc = make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    return rc == -5 ? QCC_ERR_DRIVER : rc;
}

}  // namespace qcc

using namespace qcc;

extern "C" int qcc_int8_device_error(unsigned int *out) { return read_clear_device_error(out); }

extern "C" int qcc_int8_rowwise(const void *x, int64_t M, int64_t N, int flags, void *q, float *scale, void *stream)
{
    const int recip = take_recip_div(flags);
    if (flags != 0) return QCC_ERR_ARG;
    if (M < 0 || N <= 0 || M > 0x7FFFFFFF) return QCC_ERR_SHAPE;
    if (M == 0) return 0;
    if (!x || !q || !scale) return QCC_ERR_ARG;
    if (!aligned16(x) || !aligned16(q) || !aligned16(scale)) return QCC_ERR_ALIGN;
    const uint16_t *xp = static_cast<const uint16_t *>(x);
    uint8_t *qp = static_cast<uint8_t *>(q);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
#define QCC_I8(CH) return (int)launch_maybe_pdl(int8_rowwise_kernel<CH>, dim3((unsigned)M), dim3(I8_THREADS), 0, st, true, xp, N, qp, scale, recip)
    if (N % 8 != 0 || N > 8 * 8 * I8_THREADS) QCC_I8(0);
    if (N <= 8 * I8_THREADS) QCC_I8(1);
    if (N <= 2 * 8 * I8_THREADS) QCC_I8(2);
    if (N <= 4 * 8 * I8_THREADS) QCC_I8(4);
    QCC_I8(8);
#undef QCC_I8
}

extern "C" int qcc_int8_scaled_mm(const void *a, const void *b, int64_t M, int64_t N, int64_t K, const float *scale_a, const float *scale_b,
                                  const void *bias, int out_dtype, void *out, void *stream)
{
    if (out_dtype < QCC_OUT_BF16 || out_dtype > QCC_OUT_F32) return QCC_ERR_ARG;
    if (M < 0 || N < 0 || M > 0x7FFFFF00 || N > 0x7FFFFF00 || K < 16 || K % 16 != 0 || K > QCC_INT8_MAX_K) return QCC_ERR_SHAPE;
    if (M == 0 || N == 0) return 0;
    if (!a || !b || !scale_a || !scale_b || !out) return QCC_ERR_ARG;
    if (!aligned16(a) || !aligned16(b) || !aligned16(out)) return QCC_ERR_ALIGN;
    const int kblocks = (int)((K + MM_BK - 1) / MM_BK);
    int bn, splits;
    mm_choose(M, N, kblocks, bn, splits);
    const int64_t tiles_n = (N + MM_BM - 1) / MM_BM, tiles_m = (M + bn - 1) / bn;
    if (tiles_n * tiles_m > 0x7FFFFFFF / 8) return QCC_ERR_SHAPE;
    const int64_t row = N * (out_dtype == QCC_OUT_F32 ? 4 : 2);
    const int piece = row % 16 == 0 ? 4 : row % 8 == 0 ? 3 : row % 4 == 0 ? 2 : 1;
    const MmArgs g = {scale_a, scale_b, static_cast<const uint16_t *>(bias), out, (int)M, (int)N, kblocks, (int)tiles_n, (int)tiles_m, splits, piece};
    CUtensorMap mw, mx;
    int rc = byte_map(&mw, b, N, K, MM_BM);
    if (rc == 0) rc = byte_map(&mx, a, M, K, bn);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (bn) {
    case 16: return mm_dispatch<16>(mw, mx, g, out_dtype, st);
    case 32: return mm_dispatch<32>(mw, mx, g, out_dtype, st);
    case 64: return mm_dispatch<64>(mw, mx, g, out_dtype, st);
    case 96: return mm_dispatch<96, false>(mw, mx, g, out_dtype, st);
    case 128: return mm_dispatch<128>(mw, mx, g, out_dtype, st);
    case 160: return mm_dispatch<160, false>(mw, mx, g, out_dtype, st);
    case 192: return mm_dispatch<192, false>(mw, mx, g, out_dtype, st);
    case 224: return mm_dispatch<224, false>(mw, mx, g, out_dtype, st);
    default: return mm_dispatch<256>(mw, mx, g, out_dtype, st);
    }
}
