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
// once; CH = 0: rows too long for that, or not a multiple of 8 elements, are read twice (the second time from L2).
template <int CH>
__global__ void __launch_bounds__(I8_THREADS) int8_rowwise_kernel(const uint16_t *__restrict__ x, int64_t N, uint8_t *__restrict__ q,
                                                                  float *__restrict__ scale, int recip_div)
{
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
            v[c] = k < nchunk ? ld_nc_v4(reinterpret_cast<const uint4 *>(xr) + k) : make_uint4(0, 0, 0, 0);
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
// tcgen05.mma kind::i8 on tiles of 128 output channels (the M side of the instruction: one accumulator row per thread of the
// epilogue, so a warp stores 32 neighbouring channels of a token) by BN tokens, K in blocks of 128 bytes staged by TMA.  The
// tokens are on the N side because it goes down to 16: a decode batch wastes little of the instruction.
constexpr int MM_BM = 128, MM_BK = 128, MM_THREADS = 256;
constexpr unsigned int MM_ERR = 7;   // a barrier wait of the product ran out

template <int BN> struct MmCfg {
    static constexpr int STAGE = (MM_BM + BN) * MM_BK;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int RED = BN <= 128 ? MM_BM * BN * 4 : 0;             // partial sums of one CTA (split form), in the stages' memory
    static constexpr int SMEM = (STAGE * STAGES > RED ? STAGE * STAGES : RED) + 1024 + BN * 4 * 2 + 256;
};

struct MmArgs {
    const float *sa, *sb;
    const uint16_t *bias;
    void *out;
    int M, N, kblocks, tiles_n, tiles_m, splits, out_kind;
};

__device__ __forceinline__ void mm_store(const MmArgs &g, int64_t m, int n, float y)
{
    const size_t at = (size_t)m * g.N + n;
    if (g.out_kind == 0) reinterpret_cast<__nv_bfloat16 *>(g.out)[at] = __float2bfloat16_rn(y);
    else if (g.out_kind == 1) reinterpret_cast<__half *>(g.out)[at] = __float2half_rn(y);
    else reinterpret_cast<float *>(g.out)[at] = y;
}

// groups of 8 token tiles share the weights that pass through L2
__device__ __forceinline__ void mm_tile(const MmArgs &g, int t, int &tn, int &tm)
{
    const int per = 8 * g.tiles_n, grp = t / per, first = grp * 8, rows = min(8, g.tiles_m - first), r = t - grp * per;
    tm = first + r % rows;
    tn = r / rows;
}

template <int BN, bool SPLIT>
__global__ void __launch_bounds__(MM_THREADS, 1) int8_mm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                                                                const MmArgs g)
{
    using C = MmCfg<BN>;
    extern __shared__ uint8_t raw[];
    uint8_t *stages = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    constexpr int BODY = C::STAGE * C::STAGES > C::RED ? C::STAGE * C::STAGES : C::RED;
    float *s_sa = reinterpret_cast<float *>(stages + BODY);                 // 2 x BN token scales
    uint64_t *full = reinterpret_cast<uint64_t *>(s_sa + 2 * BN), *empty = full + C::STAGES, *acc_full = empty + C::STAGES,
             *acc_empty = acc_full + 2;
    uint32_t *slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    volatile uint32_t *abort = slot + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr uint32_t ACC_COLS = BN < 32 ? 32 : BN, TMEM_COLS = SPLIT ? ACC_COLS : 2 * ACC_COLS;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::STAGES; i++) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < 2; i++) { mbar_init(acc_full + i, 1); mbar_init(acc_empty + i, 4); }
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 2) tmem_alloc(slot, TMEM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *slot;
    const int total = g.tiles_n * g.tiles_m;
    // SPLIT: the CTAs of a cluster take one tile together, each a share of the K blocks
    const int rank = SPLIT ? blockIdx.x % g.splits : 0;
    const int kb0 = SPLIT ? (int)((int64_t)g.kblocks * rank / g.splits) : 0, kb1 = SPLIT ? (int)((int64_t)g.kblocks * (rank + 1) / g.splits) : g.kblocks;
    const int t0 = SPLIT ? blockIdx.x / g.splits : blockIdx.x, step = SPLIT ? total : gridDim.x;

    if (warp == 0) {
        if (elect_one()) {
            uint32_t it = 0;
            for (int t = t0; t < total; t += step) {
                int tn, tm;
                mm_tile(g, t, tn, tm);
                for (int kb = kb0; kb < kb1; kb++, it++) {
                    const uint32_t s = it % C::STAGES, ph = (it / C::STAGES) & 1;
                    mbar_wait_abort(empty + s, ph ^ 1, MM_ERR, abort);
                    uint8_t *p = stages + s * C::STAGE;
                    mbar_expect_tx(full + s, C::STAGE);
                    tma_load_2d(p, &map_w, full + s, kb * MM_BK, tn * MM_BM);
                    tma_load_2d(p + MM_BM * MM_BK, &map_x, full + s, kb * MM_BK, tm * BN);
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(MM_BM >> 4) << 24);
            uint32_t it = 0, n = 0;
            for (int t = t0; t < total; t += step, n++) {
                const uint32_t acc = SPLIT ? 0 : n & 1, aph = SPLIT ? 0 : (n >> 1) & 1;
                mbar_wait_abort(acc_empty + acc, aph ^ 1, MM_ERR, abort);
                tc_fence_after();
                for (int kb = kb0; kb < kb1; kb++, it++) {
                    const uint32_t s = it % C::STAGES, ph = (it / C::STAGES) & 1;
                    mbar_wait_abort(full + s, ph, MM_ERR, abort);
                    tc_fence_after();
                    const uint32_t a = smem_u32(stages + s * C::STAGE);
                    const uint64_t da = desc_kmajor_sw128(a), db = desc_kmajor_sw128(a + MM_BM * MM_BK);
#pragma unroll
                    for (int k = 0; k < MM_BK / 32; k++)
                        asm volatile(
                            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem + acc * ACC_COLS),
                            "l"(da + 2 * k), "l"(db + 2 * k), "r"(idesc), "r"((kb > kb0 || k > 0) ? 1u : 0u)
                            : "memory");
                    tc_commit(empty + s);
                }
                tc_commit(acc_full + acc);
            }
        }
    } else if (warp >= 4) {
        const int w = warp - 4, et = threadIdx.x - 128;
        uint32_t n = 0;
        for (int t = t0; t < total; t += step, n++) {
            int tn, tm;
            mm_tile(g, t, tn, tm);
            const uint32_t acc = SPLIT ? 0 : n & 1, aph = SPLIT ? 0 : (n >> 1) & 1;
            const int ch = tn * MM_BM + w * 32 + lane;
            float *sa = s_sa + acc * BN;
            for (int i = et; i < BN; i += 128) sa[i] = tm * BN + i < g.M ? g.sa[(int64_t)tm * BN + i] : 0.0f;
            named_barrier(1, 128);
            const float sb = ch < g.N ? g.sb[ch] : 0.0f;
            const float bias = g.bias != nullptr && ch < g.N ? u2f((uint32_t)g.bias[ch] << 16) : 0.0f;
            mbar_wait_abort(acc_full + acc, aph, MM_ERR, abort);
            tc_fence_after();
            if (SPLIT) {
                int32_t *red = reinterpret_cast<int32_t *>(stages);
#pragma unroll 1
                for (int c = 0; c < BN; c += 16) {
                    uint32_t r[16];
                    tmem_ld16(tmem + ((uint32_t)w << 21) + c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; j++) red[(c + j) * MM_BM + w * 32 + lane] = (int32_t)r[j];
                }
            } else {
#pragma unroll 1
                for (int c = 0; c < BN; c += 16) {
                    uint32_t r[16];
                    tmem_ld16(tmem + ((uint32_t)w << 21) + acc * ACC_COLS + c, r);
                    tmem_wait_ld();
                    if (c + 16 >= BN) {                 // the accumulator is in registers: the next tile may have it
                        tc_fence_before();
                        if (lane == 0) mbar_arrive(acc_empty + acc);
                    }
                    if (ch < g.N) {
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int64_t m = (int64_t)tm * BN + c + j;
                            if (m < g.M) {
                                float y = __fmul_rn(__fmul_rn((float)(int32_t)r[j], sa[c + j]), sb);
                                if (g.bias != nullptr) y = __fadd_rn(y, bias);
                                mm_store(g, m, ch, y);
                            }
                        }
                    }
                }
            }
        }
    }
    __syncwarp();
    if (SPLIT) {
        // every CTA of the cluster adds up its share of the tokens from all shares of K; whole numbers, so in any order the same
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        int tn, tm;
        mm_tile(g, t0, tn, tm);
        const uint32_t red = smem_u32(stages);
        const int rows = min(BN, g.M - tm * BN);
        const int lo = rows * rank / g.splits, hi = rows * (rank + 1) / g.splits;
        const int ch = threadIdx.x & 127, n = tn * MM_BM + ch;
        const float sb = n < g.N ? g.sb[n] : 0.0f;
        const float bias = g.bias != nullptr && n < g.N ? u2f((uint32_t)g.bias[n] << 16) : 0.0f;
        for (int i = lo + (threadIdx.x >> 7); i < hi; i += MM_THREADS / 128) {
            int32_t sum = 0;
            for (int p = 0; p < g.splits; p++) {
                uint32_t addr;
                int32_t v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(red + (uint32_t)(i * MM_BM + ch) * 4u), "r"(p));
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr));
                sum += v;
            }
            if (n < g.N) {
                float y = __fmul_rn(__fmul_rn((float)sum, s_sa[i]), sb);
                if (g.bias != nullptr) y = __fadd_rn(y, bias);
                mm_store(g, (int64_t)tm * BN + i, n, y);
            }
        }
        // no CTA leaves while another may still read its sums
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_free(tmem, TMEM_COLS);
    }
}

template <int BN, bool SPLIT>
static int mm_launch(const CUtensorMap &mw, const CUtensorMap &mx, const MmArgs &g, cudaStream_t st)
{
    using C = MmCfg<BN>;
    static PerDeviceFlag done;
    const int dev = current_device_slot();
    if (dev < 0) return QCC_ERR_ARG;
    if (!done.get(dev)) {
        cudaError_t e = cudaFuncSetAttribute(int8_mm_kernel<BN, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        done.set(dev);
    }
    const int total = g.tiles_n * g.tiles_m;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = SPLIT ? total * g.splits : (total < sm_count() ? total : sm_count());
    cfg.blockDim = MM_THREADS;
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = SPLIT ? g.splits : 1;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = SPLIT ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, int8_mm_kernel<BN, SPLIT>, mw, mx, g);
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
#define QCC_I8(CH) int8_rowwise_kernel<CH><<<(unsigned)M, I8_THREADS, 0, st>>>(xp, N, qp, scale, recip)
    if (N % 8 != 0 || N > 8 * 8 * I8_THREADS) QCC_I8(0);
    else if (N <= 8 * I8_THREADS) QCC_I8(1);
    else if (N <= 2 * 8 * I8_THREADS) QCC_I8(2);
    else if (N <= 4 * 8 * I8_THREADS) QCC_I8(4);
    else QCC_I8(8);
#undef QCC_I8
    return (int)cudaGetLastError();
}

extern "C" int qcc_int8_scaled_mm(const void *a, const void *b, int64_t M, int64_t N, int64_t K, const float *scale_a, const float *scale_b,
                                  const void *bias, int out_dtype, void *out, void *stream)
{
    if (out_dtype < QCC_OUT_BF16 || out_dtype > QCC_OUT_F32) return QCC_ERR_ARG;
    if (M < 0 || N < 0 || M > 0x7FFFFF00 || N > 0x7FFFFF00 || K < 16 || K % 16 != 0 || K > QCC_INT8_MAX_K) return QCC_ERR_SHAPE;
    if (M == 0 || N == 0) return 0;
    if (!a || !b || !scale_a || !scale_b || !out) return QCC_ERR_ARG;
    if (!aligned16(a) || !aligned16(b) || !aligned16(out)) return QCC_ERR_ALIGN;
    int bn = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256;
    const int64_t tiles_n = (N + MM_BM - 1) / MM_BM;
    int64_t tiles_m = (M + bn - 1) / bn;
    if (tiles_n * tiles_m > 0x7FFFFFFF) return QCC_ERR_SHAPE;
    const int kblocks = (int)((K + MM_BK - 1) / MM_BK), sms = sm_count();
    int splits = 1;
    if (bn <= 128)   // fewer tiles than SMs: share K out over clusters of up to 8, at least 4 blocks of K each
        while (splits < 8 && tiles_n * tiles_m * splits * 2 <= sms && kblocks >= 4 * splits * 2) splits *= 2;
    MmArgs g = {scale_a, scale_b, static_cast<const uint16_t *>(bias), out, (int)M, (int)N, kblocks, (int)tiles_n, (int)tiles_m, splits, out_dtype};
    CUtensorMap mw, mx;
    int rc = byte_map(&mw, b, N, K, MM_BM);
    if (rc == 0) rc = byte_map(&mx, a, M, K, bn);
    if (rc) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (bn) {
    case 16: return splits > 1 ? mm_launch<16, true>(mw, mx, g, st) : mm_launch<16, false>(mw, mx, g, st);
    case 32: return splits > 1 ? mm_launch<32, true>(mw, mx, g, st) : mm_launch<32, false>(mw, mx, g, st);
    case 64: return splits > 1 ? mm_launch<64, true>(mw, mx, g, st) : mm_launch<64, false>(mw, mx, g, st);
    case 128: return splits > 1 ? mm_launch<128, true>(mw, mx, g, st) : mm_launch<128, false>(mw, mx, g, st);
    default: return mm_launch<256, false>(mw, mx, g, st);
    }
}
