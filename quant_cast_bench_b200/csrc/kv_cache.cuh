// The paged nvfp4 key/value cache: layout and decoding shared by the append, read-back and attention kernels.
//
//   cache (pages, kv heads, 2, page * 9 * D / 16) bytes.  The block of one (page, head, keys | values) holds the e2m1 codes of
//   the page's tokens, (page, D / 2) with the even element in the low nibble, then their e4m3 scales (page, D / 16).
//
// Keys and values of a (page, head) lie side by side, page * 9 * D / 8 bytes that one bulk copy brings into shared memory;
// codes of a token are one contiguous row, so appending a token writes whole 4-byte words and no token shares a byte with
// another.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace qcc {

constexpr unsigned int QCC_DEVERR_PAGE = 20u;       // a page or slot number outside the cache, or a sequence longer than its table row
constexpr unsigned int QCC_DEVERR_POSITION = 21u;   // a position outside the rotation table

template <int D> __host__ __device__ constexpr int kv_row_codes() { return D / 2; }
template <int D> __host__ __device__ constexpr int kv_row_scales() { return D / 16; }
// bytes of one token and head, keys or values
template <int D> __host__ __device__ constexpr int kv_row_bytes() { return D / 2 + D / 16; }

// eight e2m1 nibbles -> four half2, pairs (0,1), (2,3), ...; exact
__device__ __forceinline__ void e2m1x8_to_half(uint32_t w, uint32_t (&h)[4])
{
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\ncvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}\n"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
// two e4m3 bytes -> half2, the low byte in the low half; exact
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two)
{
    uint32_t h;
    asm("{\n.reg .b16 b;\ncvt.u16.u32 b, %1;\ncvt.rn.f16x2.e4m3x2 %0, b;\n}\n" : "=r"(h) : "r"(two));
    return h;
}
// an e4m3 byte as half2 with both halves its value; exact
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t byte)
{
    return e4m3x2_to_half2(byte * 0x101u);
}
__device__ __forceinline__ uint32_t hmul2_bits(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

}  // namespace qcc
