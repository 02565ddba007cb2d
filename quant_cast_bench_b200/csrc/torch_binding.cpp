// The casts as native PyTorch operators: TORCH_LIBRARY(quant_cast_cuda_native, ...) over the C ABI.
//
// A thin layer: every operator checks its tensors, allocates the outputs with the gold shapes and dtype views, and
// calls the entry point of include/quant_cast_cuda.h on the current CUDA stream of x's device.  Meta implementations
// give the same shapes without touching a device, so the operators trace (torch.compile, torch.export) and can be
// called from C++ (torch::Dispatcher / the generated torch.ops handles) without Python.  The reference's counterpart is
// the recipe layer of its Triton backend (quant_cast_triton/recipes.py:48-65 of vkuzo/quant_cast_bench).
//
//   amax(x, kind, fmt, recip_div)                           -> fp32 scalar   kind: "raw" | "fp8" | "nvfp4"
//   fp8_tensorwise(x, scale, fmt)                           -> q
//   fp8_rowwise(x, fmt, recip_div)                          -> (q, scale (M, 1))
//   fp8_colwise(x, fmt, recip_div)                          -> (q (N, M), scale (N, 1))
//   mxfp8(x, rowwise, colwise, swizzle, mode)               -> [qk, sk][qm, sm]   mode: "rceil" | "floor"
//   nvfp4(x, outer_scale, swizzle, transposed, recip_div)   -> (q, inner scales)   outer_scale: one value, (M, 1) per
//                                                               token, or the (M/128, N/128) grid of 128x128 blocks
//   nvfp4_sr(x, outer_scale, key, swizzle, transposed, recip_div) -> (q, inner scales)   key: uint64 [seed, offset]
//   nvfp4_both(x, outer_scale, swizzle, recip_div)          -> (qk, sk, qm, sm)     both orientations from one read
//   fp8_rowwise_precalc(x, scale, fmt) / fp8_colwise_precalc(x, scale, fmt) -> q   true division by given scales
//   fp8_block128(x, rowwise, colwise, recip_div)            -> [qk, sk][qm, sm]    1x128 / 128x1 blocks, fp32 scales
//   fp8_block128x128(x, recip_div)                          -> (q, scale (M/128, N/128))
//   mxfp8_32x32(x, rowwise, colwise, swizzle, transposed_data) -> [qk, sk][qm] [sm] one e8m0 scale per 32x32 block
//   mxfp4(x, swizzle)                                       -> (q (M, N/2), scale)
//   nvfp4_per_token_scale(x, recip_div)                     -> (M, 1) fp32 outer scales
//   sr_f32_to_bf16(x, key, global_row, global_col, num_col) -> bf16       fp32 input, stochastic rounding
//   int8_rowwise(x, recip_div)                              -> (q int8, scale (M, 1))
//   int8_scaled_mm(a, b, scale_a, scale_b, bias, out_dtype) -> (a @ b.T) * scale_a * scale_b.T + bias   exact int32 sums
//   nvfp4_kv_append(k, v, cache, slots, k_outer, v_outer, positions, cos_sin, interleaved, q, recip_div) -> rotated q (empty
//                                                               without q); writes the cache
//   nvfp4_kv_gather(cache, block_table, cu_kv, total, head_dim, k_outer, v_outer) -> (k, v) bf16
//   nvfp4_kv_attention(q, cache, block_table, kv_lens, k_outer, v_outer, cu_q, max_q, scale) -> (out, lse)
//
// recip_div: QCC_RECIP_DIV (divisions by a constant as eager PyTorch computes them on a CUDA device).
// Built by quant_cast_bench_b200/build.py into lib/libquant_cast_torch.so, which links against libquant_cast_cuda.so.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/quant_cast_cuda.h"

namespace {

void check_x(const at::Tensor &x)
{
    TORCH_CHECK(x.dim() == 2, "quant_cast_cuda: x must be 2-D");
    TORCH_CHECK(x.scalar_type() == at::kBFloat16, "quant_cast_cuda: x must be bfloat16");
}
void check_x_cuda(const at::Tensor &x)
{
    check_x(x);
    TORCH_CHECK(x.is_cuda() && x.is_contiguous(), "quant_cast_cuda: x must be a contiguous CUDA tensor (there is no CPU implementation)");
}
// an auxiliary tensor (scale, key) must live on x's device: the kernels read it there
void same_device(const at::Tensor &x, const at::Tensor &aux, const char *what)
{
    TORCH_CHECK(aux.device() == x.device(), "quant_cast_cuda: ", what, " is on ", aux.device(), ", x on ", x.device());
}
void *stream_of(const at::Tensor &x) { return c10::cuda::getCurrentCUDAStream(x.get_device()).stream(); }
void ok(int rc, const char *what) { TORCH_CHECK(rc == 0, "quant_cast_cuda: ", what, " failed with code ", rc); }
int fmt_of(const std::string &fmt)
{
    TORCH_CHECK(fmt == "e4m3" || fmt == "e5m2", "quant_cast_cuda: fmt must be 'e4m3' or 'e5m2'");
    return fmt == "e5m2" ? QCC_FMT_E5M2 : QCC_FMT_E4M3;
}
at::ScalarType fp8_dtype(const std::string &fmt) { return fmt_of(fmt) == QCC_FMT_E5M2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn; }
int amax_mode(const std::string &kind)
{
    TORCH_CHECK(kind == "raw" || kind == "fp8" || kind == "nvfp4", "quant_cast_cuda: kind must be 'raw', 'fp8' or 'nvfp4'");
    return kind == "raw" ? QCC_AMAX_RAW : kind == "fp8" ? QCC_AMAX_FP8_SCALE : QCC_AMAX_NVFP4_SCALE;
}
int mx_mode(const std::string &mode)
{
    TORCH_CHECK(mode == "rceil" || mode == "floor", "quant_cast_cuda: mode must be 'rceil' or 'floor'");
    return mode == "floor" ? QCC_FLOOR : 0;
}
std::vector<int64_t> blocked_shape(int64_t rows, int64_t cols) { return {(rows + 127) / 128, (cols + 3) / 4, 32, 16}; }
std::vector<int64_t> scale_shape(int64_t rows, int64_t cols, bool swizzle)
{
    return swizzle ? blocked_shape(rows, cols) : std::vector<int64_t>{rows, cols};
}
at::Tensor bytes(at::IntArrayRef shape, const at::Tensor &like) { return at::empty(shape, like.options().dtype(at::kByte)); }

// ---------------------------------------------------------------------------------------- CUDA implementations
at::Tensor amax_cuda(const at::Tensor &x, std::string kind, std::string fmt, bool recip_div)
{
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.scalar_type() == at::kBFloat16, "quant_cast_cuda: x must be contiguous CUDA bfloat16");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty({}, x.options().dtype(at::kFloat));
    const size_t ws_bytes = qcc_amax_workspace_bytes();
    at::Tensor ws = at::empty({(int64_t)ws_bytes}, x.options().dtype(at::kByte));   // two launches: any contents will do
    ok(qcc_amax_bf16(x.data_ptr(), x.numel(), amax_mode(kind) | (recip_div ? QCC_RECIP_DIV : 0), fmt_of(fmt), out.data_ptr<float>(),
                     ws.data_ptr(), ws_bytes, stream_of(x)),
       "amax");
    return out;
}

at::Tensor fp8_tensorwise_cuda(const at::Tensor &x, const at::Tensor &scale, std::string fmt)
{
    check_x_cuda(x);
    TORCH_CHECK(scale.is_cuda() && scale.scalar_type() == at::kFloat && scale.numel() == 1, "quant_cast_cuda: scale must be one CUDA fp32 value");
    same_device(x, scale, "scale");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor q = bytes(x.sizes(), x);
    ok(qcc_fp8_tensorwise(x.data_ptr(), x.numel(), scale.data_ptr<float>(), fmt_of(fmt), q.data_ptr(), stream_of(x)), "fp8_tensorwise");
    return q.view(fp8_dtype(fmt));
}

std::tuple<at::Tensor, at::Tensor> fp8_rowwise_cuda(const at::Tensor &x, std::string fmt, bool recip_div)
{
    check_x_cuda(x);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    at::Tensor q = bytes({M, N}, x), s = at::empty({M, 1}, x.options().dtype(at::kFloat));
    ok(qcc_fp8_rowwise(x.data_ptr(), M, N, fmt_of(fmt) | (recip_div ? QCC_RECIP_DIV : 0), q.data_ptr(), s.data_ptr<float>(), stream_of(x)),
       "fp8_rowwise");
    return {q.view(fp8_dtype(fmt)), s};
}

std::tuple<at::Tensor, at::Tensor> fp8_colwise_cuda(const at::Tensor &x, std::string fmt, bool recip_div)
{
    check_x_cuda(x);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK(M % 16 == 0 && N % 8 == 0, "quant_cast_cuda: colwise fp8 needs M % 16 == 0 and N % 8 == 0");
    at::Tensor q = bytes({N, M}, x), s = at::empty({N, 1}, x.options().dtype(at::kFloat));
    const size_t ws_bytes = qcc_fp8_colwise_workspace_bytes(M, N);
    at::Tensor ws = at::empty({(int64_t)ws_bytes}, x.options().dtype(at::kByte));
    ok(qcc_fp8_colwise(x.data_ptr(), M, N, fmt_of(fmt) | (recip_div ? QCC_RECIP_DIV : 0), q.data_ptr(), s.data_ptr<float>(), ws.data_ptr(),
                       ws_bytes, stream_of(x)),
       "fp8_colwise");
    return {q.view(fp8_dtype(fmt)), s};
}

std::vector<at::Tensor> mxfp8_cuda(const at::Tensor &x, bool rowwise, bool colwise, bool swizzle, std::string mode)
{
    check_x_cuda(x);
    TORCH_CHECK(rowwise || colwise, "quant_cast_cuda: mxfp8 needs at least one direction");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK((!rowwise || N % 32 == 0) && (!colwise || (M % 32 == 0 && N % 8 == 0)), "quant_cast_cuda: mxfp8 blocks need N % 32 == 0 (rowwise) / M % 32 == 0 (colwise)");
    at::Tensor qk, sk, qm, sm;
    if (rowwise) { qk = bytes({M, N}, x); sk = bytes(scale_shape(M, N / 32, swizzle), x); }
    if (colwise) { qm = bytes({N, M}, x); sm = bytes(scale_shape(N, M / 32, swizzle), x); }
    const int flags = (rowwise ? QCC_ROWWISE : 0) | (colwise ? QCC_COLWISE : 0) | (swizzle ? QCC_SWIZZLE : 0) | mx_mode(mode);
    ok(qcc_mxfp8(x.data_ptr(), M, N, flags, rowwise ? qk.data_ptr() : nullptr, rowwise ? sk.data_ptr() : nullptr,
                 colwise ? qm.data_ptr() : nullptr, colwise ? sm.data_ptr() : nullptr, stream_of(x)),
       "mxfp8");
    std::vector<at::Tensor> outs;
    if (rowwise) { outs.push_back(qk.view(at::kFloat8_e4m3fn)); outs.push_back(sk.view(at::kFloat8_e8m0fnu)); }
    if (colwise) { outs.push_back(qm.view(at::kFloat8_e4m3fn)); outs.push_back(sm.view(at::kFloat8_e8m0fnu)); }
    return outs;
}

// which outer scale: 0 one value, 1 one per row (M, 1), 2 one per 128x128 block (M/128, N/128)
int outer_kind(const at::Tensor &x, const at::Tensor &outer)
{
    const int64_t M = x.size(0), N = x.size(1);
    if (outer.numel() == 1 && outer.dim() < 2) return 0;
    if (outer.dim() == 2 && outer.size(0) == M && outer.size(1) == 1) return 1;
    if (outer.dim() == 2 && M % 128 == 0 && N % 128 == 0 && outer.size(0) == M / 128 && outer.size(1) == N / 128) return 2;
    if (outer.numel() == 1) return 0;
    TORCH_CHECK(false, "quant_cast_cuda: outer_scale must be one value, (M, 1), or (M/128, N/128)");
    return -1;
}

std::tuple<at::Tensor, at::Tensor> nvfp4_impl(const at::Tensor &x, const at::Tensor &outer_in, const uint64_t *key, bool swizzle,
                                              bool transposed, bool recip_div)
{
    check_x_cuda(x);
    TORCH_CHECK(outer_in.is_cuda() && outer_in.scalar_type() == at::kFloat, "quant_cast_cuda: outer_scale must be a CUDA fp32 tensor");
    same_device(x, outer_in, "outer_scale");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    const at::Tensor outer = outer_in.contiguous();
    const int kind = outer_kind(x, outer);
    const int flags = (swizzle ? QCC_SWIZZLE : 0) | (recip_div ? QCC_RECIP_DIV : 0) | (key ? QCC_SR : 0);
    at::Tensor q, s;
    if (transposed) {
        TORCH_CHECK(kind == 0, "quant_cast_cuda: the transposed nvfp4 cast takes one outer scale");
        TORCH_CHECK(M % 32 == 0 && N % 8 == 0, "quant_cast_cuda: transposed nvfp4 needs M % 32 == 0 and N % 8 == 0");
        q = bytes({N, M / 2}, x);
        s = bytes(scale_shape(N, M / 16, swizzle), x);
        ok(qcc_nvfp4_transposed(x.data_ptr(), M, N, outer.data_ptr<float>(), flags, key, q.data_ptr(), s.data_ptr(), stream_of(x)),
           "nvfp4 transposed");
    } else {
        TORCH_CHECK(N % 16 == 0, "quant_cast_cuda: nvfp4 needs N % 16 == 0");
        TORCH_CHECK(kind != 2 || (swizzle && !key), "quant_cast_cuda: a blocked outer scale goes with blocked inner scales and round to nearest");
        q = bytes({M, N / 2}, x);
        s = bytes(scale_shape(M, N / 16, swizzle), x);
        ok(qcc_nvfp4(x.data_ptr(), M, N, outer.data_ptr<float>(), kind, flags, key, q.data_ptr(), s.data_ptr(), stream_of(x)), "nvfp4");
    }
    return {q.view(at::kFloat4_e2m1fn_x2), s.view(at::kFloat8_e4m3fn)};
}

std::tuple<at::Tensor, at::Tensor> nvfp4_cuda(const at::Tensor &x, const at::Tensor &outer_scale, bool swizzle, bool transposed,
                                              bool recip_div)
{
    return nvfp4_impl(x, outer_scale, nullptr, swizzle, transposed, recip_div);
}

std::tuple<at::Tensor, at::Tensor> nvfp4_sr_cuda(const at::Tensor &x, const at::Tensor &outer_scale, const at::Tensor &key, bool swizzle,
                                                 bool transposed, bool recip_div)
{
    TORCH_CHECK(key.is_cuda() && key.element_size() == 8 && key.numel() >= 2 && key.is_contiguous(),
                "quant_cast_cuda: key must be a CUDA tensor of two 64-bit words [seed, offset]");
    same_device(x, key, "key");
    return nvfp4_impl(x, outer_scale, static_cast<const uint64_t *>(key.data_ptr()), swizzle, transposed, recip_div);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> nvfp4_both_cuda(const at::Tensor &x, const at::Tensor &outer_scale, bool swizzle,
                                                                         bool recip_div)
{
    check_x_cuda(x);
    TORCH_CHECK(outer_scale.is_cuda() && outer_scale.scalar_type() == at::kFloat && outer_scale.numel() == 1,
                "quant_cast_cuda: outer_scale must be one CUDA fp32 value");
    same_device(x, outer_scale, "outer_scale");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK(M % 32 == 0 && N % 32 == 0, "quant_cast_cuda: nvfp4 in both orientations needs M % 32 == 0 and N % 32 == 0");
    at::Tensor qk = bytes({M, N / 2}, x), sk = bytes(scale_shape(M, N / 16, swizzle), x);
    at::Tensor qm = bytes({N, M / 2}, x), sm = bytes(scale_shape(N, M / 16, swizzle), x);
    ok(qcc_nvfp4_both(x.data_ptr(), M, N, outer_scale.data_ptr<float>(), (swizzle ? QCC_SWIZZLE : 0) | (recip_div ? QCC_RECIP_DIV : 0),
                      qk.data_ptr(), sk.data_ptr(), qm.data_ptr(), sm.data_ptr(), stream_of(x)),
       "nvfp4 both");
    return {qk.view(at::kFloat4_e2m1fn_x2), sk.view(at::kFloat8_e4m3fn), qm.view(at::kFloat4_e2m1fn_x2), sm.view(at::kFloat8_e4m3fn)};
}

at::Tensor fp8_rowwise_precalc_cuda(const at::Tensor &x, const at::Tensor &scale, std::string fmt)
{
    check_x_cuda(x);
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK(scale.is_cuda() && scale.scalar_type() == at::kFloat && scale.numel() == M, "quant_cast_cuda: scale must hold one CUDA fp32 value per row");
    same_device(x, scale, "scale");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor sc = scale.contiguous();
    at::Tensor q = bytes({M, N}, x);
    ok(qcc_fp8_rowwise_precalc(x.data_ptr(), M, N, sc.data_ptr<float>(), fmt_of(fmt), q.data_ptr(), stream_of(x)), "fp8_rowwise_precalc");
    return q.view(fp8_dtype(fmt));
}

at::Tensor fp8_colwise_precalc_cuda(const at::Tensor &x, const at::Tensor &scale, std::string fmt)
{
    check_x_cuda(x);
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK(scale.is_cuda() && scale.scalar_type() == at::kFloat && scale.numel() == N, "quant_cast_cuda: scale must hold one CUDA fp32 value per column");
    same_device(x, scale, "scale");
    TORCH_CHECK(M % 16 == 0 && N % 8 == 0, "quant_cast_cuda: colwise fp8 needs M % 16 == 0 and N % 8 == 0");
    const c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor sc = scale.contiguous();
    at::Tensor q = bytes({N, M}, x);
    ok(qcc_fp8_colwise_precalc(x.data_ptr(), M, N, sc.data_ptr<float>(), fmt_of(fmt), q.data_ptr(), stream_of(x)), "fp8_colwise_precalc");
    return q.view(fp8_dtype(fmt));
}

std::vector<at::Tensor> fp8_block128_cuda(const at::Tensor &x, bool rowwise, bool colwise, bool recip_div)
{
    check_x_cuda(x);
    TORCH_CHECK(rowwise || colwise, "quant_cast_cuda: fp8_block128 needs at least one direction");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK((!rowwise || N % 128 == 0) && (!colwise || (M % 128 == 0 && N % 8 == 0)),
                "quant_cast_cuda: 1x128 blocks need N % 128 == 0, 128x1 blocks M % 128 == 0 and N % 8 == 0");
    at::Tensor qk, sk, qm, sm;
    if (rowwise) { qk = bytes({M, N}, x); sk = at::empty({M, N / 128}, x.options().dtype(at::kFloat)); }
    if (colwise) { qm = bytes({N, M}, x); sm = at::empty({N, M / 128}, x.options().dtype(at::kFloat)); }
    const int flags = (rowwise ? QCC_ROWWISE : 0) | (colwise ? QCC_COLWISE : 0) | (recip_div ? QCC_RECIP_DIV : 0);
    ok(qcc_fp8_block128(x.data_ptr(), M, N, flags, rowwise ? qk.data_ptr() : nullptr, rowwise ? sk.data_ptr<float>() : nullptr,
                        colwise ? qm.data_ptr() : nullptr, colwise ? sm.data_ptr<float>() : nullptr, stream_of(x)),
       "fp8_block128");
    std::vector<at::Tensor> outs;
    if (rowwise) { outs.push_back(qk.view(at::kFloat8_e4m3fn)); outs.push_back(sk); }
    if (colwise) { outs.push_back(qm.view(at::kFloat8_e4m3fn)); outs.push_back(sm); }
    return outs;
}

std::tuple<at::Tensor, at::Tensor> fp8_block128x128_cuda(const at::Tensor &x, bool recip_div)
{
    check_x_cuda(x);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK(M % 128 == 0 && N % 128 == 0, "quant_cast_cuda: 128x128 blocks need M % 128 == 0 and N % 128 == 0");
    at::Tensor q = bytes({M, N}, x), s = at::empty({M / 128, N / 128}, x.options().dtype(at::kFloat));
    ok(qcc_fp8_block128x128(x.data_ptr(), M, N, recip_div ? QCC_RECIP_DIV : 0, q.data_ptr(), s.data_ptr<float>(), stream_of(x)), "fp8_block128x128");
    return {q.view(at::kFloat8_e4m3fn), s};
}

std::vector<at::Tensor> mxfp8_32x32_cuda(const at::Tensor &x, bool rowwise, bool colwise, bool swizzle, bool transposed_data)
{
    check_x_cuda(x);
    TORCH_CHECK(rowwise || colwise, "quant_cast_cuda: mxfp8_32x32 needs at least one direction");
    TORCH_CHECK(!colwise || swizzle, "quant_cast_cuda: the transposed 32x32 outputs come with blocked scales only");
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK(M % 32 == 0 && N % 32 == 0, "quant_cast_cuda: 32x32 blocks need M % 32 == 0 and N % 32 == 0");
    at::Tensor qk, sk, qm, sm;
    if (rowwise) { qk = bytes({M, N}, x); sk = swizzle ? bytes(blocked_shape(M, N / 32), x) : bytes({M / 32, N / 32}, x); }
    if (colwise) { if (transposed_data) qm = bytes({N, M}, x); sm = bytes(blocked_shape(N, M / 32), x); }
    const int flags = QCC_BLOCK32 | (rowwise ? QCC_ROWWISE : 0) | (colwise ? QCC_COLWISE : 0) | (swizzle ? QCC_SWIZZLE : 0);
    ok(qcc_mxfp8(x.data_ptr(), M, N, flags, rowwise ? qk.data_ptr() : nullptr, rowwise ? sk.data_ptr() : nullptr,
                 qm.defined() ? qm.data_ptr() : nullptr, colwise ? sm.data_ptr() : nullptr, stream_of(x)),
       "mxfp8 32x32");
    std::vector<at::Tensor> outs;
    if (rowwise) { outs.push_back(qk.view(at::kFloat8_e4m3fn)); outs.push_back(sk.view(at::kFloat8_e8m0fnu)); }
    if (colwise) { if (transposed_data) outs.push_back(qm.view(at::kFloat8_e4m3fn)); outs.push_back(sm.view(at::kFloat8_e8m0fnu)); }
    return outs;
}

std::tuple<at::Tensor, at::Tensor> mxfp4_cuda(const at::Tensor &x, bool swizzle)
{
    check_x_cuda(x);
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t M = x.size(0), N = x.size(1);
    TORCH_CHECK(N % 32 == 0, "quant_cast_cuda: mxfp4 needs N % 32 == 0");
    at::Tensor q = bytes({M, N / 2}, x), s = bytes(scale_shape(M, N / 32, swizzle), x);
    ok(qcc_mxfp4(x.data_ptr(), M, N, swizzle ? QCC_SWIZZLE : 0, q.data_ptr(), s.data_ptr(), stream_of(x)), "mxfp4");
    return {q.view(at::kFloat4_e2m1fn_x2), s.view(at::kFloat8_e8m0fnu)};
}

at::Tensor nvfp4_per_token_scale_cuda(const at::Tensor &x, bool recip_div)
{
    check_x_cuda(x);
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor s = at::empty({x.size(0), 1}, x.options().dtype(at::kFloat));
    ok(qcc_nvfp4_per_token_scale(x.data_ptr(), x.size(0), x.size(1), recip_div ? QCC_RECIP_DIV : 0, s.data_ptr<float>(), stream_of(x)),
       "nvfp4_per_token_scale");
    return s;
}

at::Tensor sr_f32_to_bf16_cuda(const at::Tensor &x, const at::Tensor &key, int64_t global_row, int64_t global_col, int64_t num_col)
{
    TORCH_CHECK(x.is_cuda() && x.is_contiguous() && x.dim() == 2 && x.scalar_type() == at::kFloat,
                "quant_cast_cuda: sr_f32_to_bf16 takes a contiguous 2-D CUDA fp32 tensor");
    TORCH_CHECK(key.is_cuda() && key.element_size() == 8 && key.numel() >= 2 && key.is_contiguous(),
                "quant_cast_cuda: key must be a CUDA tensor of two 64-bit words [seed, offset]");
    same_device(x, key, "key");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor out = at::empty(x.sizes(), x.options().dtype(at::kBFloat16));
    ok(qcc_sr_f32_to_bf16(x.data_ptr(), x.size(0), x.size(1), static_cast<const uint64_t *>(key.data_ptr()), global_row, global_col,
                          num_col < 0 ? x.size(1) : num_col, out.data_ptr(), stream_of(x)),
       "sr_f32_to_bf16");
    return out;
}

// ---- int8 linear layer
void check_codes(const at::Tensor &t, const char *what)
{
    TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kChar, "quant_cast_cuda: ", what, " must be 2-D int8");
}
void check_product(const at::Tensor &a, const at::Tensor &b)
{
    check_codes(a, "a");
    check_codes(b, "b");
    const int64_t K = a.size(1);
    TORCH_CHECK(b.size(1) == K, "quant_cast_cuda: a has ", K, " columns, b ", b.size(1));
    TORCH_CHECK(K % 16 == 0 && K >= 16 && K <= QCC_INT8_MAX_K, "quant_cast_cuda: int8_scaled_mm needs K % 16 == 0 and 16 <= K <= ", QCC_INT8_MAX_K, ", got ", K);
}
int out_kind(at::ScalarType t)
{
    TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, "quant_cast_cuda: out_dtype must be bfloat16, float16 or float32");
    return t == at::kBFloat16 ? QCC_OUT_BF16 : t == at::kHalf ? QCC_OUT_F16 : QCC_OUT_F32;
}

std::tuple<at::Tensor, at::Tensor> int8_rowwise_cuda(const at::Tensor &x, bool recip_div)
{
    check_x_cuda(x);
    TORCH_CHECK(x.size(1) >= 1, "quant_cast_cuda: int8_rowwise needs at least one column");
    const c10::cuda::CUDAGuard guard(x.device());
    at::Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar)), s = at::empty({x.size(0), 1}, x.options().dtype(at::kFloat));
    ok(qcc_int8_rowwise(x.data_ptr(), x.size(0), x.size(1), recip_div ? QCC_RECIP_DIV : 0, q.data_ptr(), s.data_ptr<float>(), stream_of(x)), "int8_rowwise");
    return {q, s};
}

at::Tensor int8_scaled_mm_cuda(const at::Tensor &a, const at::Tensor &b, const at::Tensor &scale_a, const at::Tensor &scale_b,
                               const std::optional<at::Tensor> &bias, at::ScalarType out_dtype)
{
    check_product(a, b);
    TORCH_CHECK(a.is_cuda() && a.is_contiguous() && b.is_contiguous(), "quant_cast_cuda: a and b must be contiguous CUDA tensors (there is no CPU implementation)");
    const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
    TORCH_CHECK(scale_a.scalar_type() == at::kFloat && scale_a.numel() == M && scale_a.is_contiguous() && scale_b.scalar_type() == at::kFloat &&
                    scale_b.numel() == N && scale_b.is_contiguous(),
                "quant_cast_cuda: scale_a and scale_b must be contiguous fp32, one value a row of a and of b");
    same_device(a, b, "b");
    same_device(a, scale_a, "scale_a");
    same_device(a, scale_b, "scale_b");
    if (bias) {
        TORCH_CHECK(bias->scalar_type() == at::kBFloat16 && bias->numel() == N && bias->is_contiguous(), "quant_cast_cuda: bias must be N contiguous bfloat16 values");
        same_device(a, *bias, "bias");
    }
    const int kind = out_kind(out_dtype);
    const c10::cuda::CUDAGuard guard(a.device());
    at::Tensor out = at::empty({M, N}, a.options().dtype(out_dtype));
    ok(qcc_int8_scaled_mm(a.data_ptr(), b.data_ptr(), M, N, K, scale_a.data_ptr<float>(), scale_b.data_ptr<float>(), bias ? bias->data_ptr() : nullptr, kind,
                          out.data_ptr(), stream_of(a)),
       "int8_scaled_mm");
    return out;
}

// ---- paged nvfp4 key/value cache
struct CacheShape {
    int heads, page;
};
CacheShape check_cache(const at::Tensor &cache, int64_t head_dim)
{
    TORCH_CHECK(head_dim == 64 || head_dim == 128, "quant_cast_cuda: head_dim must be 64 or 128");
    TORCH_CHECK(cache.is_cuda() && cache.scalar_type() == at::kByte && cache.dim() == 4 && cache.size(2) == 2 && cache.is_contiguous(),
                "quant_cast_cuda: cache must be a contiguous CUDA uint8 tensor (pages, kv_heads, 2, page * 9 * head_dim / 16)");
    const int64_t unit = 9 * head_dim / 16, page = cache.size(3) / unit;
    TORCH_CHECK(cache.size(3) % unit == 0 && (page == 16 || page == 32 || page == 64 || page == 128) && cache.size(1) >= 1 && cache.size(1) <= 4096,
                "quant_cast_cuda: a page block of ", cache.size(3), " bytes is no page of 16, 32, 64 or 128 tokens");
    return {(int)cache.size(1), (int)page};
}
void check_rows(const at::Tensor &t, const at::Tensor &cache, const char *what)
{
    TORCH_CHECK(t.dim() == 3 && t.scalar_type() == at::kBFloat16, "quant_cast_cuda: ", what, " must be 3-D bfloat16");
    same_device(cache, t, what);
    TORCH_CHECK(t.stride(2) == 1 && (t.numel() == 0 || (t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)),
                "quant_cast_cuda: rows of ", what, " must be contiguous and 16-byte aligned");
}
const float *outer_of(const at::Tensor &t, const at::Tensor &cache, const char *what)
{
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == 1, "quant_cast_cuda: ", what, " must be one fp32 value");
    same_device(cache, t, what);
    return t.data_ptr<float>();
}
void check_numbers(const at::Tensor &t, at::ScalarType dt, int64_t n, const at::Tensor &cache, const char *what)
{
    TORCH_CHECK(t.scalar_type() == dt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), "quant_cast_cuda: ", what, " must be ", n, " contiguous ", dt, " values");
    same_device(cache, t, what);
}
void check_table(const at::Tensor &t, const at::Tensor &cache)
{
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && t.stride(0) >= 0 && t.size(1) <= 0x7FFFFFFF && t.size(0) <= 0x7FFFFFFE,
                "quant_cast_cuda: block_table must be int32 (seqs, pages) with contiguous rows");
    same_device(cache, t, "block_table");
}

at::Tensor nvfp4_kv_append_cuda(const at::Tensor &k, const at::Tensor &v, at::Tensor cache, const at::Tensor &slots, const at::Tensor &k_outer,
                                const at::Tensor &v_outer, const std::optional<at::Tensor> &positions, const std::optional<at::Tensor> &cos_sin,
                                bool interleaved, const std::optional<at::Tensor> &q, bool recip_div)
{
    TORCH_CHECK(k.dim() == 3, "quant_cast_cuda: k must be (tokens, kv_heads, head_dim)");
    const int64_t T = k.size(0), D = k.size(2);
    const CacheShape c = check_cache(cache, D);
    check_rows(k, cache, "k");
    check_rows(v, cache, "v");
    TORCH_CHECK(v.sizes() == k.sizes() && k.size(1) == c.heads, "quant_cast_cuda: k and v must have the cache's heads and one shape");
    check_numbers(slots, at::kLong, T, cache, "slots");
    qcc_kv_append_args a = {};
    a.k_outer = outer_of(k_outer, cache, "k_outer");
    a.v_outer = outer_of(v_outer, cache, "v_outer");
    if (cos_sin) {
        TORCH_CHECK(cos_sin->scalar_type() == at::kFloat && cos_sin->dim() == 2 && cos_sin->is_contiguous() && cos_sin->size(0) > 0 && cos_sin->size(1) > 0 &&
                        cos_sin->size(1) <= D && cos_sin->size(1) % 32 == 0,
                    "quant_cast_cuda: cos_sin must be contiguous fp32 (max_pos, rot) with rot a multiple of 32 up to ", D);
        same_device(cache, *cos_sin, "cos_sin");
        TORCH_CHECK(positions.has_value(), "quant_cast_cuda: a rotation needs positions");
        check_numbers(*positions, at::kLong, T, cache, "positions");
        a.cos_sin = cos_sin->data_ptr<float>();
        a.positions = positions->data_ptr<int64_t>();
        a.max_pos = cos_sin->size(0);
        a.rot = (int)cos_sin->size(1);
    }
    const c10::cuda::CUDAGuard guard(cache.device());
    at::Tensor out = at::empty({q ? T : 0, q ? q->size(1) : 0, D}, k.options());
    if (q) {
        check_rows(*q, cache, "q");
        TORCH_CHECK(q->size(0) == T && q->size(2) == D && q->size(1) <= 4096, "quant_cast_cuda: q must have k's tokens and head_dim");
        a.q = q->data_ptr();
        a.q_out = out.data_ptr();
        a.q_heads = (int)q->size(1);
        a.q_stride[0] = q->stride(0);
        a.q_stride[1] = q->stride(1);
    }
    if (T == 0) return out;
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.k_stride[0] = k.stride(0); a.k_stride[1] = k.stride(1);
    a.v_stride[0] = v.stride(0); a.v_stride[1] = v.stride(1);
    a.tokens = T;
    a.cache = cache.data_ptr();
    a.num_pages = cache.size(0);
    a.slots = slots.data_ptr<int64_t>();
    a.kv_heads = c.heads;
    a.head_dim = (int)D;
    a.page = c.page;
    a.flags = (interleaved ? QCC_ROPE_INTERLEAVED : 0) | (recip_div ? QCC_RECIP_DIV : 0);
    ok(qcc_nvfp4_kv_append(&a, stream_of(cache)), "nvfp4_kv_append");
    return out;
}

std::tuple<at::Tensor, at::Tensor> nvfp4_kv_gather_cuda(const at::Tensor &cache, const at::Tensor &block_table, const at::Tensor &cu_kv, int64_t total,
                                                        int64_t head_dim, const at::Tensor &k_outer, const at::Tensor &v_outer)
{
    const CacheShape c = check_cache(cache, head_dim);
    check_table(block_table, cache);
    check_numbers(cu_kv, at::kInt, block_table.size(0) + 1, cache, "cu_kv");
    const float *ko = outer_of(k_outer, cache, "k_outer"), *vo = outer_of(v_outer, cache, "v_outer");
    TORCH_CHECK(total >= 0, "quant_cast_cuda: total must not be negative");
    const c10::cuda::CUDAGuard guard(cache.device());
    at::Tensor k = at::empty({total, c.heads, head_dim}, cache.options().dtype(at::kBFloat16)), v = at::empty_like(k);
    ok(qcc_nvfp4_kv_gather(cache.data_ptr(), cache.size(0), c.heads, c.page, (int)head_dim, block_table.data_ptr<int32_t>(), block_table.stride(0),
                           (int)block_table.size(1), cu_kv.data_ptr<int32_t>(), (int)block_table.size(0), total, ko, vo, k.data_ptr(), v.data_ptr(), stream_of(cache)),
       "nvfp4_kv_gather");
    return {k, v};
}

void check_scale(const std::optional<double> &scale) { TORCH_CHECK(!scale || *scale > 0, "quant_cast_cuda: scale must be positive, got ", *scale); }

std::tuple<at::Tensor, at::Tensor> nvfp4_kv_attention_cuda(const at::Tensor &q, const at::Tensor &cache, const at::Tensor &block_table, const at::Tensor &kv_lens,
                                                           const at::Tensor &k_outer, const at::Tensor &v_outer, const std::optional<at::Tensor> &cu_q,
                                                           int64_t max_q, std::optional<double> scale)
{
    check_scale(scale);
    TORCH_CHECK(q.dim() == 3, "quant_cast_cuda: q must be (rows, q_heads, head_dim)");
    const int64_t rows = q.size(0), hq = q.size(1), D = q.size(2), seqs = block_table.size(0);
    const CacheShape c = check_cache(cache, D);
    check_rows(q, cache, "q");
    TORCH_CHECK(hq >= c.heads && hq % c.heads == 0 && hq <= 4096, "quant_cast_cuda: ", hq, " query heads do not divide among ", c.heads, " kv heads");
    check_table(block_table, cache);
    check_numbers(kv_lens, at::kInt, seqs, cache, "kv_lens");
    qcc_kv_attention_args a = {};
    a.k_outer = outer_of(k_outer, cache, "k_outer");
    a.v_outer = outer_of(v_outer, cache, "v_outer");
    if (cu_q) {
        check_numbers(*cu_q, at::kInt, seqs + 1, cache, "cu_q");
        TORCH_CHECK(max_q >= 1, "quant_cast_cuda: cu_q needs max_q >= 1");
        max_q = std::min<int64_t>(max_q, 0x7FFFFFFF);
    } else {
        TORCH_CHECK(rows == seqs, "quant_cast_cuda: ", rows, " query rows for ", seqs, " sequences: several queries a sequence need cu_q");
        max_q = 1;
    }
    const c10::cuda::CUDAGuard guard(cache.device());
    at::Tensor out = at::empty({rows, hq, D}, q.options()), lse = at::empty({rows, hq}, q.options().dtype(at::kFloat));
    if (rows == 0 || seqs == 0) {
        out.zero_();
        lse.fill_(-std::numeric_limits<float>::infinity());
        return {out, lse};
    }
    const size_t ws_bytes = qcc_nvfp4_kv_attention_workspace_bytes(rows, (int)std::min<int64_t>(seqs, 1 << 20), (int)max_q, (int)hq, c.heads, (int)D);
    at::Tensor ws = at::empty({(int64_t)ws_bytes}, cache.options());
    a.q = q.data_ptr();
    a.q_stride[0] = q.stride(0); a.q_stride[1] = q.stride(1);
    a.rows = rows;
    a.cache = cache.data_ptr();
    a.num_pages = cache.size(0);
    a.table = block_table.data_ptr<int32_t>();
    a.table_stride = block_table.stride(0);
    a.table_width = (int)block_table.size(1);
    a.kv_lens = kv_lens.data_ptr<int32_t>();
    a.cu_q = cu_q ? cu_q->data_ptr<int32_t>() : nullptr;
    a.seqs = (int)std::min<int64_t>(seqs, 1 << 20);
    a.max_q = (int)max_q;
    a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)D));
    a.q_heads = (int)hq;
    a.kv_heads = c.heads;
    a.head_dim = (int)D;
    a.page = c.page;
    a.out = out.data_ptr();
    a.lse = lse.data_ptr<float>();
    ok(qcc_nvfp4_kv_attention(&a, ws.data_ptr(), ws_bytes, stream_of(cache)), "nvfp4_kv_attention");
    return {out, lse};
}

// ---------------------------------------------------------------------------------------- Meta (shape) implementations
at::Tensor like(const at::Tensor &x, std::vector<int64_t> shape, at::ScalarType dt) { return at::empty(shape, x.options().dtype(dt)); }

at::Tensor amax_meta(const at::Tensor &x, std::string kind, std::string fmt, bool)
{
    amax_mode(kind);
    fmt_of(fmt);
    return like(x, {}, at::kFloat);
}
at::Tensor fp8_tensorwise_meta(const at::Tensor &x, const at::Tensor &, std::string fmt) { return like(x, x.sizes().vec(), fp8_dtype(fmt)); }
std::tuple<at::Tensor, at::Tensor> fp8_rowwise_meta(const at::Tensor &x, std::string fmt, bool)
{
    check_x(x);
    return {like(x, {x.size(0), x.size(1)}, fp8_dtype(fmt)), like(x, {x.size(0), 1}, at::kFloat)};
}
std::tuple<at::Tensor, at::Tensor> fp8_colwise_meta(const at::Tensor &x, std::string fmt, bool)
{
    check_x(x);
    return {like(x, {x.size(1), x.size(0)}, fp8_dtype(fmt)), like(x, {x.size(1), 1}, at::kFloat)};
}
std::vector<at::Tensor> mxfp8_meta(const at::Tensor &x, bool rowwise, bool colwise, bool swizzle, std::string mode)
{
    check_x(x);
    mx_mode(mode);
    const int64_t M = x.size(0), N = x.size(1);
    std::vector<at::Tensor> outs;
    if (rowwise) { outs.push_back(like(x, {M, N}, at::kFloat8_e4m3fn)); outs.push_back(like(x, scale_shape(M, N / 32, swizzle), at::kFloat8_e8m0fnu)); }
    if (colwise) { outs.push_back(like(x, {N, M}, at::kFloat8_e4m3fn)); outs.push_back(like(x, scale_shape(N, M / 32, swizzle), at::kFloat8_e8m0fnu)); }
    return outs;
}
std::tuple<at::Tensor, at::Tensor> nvfp4_meta(const at::Tensor &x, const at::Tensor &, bool swizzle, bool transposed, bool)
{
    check_x(x);
    const int64_t rows = transposed ? x.size(1) : x.size(0), cols = transposed ? x.size(0) : x.size(1);
    return {like(x, {rows, cols / 2}, at::kFloat4_e2m1fn_x2), like(x, scale_shape(rows, cols / 16, swizzle), at::kFloat8_e4m3fn)};
}

std::tuple<at::Tensor, at::Tensor> nvfp4_sr_meta(const at::Tensor &x, const at::Tensor &o, const at::Tensor &, bool swizzle, bool transposed,
                                                 bool r)
{
    return nvfp4_meta(x, o, swizzle, transposed, r);
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> nvfp4_both_meta(const at::Tensor &x, const at::Tensor &, bool swizzle, bool)
{
    check_x(x);
    const int64_t M = x.size(0), N = x.size(1);
    return {like(x, {M, N / 2}, at::kFloat4_e2m1fn_x2), like(x, scale_shape(M, N / 16, swizzle), at::kFloat8_e4m3fn),
            like(x, {N, M / 2}, at::kFloat4_e2m1fn_x2), like(x, scale_shape(N, M / 16, swizzle), at::kFloat8_e4m3fn)};
}
at::Tensor fp8_rowwise_precalc_meta(const at::Tensor &x, const at::Tensor &, std::string fmt)
{
    check_x(x);
    return like(x, {x.size(0), x.size(1)}, fp8_dtype(fmt));
}
at::Tensor fp8_colwise_precalc_meta(const at::Tensor &x, const at::Tensor &, std::string fmt)
{
    check_x(x);
    return like(x, {x.size(1), x.size(0)}, fp8_dtype(fmt));
}
std::vector<at::Tensor> fp8_block128_meta(const at::Tensor &x, bool rowwise, bool colwise, bool)
{
    check_x(x);
    const int64_t M = x.size(0), N = x.size(1);
    std::vector<at::Tensor> outs;
    if (rowwise) { outs.push_back(like(x, {M, N}, at::kFloat8_e4m3fn)); outs.push_back(like(x, {M, N / 128}, at::kFloat)); }
    if (colwise) { outs.push_back(like(x, {N, M}, at::kFloat8_e4m3fn)); outs.push_back(like(x, {N, M / 128}, at::kFloat)); }
    return outs;
}
std::tuple<at::Tensor, at::Tensor> fp8_block128x128_meta(const at::Tensor &x, bool)
{
    check_x(x);
    return {like(x, {x.size(0), x.size(1)}, at::kFloat8_e4m3fn), like(x, {x.size(0) / 128, x.size(1) / 128}, at::kFloat)};
}
std::vector<at::Tensor> mxfp8_32x32_meta(const at::Tensor &x, bool rowwise, bool colwise, bool swizzle, bool transposed_data)
{
    check_x(x);
    const int64_t M = x.size(0), N = x.size(1);
    std::vector<at::Tensor> outs;
    if (rowwise) {
        outs.push_back(like(x, {M, N}, at::kFloat8_e4m3fn));
        outs.push_back(like(x, swizzle ? blocked_shape(M, N / 32) : std::vector<int64_t>{M / 32, N / 32}, at::kFloat8_e8m0fnu));
    }
    if (colwise) {
        if (transposed_data) outs.push_back(like(x, {N, M}, at::kFloat8_e4m3fn));
        outs.push_back(like(x, blocked_shape(N, M / 32), at::kFloat8_e8m0fnu));
    }
    return outs;
}
std::tuple<at::Tensor, at::Tensor> mxfp4_meta(const at::Tensor &x, bool swizzle)
{
    check_x(x);
    return {like(x, {x.size(0), x.size(1) / 2}, at::kFloat4_e2m1fn_x2), like(x, scale_shape(x.size(0), x.size(1) / 32, swizzle), at::kFloat8_e8m0fnu)};
}

at::Tensor nvfp4_per_token_scale_meta(const at::Tensor &x, bool)
{
    check_x(x);
    return like(x, {x.size(0), 1}, at::kFloat);
}
at::Tensor sr_f32_to_bf16_meta(const at::Tensor &x, const at::Tensor &, int64_t, int64_t, int64_t)
{
    TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kFloat, "quant_cast_cuda: sr_f32_to_bf16 takes a 2-D fp32 tensor");
    return like(x, x.sizes().vec(), at::kBFloat16);
}

std::tuple<at::Tensor, at::Tensor> int8_rowwise_meta(const at::Tensor &x, bool)
{
    check_x(x);
    return {like(x, {x.size(0), x.size(1)}, at::kChar), like(x, {x.size(0), 1}, at::kFloat)};
}
at::Tensor int8_scaled_mm_meta(const at::Tensor &a, const at::Tensor &b, const at::Tensor &, const at::Tensor &, const std::optional<at::Tensor> &, at::ScalarType out_dtype)
{
    check_product(a, b);
    out_kind(out_dtype);
    return like(a, {a.size(0), b.size(0)}, out_dtype);
}
at::Tensor nvfp4_kv_append_meta(const at::Tensor &k, const at::Tensor &, at::Tensor, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                                const std::optional<at::Tensor> &, const std::optional<at::Tensor> &, bool, const std::optional<at::Tensor> &q, bool)
{
    TORCH_CHECK(k.dim() == 3 && (!q || q->dim() == 3), "quant_cast_cuda: k and q must be 3-D");
    return like(k, {q ? k.size(0) : 0, q ? q->size(1) : 0, k.size(2)}, at::kBFloat16);
}
std::tuple<at::Tensor, at::Tensor> nvfp4_kv_gather_meta(const at::Tensor &cache, const at::Tensor &, const at::Tensor &, int64_t total, int64_t head_dim,
                                                        const at::Tensor &, const at::Tensor &)
{
    TORCH_CHECK(cache.dim() == 4, "quant_cast_cuda: cache must be 4-D");
    return {like(cache, {total, cache.size(1), head_dim}, at::kBFloat16), like(cache, {total, cache.size(1), head_dim}, at::kBFloat16)};
}
std::tuple<at::Tensor, at::Tensor> nvfp4_kv_attention_meta(const at::Tensor &q, const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                                                           const at::Tensor &, const std::optional<at::Tensor> &, int64_t, std::optional<double> scale)
{
    check_scale(scale);
    TORCH_CHECK(q.dim() == 3, "quant_cast_cuda: q must be (rows, q_heads, head_dim)");
    return {like(q, q.sizes().vec(), at::kBFloat16), like(q, {q.size(0), q.size(1)}, at::kFloat)};
}

}  // namespace

TORCH_LIBRARY(quant_cast_cuda_native, m)
{
    m.def("amax(Tensor x, str kind, str fmt, bool recip_div=False) -> Tensor");
    m.def("fp8_tensorwise(Tensor x, Tensor scale, str fmt) -> Tensor");
    m.def("fp8_rowwise(Tensor x, str fmt, bool recip_div=False) -> (Tensor, Tensor)");
    m.def("fp8_colwise(Tensor x, str fmt, bool recip_div=False) -> (Tensor, Tensor)");
    m.def("mxfp8(Tensor x, bool rowwise, bool colwise, bool swizzle, str mode) -> Tensor[]");
    m.def("nvfp4(Tensor x, Tensor outer_scale, bool swizzle, bool transposed, bool recip_div=False) -> (Tensor, Tensor)");
    m.def("nvfp4_sr(Tensor x, Tensor outer_scale, Tensor key, bool swizzle, bool transposed, bool recip_div=False) -> (Tensor, Tensor)");
    m.def("nvfp4_both(Tensor x, Tensor outer_scale, bool swizzle, bool recip_div=False) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("fp8_rowwise_precalc(Tensor x, Tensor scale, str fmt) -> Tensor");
    m.def("fp8_colwise_precalc(Tensor x, Tensor scale, str fmt) -> Tensor");
    m.def("fp8_block128(Tensor x, bool rowwise, bool colwise, bool recip_div=False) -> Tensor[]");
    m.def("fp8_block128x128(Tensor x, bool recip_div=False) -> (Tensor, Tensor)");
    m.def("mxfp8_32x32(Tensor x, bool rowwise, bool colwise, bool swizzle, bool transposed_data=True) -> Tensor[]");
    m.def("mxfp4(Tensor x, bool swizzle) -> (Tensor, Tensor)");
    m.def("nvfp4_per_token_scale(Tensor x, bool recip_div=False) -> Tensor");
    m.def("int8_rowwise(Tensor x, bool recip_div=False) -> (Tensor, Tensor)");
    m.def("int8_scaled_mm(Tensor a, Tensor b, Tensor scale_a, Tensor scale_b, Tensor? bias=None, ScalarType out_dtype=bfloat16) -> Tensor");
    m.def("nvfp4_kv_append(Tensor k, Tensor v, Tensor(a!) cache, Tensor slots, Tensor k_outer, Tensor v_outer, Tensor? positions=None, "
          "Tensor? cos_sin=None, bool interleaved=False, Tensor? q=None, bool recip_div=False) -> Tensor");
    m.def("nvfp4_kv_gather(Tensor cache, Tensor block_table, Tensor cu_kv, int total, int head_dim, Tensor k_outer, Tensor v_outer) -> (Tensor, Tensor)");
    m.def("nvfp4_kv_attention(Tensor q, Tensor cache, Tensor block_table, Tensor kv_lens, Tensor k_outer, Tensor v_outer, Tensor? cu_q=None, "
          "int max_q=1, float? scale=None) -> (Tensor, Tensor)");
    m.def("sr_f32_to_bf16(Tensor x, Tensor key, int global_row=0, int global_col=0, int num_col=-1) -> Tensor");
}

TORCH_LIBRARY_IMPL(quant_cast_cuda_native, CUDA, m)
{
    m.impl("amax", amax_cuda);
    m.impl("fp8_tensorwise", fp8_tensorwise_cuda);
    m.impl("fp8_rowwise", fp8_rowwise_cuda);
    m.impl("fp8_colwise", fp8_colwise_cuda);
    m.impl("mxfp8", mxfp8_cuda);
    m.impl("nvfp4", nvfp4_cuda);
    m.impl("nvfp4_sr", nvfp4_sr_cuda);
    m.impl("nvfp4_both", nvfp4_both_cuda);
    m.impl("fp8_rowwise_precalc", fp8_rowwise_precalc_cuda);
    m.impl("fp8_colwise_precalc", fp8_colwise_precalc_cuda);
    m.impl("fp8_block128", fp8_block128_cuda);
    m.impl("fp8_block128x128", fp8_block128x128_cuda);
    m.impl("mxfp8_32x32", mxfp8_32x32_cuda);
    m.impl("mxfp4", mxfp4_cuda);
    m.impl("nvfp4_per_token_scale", nvfp4_per_token_scale_cuda);
    m.impl("int8_rowwise", int8_rowwise_cuda);
    m.impl("int8_scaled_mm", int8_scaled_mm_cuda);
    m.impl("nvfp4_kv_append", nvfp4_kv_append_cuda);
    m.impl("nvfp4_kv_gather", nvfp4_kv_gather_cuda);
    m.impl("nvfp4_kv_attention", nvfp4_kv_attention_cuda);
    m.impl("sr_f32_to_bf16", sr_f32_to_bf16_cuda);
}

TORCH_LIBRARY_IMPL(quant_cast_cuda_native, Meta, m)
{
    m.impl("amax", amax_meta);
    m.impl("fp8_tensorwise", fp8_tensorwise_meta);
    m.impl("fp8_rowwise", fp8_rowwise_meta);
    m.impl("fp8_colwise", fp8_colwise_meta);
    m.impl("mxfp8", mxfp8_meta);
    m.impl("nvfp4", nvfp4_meta);
    m.impl("nvfp4_sr", nvfp4_sr_meta);
    m.impl("nvfp4_both", nvfp4_both_meta);
    m.impl("fp8_rowwise_precalc", fp8_rowwise_precalc_meta);
    m.impl("fp8_colwise_precalc", fp8_colwise_precalc_meta);
    m.impl("fp8_block128", fp8_block128_meta);
    m.impl("fp8_block128x128", fp8_block128x128_meta);
    m.impl("mxfp8_32x32", mxfp8_32x32_meta);
    m.impl("mxfp4", mxfp4_meta);
    m.impl("nvfp4_per_token_scale", nvfp4_per_token_scale_meta);
    m.impl("int8_rowwise", int8_rowwise_meta);
    m.impl("int8_scaled_mm", int8_scaled_mm_meta);
    m.impl("nvfp4_kv_append", nvfp4_kv_append_meta);
    m.impl("nvfp4_kv_gather", nvfp4_kv_gather_meta);
    m.impl("nvfp4_kv_attention", nvfp4_kv_attention_meta);
    m.impl("sr_f32_to_bf16", sr_f32_to_bf16_meta);
}
