"""8-bit integer linear layer: the int8 cast of activations (one scale per token, the sibling of rowwise_fp8_cuda) and the
product that consumes it (scales per token and per output channel).  No counterpart in the reference.

    q, s = rowwise_int8_cuda(x)                        # x (M, K) bf16 -> int8 (M, K), fp32 (M, 1)
    w, ws = rowwise_int8_cuda(weight)                  # once: weight (N, K)
    y = int8_scaled_mm_cuda(q, w, s, ws, bias=bias)    # (M, N)
"""
import torch

from . import _lib as L
from .recipes import _check_x, _on_device, _p, _stream

_OUT = {torch.bfloat16: L.OUT_BF16, torch.float16: L.OUT_F16, torch.float32: L.OUT_F32}


def rowwise_int8_cuda(x):
    """(qdata (M, N) int8, scale (M, 1) fp32): scale = max(amax, bf16(1e-12)) / 127, q = round(x * (1 / scale)), ties to even:
    the recipe of rowwise_fp8_f (G:301-307) with 127 for the fp8 maximum.  A row with a NaN gets a NaN scale."""
    lib = L.load()
    _check_x(x)
    M, N = x.shape
    assert N >= 1, "rowwise_int8 needs at least one column"
    q = torch.empty((M, N), dtype=torch.int8, device=x.device)
    s = torch.empty((M, 1), dtype=torch.float32, device=x.device)
    with _on_device(x.device):
        L.check(lib.qcc_int8_rowwise(_p(x), M, N, L.div_flag(), _p(q), _p(s), _stream(x)), "int8_rowwise")
    L.launch_count += 1
    return q, s


def int8_scaled_mm_cuda(a, b, scale_a, scale_b, bias=None, out_dtype=torch.bfloat16):
    """out (M, N) = (a @ b.T) * scale_a * scale_b.T + bias.  a (M, K), b (N, K) contiguous int8; scale_a M and scale_b N fp32
    values; bias N bf16 values or None; out_dtype bf16, fp16 or fp32.  The sum is exact (32-bit integers), the scales are applied in fp32,
    one rounding to out_dtype.  K % 16 == 0, 16 <= K <= 131056; any M and N."""
    lib = L.load()
    if not (isinstance(a, torch.Tensor) and a.is_cuda):
        raise ValueError("a must be a CUDA tensor (quant_cast_cuda has no CPU path)")
    for t, name in ((a, "a"), (b, "b")):
        assert t.dtype == torch.int8 and t.dim() == 2 and t.is_contiguous() and t.device == a.device, f"{name} must be a contiguous 2-D int8 tensor on a's device"
    M, K = a.shape
    N = b.shape[0]
    assert b.shape[1] == K, f"a is {M}x{K}, b is {N}x{b.shape[1]}: the second dimensions differ"
    assert K % 16 == 0 and 16 <= K <= L.INT8_MAX_K, f"int8_scaled_mm needs K % 16 == 0 and 16 <= K <= {L.INT8_MAX_K}, got K={K}"
    for t, n, name in ((scale_a, M, "scale_a"), (scale_b, N, "scale_b")):
        assert t.device == a.device and t.dtype == torch.float32 and t.numel() == n and t.is_contiguous(), f"{name}: {n} contiguous fp32 values on a's device"
    assert bias is None or (bias.device == a.device and bias.dtype == torch.bfloat16 and bias.numel() == N and bias.is_contiguous()), "bias: N contiguous bf16 values on a's device"
    if out_dtype not in _OUT:
        raise ValueError(f"out_dtype must be bfloat16, float16 or float32, not {out_dtype}")
    out = torch.empty((M, N), dtype=out_dtype, device=a.device)
    with _on_device(a.device):
        L.check(lib.qcc_int8_scaled_mm(_p(a), _p(b), M, N, K, _p(scale_a), _p(scale_b), _p(bias), _OUT[out_dtype], _p(out), _stream(a)), "int8_scaled_mm")
    L.launch_count += 1
    return out
