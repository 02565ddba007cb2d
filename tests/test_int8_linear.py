"""The 8-bit integer linear layer: cast bit for bit, product against 64-bit sums.

Product tolerance: the integer sum is exact; it is rounded to fp32 (2^-24), multiplied by two scales (2^-24 each), a bias is
added (2^-24 of the result), and the result is rounded to the output type (half a step, finfo.eps / 2; fp16 below its smallest
normal number: half of 2^-24)."""
import pytest
import torch

from quant_cast_bench_b200 import quant_cast_cuda as Q
from quant_cast_bench_b200.quant_cast_cuda import _lib as L

gpu = pytest.mark.gpu


def cast_ref(x, mode="ieee"):
    """rowwise int8 in fp32 on the CPU, every operation rounded on its own."""
    f = x.float()
    a = f.abs().amax(1, keepdim=True)
    a = torch.where(a < 1e-12, torch.tensor(1e-12, dtype=torch.bfloat16).float(), a)
    s = a / 127.0 if mode == "ieee" else a * (torch.tensor(1.0) / torch.tensor(127.0))
    return (f * (1.0 / s)).round().to(torch.int8), s


def product_ref(a, b, sa, sb, bias, dtype):
    """64-bit result and the tolerance of the module's docstring."""
    y = (a.double() @ b.double().T) * sa.double().view(-1, 1) * sb.double().view(1, -1)
    tol = 3.01 * 2.0 ** -24 * y.abs()
    if bias is not None:
        y = y + bias.double().view(1, -1)
        tol = tol + 1.01 * 2.0 ** -24 * y.abs()
    tol = tol + (y.abs() + tol) * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    return y, tol


def random_codes(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, dtype=torch.int8)


def make(M, N, K, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    a, b = random_codes(g, M, K), random_codes(g, N, K)
    sa = torch.rand(M, 1, generator=g) * 0.01 + 1e-4
    sb = torch.rand(N, 1, generator=g) * 0.001 + 1e-5
    return a, b, sa, sb, torch.randn(N, generator=g).to(torch.bfloat16) if bias else None


def run(a, b, sa, sb, bias, dtype, fn=None):
    return (fn or Q.int8_scaled_mm_cuda)(a.cuda(), b.cuda(), sa.cuda(), sb.cuda(), bias=None if bias is None else bias.cuda(), out_dtype=dtype)


def check(a, b, sa, sb, bias, dtype, fn=None):
    y, tol = product_ref(a, b, sa, sb, bias, dtype)
    got = run(a, b, sa, sb, bias, dtype, fn)
    assert got.dtype == dtype and got.shape == y.shape
    err = (got.cpu().double() - y).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max())} of the tolerance"
    return got


# ------------------------------------------------------------------------------------------------ refusals, no GPU needed
def test_python_refusals_on_cpu():
    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        Q.rowwise_int8_cuda(x)
    with pytest.raises(ValueError):
        Q.int8_scaled_mm_cuda(x.to(torch.int8), x.to(torch.int8), torch.ones(4), torch.ones(4))


def test_c_refusals():
    lib = L.load()
    p = 1 << 20      # a 16-byte aligned number; nothing is launched
    assert lib.qcc_int8_rowwise(p, 4, 0, 0, p, p, None) == -1
    assert lib.qcc_int8_rowwise(p, -1, 8, 0, p, p, None) == -1
    assert lib.qcc_int8_rowwise(p, 4, 8, 1, p, p, None) == -3
    assert lib.qcc_int8_rowwise(None, 4, 8, 0, p, p, None) == -3
    assert lib.qcc_int8_rowwise(p + 2, 4, 8, 0, p, p, None) == -2
    assert lib.qcc_int8_rowwise(None, 0, 8, 0, None, None, None) == 0

    def mm(a=p, b=p, M=4, N=4, K=32, sa=p, sb=p, kind=0, out=p):
        return lib.qcc_int8_scaled_mm(a, b, M, N, K, sa, sb, None, kind, out, None)
    assert mm(K=0) == -1 and mm(K=24) == -1 and mm(K=131072) == -1 and mm(M=-1) == -1
    assert mm(kind=3) == -3 and mm(a=None) == -3 and mm(sb=None) == -3
    assert mm(a=p + 1) == -2 and mm(out=p + 2) == -2
    assert mm(M=0, a=None) == 0 and mm(N=0, b=None) == 0


# ------------------------------------------------------------------------------------------------ cast
@gpu
@pytest.mark.parametrize("M,N", [(1, 1), (1, 4096), (3, 7), (5, 8), (17, 2048), (2, 2056), (9, 4104), (4, 8200), (3, 16384), (2, 16400), (2, 16385), (130, 333)])
def test_cast_bits(M, N):
    g = torch.Generator().manual_seed(M * 1000 + N)
    x = (torch.randn(M, N, generator=g) * torch.exp(2 * torch.randn(M, 1, generator=g))).to(torch.bfloat16)
    x[0, 0] = 3.0 if M > 1 else x[0, 0]
    if M > 2:
        x[1] = 0                                     # an empty row
        x[2] = torch.where(torch.rand(N, generator=g) < 0.5, 1e-20, -1e-30).to(torch.bfloat16)
    for mode in ("ieee", "cuda_eager"):
        with Q.scalar_division(mode):
            q, s = Q.rowwise_int8_cuda(x.cuda())
        wq, ws = cast_ref(x, mode)
        assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)


@gpu
def test_cast_ties_go_to_even_and_extremes():
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -127.0, 126.5]], dtype=torch.bfloat16)
    q, s = Q.rowwise_int8_cuda(x.cuda())
    assert float(s) == 1.0 and q.cpu().tolist() == [[127, 0, 2, 2, 0, -2, -127, 126]]
    big = torch.tensor([[3e38, -3e38, 1e38, 0.0]], dtype=torch.bfloat16)
    q, s = Q.rowwise_int8_cuda(big.cuda())
    wq, ws = cast_ref(big)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


@gpu
@pytest.mark.parametrize("N", [8, 333, 20000])
def test_cast_nan_and_inf_reach_the_scale_only_of_their_row(N):
    x = torch.ones(4, N, dtype=torch.bfloat16)
    x[1, N - 1] = float("nan")
    x[2, N // 2] = float("-inf")
    q, s = Q.rowwise_int8_cuda(x.cuda())
    s = s.cpu().view(-1)
    assert float(s[0]) == float(s[3]) and torch.isnan(s[1]) and torch.isinf(s[2])
    assert bool((q.cpu()[[0, 3]] == 127).all())
    w = torch.ones(16, 16 * (N // 16 + 1), dtype=torch.int8)
    a = torch.zeros(4, w.shape[1], dtype=torch.int8)
    a[:, :N] = q.cpu()
    y = Q.int8_scaled_mm_cuda(a.cuda(), w.cuda(), s.view(-1, 1).cuda(), torch.ones(16, 1).cuda())
    assert not bool(torch.isfinite(y[1:3]).any()) and bool(torch.isfinite(y[[0, 3]]).all())


@gpu
def test_cast_empty():
    q, s = Q.rowwise_int8_cuda(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 64) and s.shape == (0, 1)


# ------------------------------------------------------------------------------------------------ product
@gpu
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 64, 65, 128, 129, 255, 257, 600])
@pytest.mark.parametrize("N,K", [(1, 16), (127, 128), (129, 144), (300, 2064), (1000, 4096)])
def test_product_shapes(M, N, K):
    check(*make(M, N, K, bias=(M + N) % 2 == 0, seed=M), dtype=torch.float32)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M", [3, 130, 513])
def test_product_types(dtype, bias, M):
    check(*make(M, 389, 528, bias, seed=5), dtype=dtype)


@gpu
@pytest.mark.parametrize("M,N,K", [(4, 128, 131056), (200, 300, 32768)])
def test_product_of_the_largest_codes_does_not_overflow(M, N, K):
    for u, v in ((-128, -128), (127, 127), (127, -128)):
        a, b = torch.full((M, K), u, dtype=torch.int8), torch.full((N, K), v, dtype=torch.int8)
        check(a, b, torch.full((M, 1), 0.25), torch.full((N, 1), 2.0 ** -10), None, torch.float32)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(90, 10001, 256), (150, 10001, 272), (190, 10000, 256), (200, 10001, 272), (600, 4096, 2048), (1111, 5003, 272), (2000, 4096, 1040)])
def test_product_tiles_between_the_powers_of_two(M, N, K, dtype):
    """Shapes that on 148 SMs take tiles of 96, 160, 192 and 224 tokens, one tile a CTA and several."""
    check(*make(M, N, K, True, seed=M), dtype=dtype)


@gpu
def test_product_many_tiles_and_rows():
    """More tiles than SMs, several groups of token tiles, both accumulators of the persistent loop."""
    check(*make(2600, 1300, 256, True, seed=9), dtype=torch.bfloat16)
    check(*make(1, 40000, 64, False, seed=10), dtype=torch.bfloat16)
    check(*make(20000, 130, 64, False, seed=11), dtype=torch.float16)


@gpu
def test_product_empty():
    z = torch.empty(0, 32, dtype=torch.int8, device="cuda")
    b = torch.ones(5, 32, dtype=torch.int8, device="cuda")
    assert Q.int8_scaled_mm_cuda(z, b, torch.empty(0, 1, device="cuda"), torch.ones(5, 1, device="cuda")).shape == (0, 5)
    assert Q.int8_scaled_mm_cuda(b, z, torch.ones(5, 1, device="cuda"), torch.empty(0, 1, device="cuda")).shape == (5, 0)


@gpu
def test_product_refusals():
    a = torch.ones(4, 32, dtype=torch.int8, device="cuda")
    s = torch.ones(4, 1, device="cuda")
    for bad in (lambda: Q.int8_scaled_mm_cuda(a, a[:, :16], s, s), lambda: Q.int8_scaled_mm_cuda(a, a[:, :24].contiguous(), s, s),
                lambda: Q.int8_scaled_mm_cuda(a.float(), a, s, s), lambda: Q.int8_scaled_mm_cuda(a, a, s[:3], s),
                lambda: Q.int8_scaled_mm_cuda(a, a, s.double(), s), lambda: Q.int8_scaled_mm_cuda(a, a, s, s, bias=torch.ones(4, device="cuda")),
                lambda: Q.int8_scaled_mm_cuda(a, a.cpu(), s, s), lambda: Q.int8_scaled_mm_cuda(a[:, :24], a[:, :24], s, s)):
        with pytest.raises((AssertionError, ValueError)):
            bad()
    with pytest.raises(ValueError):
        Q.int8_scaled_mm_cuda(a, a, s, s, out_dtype=torch.int32)


@gpu
def test_product_on_a_stream_and_in_a_graph():
    a, b, sa, sb, bias = make(5, 777, 1024, True, seed=3)
    want = run(a, b, sa, sb, bias, torch.bfloat16)
    big = make(700, 777, 1024, True, seed=4)
    want_big = run(*big, torch.bfloat16)
    dev = [t.cuda() for t in (a, b, sa, sb, bias)]
    devb = [t.cuda() for t in big]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = Q.int8_scaled_mm_cuda(*dev)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = Q.int8_scaled_mm_cuda(*dev)
        z = Q.int8_scaled_mm_cuda(*devb)
    for _ in range(3):
        y.zero_()
        z.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want_big)


@gpu
def test_native_operators_give_the_same_bits():
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops as N
    x = torch.randn(37, 528, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    q, s = Q.rowwise_int8_cuda(x)
    nq, ns = N.rowwise_int8_native(x)
    assert torch.equal(q, nq) and torch.equal(s, ns)
    a = make(37, 100, 528, True, seed=2)
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        assert torch.equal(run(*a, dt), run(*a, dt, fn=N.int8_scaled_mm_native))
    with pytest.raises(RuntimeError):
        N.int8_scaled_mm_native(q, q[:, :512].contiguous(), s, s)
    with pytest.raises(RuntimeError):
        N.int8_scaled_mm_native(q, q, s[:5], s)


def test_native_shapes_without_a_gpu():
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops as N
    x = torch.empty(6, 64, dtype=torch.bfloat16, device="meta")
    q, s = N.rowwise_int8_native(x)
    assert q.shape == (6, 64) and q.dtype == torch.int8 and s.shape == (6, 1) and s.dtype == torch.float32
    y = N.int8_scaled_mm_native(q, torch.empty(9, 64, dtype=torch.int8, device="meta"), s, torch.empty(9, 1, device="meta"), out_dtype=torch.float16)
    assert y.shape == (6, 9) and y.dtype == torch.float16
    with pytest.raises((RuntimeError, NotImplementedError)):
        N.rowwise_int8_native(torch.zeros(2, 32, dtype=torch.bfloat16))
    for k in (24, 0):      # a refusal whose text holds numbers
        with pytest.raises(RuntimeError, match=f"131056, got {k}"):
            N.int8_scaled_mm_native(q[:, :k], torch.empty(9, k, dtype=torch.int8, device="meta"), s, s)
