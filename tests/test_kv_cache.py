"""The paged nvfp4 key/value cache: append and read-back bit for bit against fp32 arithmetic on the CPU, attention against 64 bits.

Attention tolerance, element by element, with p the exact probabilities, A = sum p |v|, N keys and D elements:
  scores: a dot product of D exact products summed in fp32, at most D * 2^-23 * sum |q k| * scale, then one factor 2^-23 |s|;
  an error e of all scores changes a probability by at most e, its weight and the sum: 2 e A;
  P is rounded to fp16: 2^-11 A, and below fp16's normal numbers by half of 2^-24 against a largest P of at least 1: N 2^-25 max |v|;
  exp2 and the fp32 sums: (N + 64) 2^-23 A;   the result is rounded to bf16: 2^-8 |o|.
lse: e, the sum's (N + 64) 2^-23, and 2^-22 of its size for the logarithm and the products."""
import math

import pytest
import torch

from quant_cast_bench_b200 import quant_cast_cuda as Q
from quant_cast_bench_b200.quant_cast_cuda import _lib as L

gpu = pytest.mark.gpu
CODE = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)


def planes(cache, D):
    page = cache.shape[-1] * 16 // (9 * D)
    return cache[..., :page * D // 2].unflatten(-1, (page, D // 2)), cache[..., page * D // 2:].unflatten(-1, (page, D // 16))


def values(cache, D):
    """(pages, heads, 2, page, D) in 64 bits, without the outer scales."""
    codes, scales = planes(cache.cpu(), D)
    v = torch.stack([CODE[(codes & 15).long()], CODE[(codes >> 4).long()]], -1).flatten(-2)
    return v * scales.contiguous().view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)


def nvfp4_ref(x, outer, mode="ieee"):
    """Codes and scale bytes of x (..., D) in fp32 on the CPU."""
    b = x.float().unflatten(-1, (-1, 16))
    amax = b.abs().amax(-1)
    six = amax / 6.0 if mode == "ieee" else amax * (torch.tensor(1.0) / torch.tensor(6.0))
    inner = (six / outer).clamp(0.015625, 448.0).to(torch.float8_e4m3fn)
    y = b * ((1.0 / outer) / inner.float()).unsqueeze(-1)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0) + 8 * torch.signbit(y)).flatten(-2)
    code = code.byte()
    return code[..., 0::2] + 16 * code[..., 1::2], inner.view(torch.uint8)


def rotate_ref(x, cos, sin, interleaved):
    x = x.float().clone()
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2].clone(), x[..., 1:r:2].clone()) if interleaved else (x[..., :r // 2].clone(), x[..., r // 2:r].clone())
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    ra, rb = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:r:2], x[..., 1:r:2] = ra, rb
    else:
        x[..., :r // 2], x[..., r // 2:r] = ra, rb
    return x


def rotation_table(n, rot):
    t = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return torch.cat([t.cos(), t.sin()], 1).float()


def random_cache(g, pages, heads, page, D):
    """A cache of quantised normals and its outer scales, on the CPU."""
    ko, vo = torch.tensor([0.0041]), torch.tensor([0.0033])
    cache = torch.empty(pages, heads, 2, page * 9 * D // 16, dtype=torch.uint8)
    codes, scales = planes(cache, D)
    for w, o in ((0, ko), (1, vo)):
        c, s = nvfp4_ref(torch.randn(pages, heads, page, D, generator=g) * 1.5, o)
        codes[:, :, w], scales[:, :, w] = c, s
    return cache, ko, vo


def batch(g, lens, page, spare=3):
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)     # entries behind a sequence are never followed
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


# ------------------------------------------------------------------------------------------------ refusals, no GPU needed
def test_python_refusals_on_cpu():
    k = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    cache = torch.zeros(1, 1, 2, 16 * 36, dtype=torch.uint8)
    o = torch.ones(1)
    with pytest.raises(ValueError):
        Q.nvfp4_kv_append_cuda(k, k, cache, torch.zeros(1, dtype=torch.int64), o, o)
    with pytest.raises(ValueError):
        Q.nvfp4_kv_gather_cuda(cache, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 0, 64, o, o)
    with pytest.raises(ValueError):
        Q.nvfp4_kv_attention_cuda(k, cache, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), o, o)
    for args in ((4, 1, 24, 64), (4, 1, 16, 96), (4, 0, 16, 64)):
        with pytest.raises(AssertionError):
            Q.nvfp4_kv_cache_cuda(*args, device="cpu")
    assert Q.nvfp4_kv_cache_cuda(4, 2, 16, 64, device="cpu").shape == (4, 2, 2, 16 * 36)


def test_c_refusals():
    import ctypes
    lib = L.load()
    p = 1 << 20       # a 16-byte aligned number; nothing is launched
    assert lib.qcc_nvfp4_kv_page_bytes(8, 16, 128) == 8 * 2 * 16 * 72 and lib.qcc_nvfp4_kv_page_bytes(8, 24, 128) == 0
    assert lib.qcc_nvfp4_kv_page_bytes(8, 16, 96) == 0

    def append(**kw):
        d = dict(k=p, v=p, q=p, q_out=p, k_stride=(512, 64), v_stride=(512, 64), q_stride=(512, 64), tokens=4, cache=p, num_pages=4, slots=p, positions=p,
                 cos_sin=p, max_pos=10, k_outer=p, v_outer=p, kv_heads=2, q_heads=4, head_dim=64, page=16, rot=64, flags=0) | kw
        for s in ("k_stride", "v_stride", "q_stride"):
            d[s] = (ctypes.c_int64 * 2)(*d[s])
        return lib.qcc_nvfp4_kv_append(ctypes.byref(L.KvAppendArgs(**d)), None)
    for kw in (dict(head_dim=96), dict(page=24), dict(kv_heads=0), dict(rot=48), dict(rot=128), dict(rot=-32), dict(tokens=-1), dict(q_heads=-1)):
        assert append(**kw) == -1, kw
    for kw in (dict(k=None), dict(slots=None), dict(v_outer=None), dict(cos_sin=None), dict(positions=None), dict(q=None), dict(flags=1), dict(max_pos=0)):
        assert append(**kw) == -3, kw
    for kw in (dict(k=p + 8), dict(cache=p + 4), dict(k_stride=(512, 60)), dict(q_stride=(500, 64)), dict(cos_sin=p + 4), dict(q_out=p + 2)):
        assert append(**kw) == -2, kw
    assert append(tokens=0, k=None) == 0 and lib.qcc_nvfp4_kv_append(None, None) == -3

    def gather(heads=2, page=16, D=64, total=4, cache=p, k=p, table=p, width=4):
        return lib.qcc_nvfp4_kv_gather(cache, 4, heads, page, D, table, 4, width, p, 1, total, p, p, k, p, None)
    assert gather(heads=0) == -1 and gather(page=8) == -1 and gather(D=32) == -1 and gather(total=-1) == -1
    assert gather(cache=None) == -3 and gather(table=None) == -3 and gather(k=p + 2) == -2 and gather(total=0, cache=None) == 0

    def attention(ws=p, ws_bytes=1 << 40, **kw):
        d = dict(q=p, q_stride=(512, 64), rows=4, cache=p, num_pages=4, table=p, table_stride=4, table_width=4, kv_lens=p, cu_q=None, seqs=4, max_q=1,
                 k_outer=p, v_outer=p, scale=1.0, q_heads=4, kv_heads=2, head_dim=64, page=16, out=p, lse=p) | kw
        d["q_stride"] = (ctypes.c_int64 * 2)(*d["q_stride"])
        return lib.qcc_nvfp4_kv_attention(ctypes.byref(L.KvAttentionArgs(**d)), ws, ws_bytes, None)
    for kw in (dict(head_dim=96), dict(page=24), dict(kv_heads=3), dict(kv_heads=8), dict(seqs=5000, rows=5000), dict(rows=3), dict(max_q=0), dict(table_width=1 << 27)):
        assert attention(**kw) == -1, kw
    for kw in (dict(q=None), dict(cache=None), dict(kv_lens=None), dict(table=None), dict(out=None)):
        assert attention(**kw) == -3, kw
    assert attention(q=p + 2) == -2 and attention(q_stride=(512, 60)) == -2
    assert attention(ws=None) == -4 and attention(ws_bytes=16) == -4 and attention(ws=p + 4) == -2
    assert attention(seqs=0, rows=0, q=None) == 0 and lib.qcc_nvfp4_kv_attention(None, p, 1, None) == -3


def test_c_refuses_a_scale_that_is_not_positive():
    import ctypes
    lib, p = L.load(), 1 << 20
    for scale in (0.0, -0.125, float("nan")):
        a = L.KvAttentionArgs(p, (ctypes.c_int64 * 2)(512, 64), 4, p, 4, p, 4, 4, p, None, 4, 1, p, p, scale, 4, 2, 64, 16, p, p)
        assert lib.qcc_nvfp4_kv_attention(ctypes.byref(a), p, 1 << 40, None) == -3


def test_native_shapes_without_a_gpu():
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops as N

    def meta(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="meta")
    cache, o = meta(4, 2, 2, 16 * 36, dtype=torch.uint8), meta(1, dtype=torch.float32)
    q = N.nvfp4_kv_append_native(meta(3, 2, 64), meta(3, 2, 64), cache, meta(3, dtype=torch.int64), o, o, q=meta(3, 4, 64))
    assert q.shape == (3, 4, 64)
    k, v = N.nvfp4_kv_gather_native(cache, meta(1, 4, dtype=torch.int32), meta(2, dtype=torch.int32), 7, 64, o, o)
    assert k.shape == v.shape == (7, 2, 64) and k.dtype == torch.bfloat16
    out, lse = N.nvfp4_kv_attention_native(q, cache, meta(3, 4, dtype=torch.int32), meta(3, dtype=torch.int32), o, o)
    assert out.shape == (3, 4, 64) and lse.shape == (3, 4) and lse.dtype == torch.float32


# ------------------------------------------------------------------------------------------------ append and read-back
APPEND = [  # D, page, kv heads, q heads, rot, interleaved, tokens
    (128, 16, 8, 32, 128, False, 5), (128, 32, 2, 0, 128, False, 67), (128, 64, 1, 4, 64, False, 33), (128, 128, 3, 3, 32, False, 130),
    (128, 16, 2, 10, 96, False, 9), (64, 16, 2, 4, 64, False, 40), (64, 32, 1, 12, 32, True, 21), (64, 64, 4, 4, 64, True, 1),
    (128, 16, 2, 2, 128, True, 50), (128, 32, 2, 2, 64, True, 7), (64, 128, 5, 0, 0, False, 300), (128, 16, 1, 1, 0, False, 1), (64, 16, 1, 0, 32, False, 2),
    (128, 32, 8, 32, 128, False, 1500), (128, 64, 4, 17, 128, True, 1100),       # millions of roundings
]


def append_inputs(D, page, heads, qh, rot, tokens, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(tokens, qh + 2 * heads, D, generator=g).to(torch.bfloat16)
    pages = -(-tokens // page) + 3
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots = torch.where(torch.rand(tokens, generator=g) < 0.1, -1 - slots, slots)        # some rows are padding
    pos = torch.randint(0, 500, (tokens,), generator=g)
    cache = torch.randint(0, 256, (pages, heads, 2, page * 9 * D // 16), generator=g, dtype=torch.uint8)
    return qkv, slots, pos, cache, torch.tensor([0.0037]), torch.tensor([0.0021]), rotation_table(500, rot) if rot else None


def append_ref(qkv, qh, heads, slots, pos, cache, ko, vo, table, interleaved, mode="ieee"):
    D = qkv.shape[2]
    page = cache.shape[3] * 16 // (9 * D)
    k, v, q = qkv[:, qh:qh + heads], qkv[:, qh + heads:], qkv[:, :qh]
    if table is not None:
        cos, sin = table[pos].chunk(2, 1)
        k, q = rotate_ref(k, cos, sin, interleaved), rotate_ref(q, cos, sin, interleaved)
    codes, scales = planes(cache, D)
    keep = slots >= 0
    at, off = slots[keep] // page, slots[keep] % page
    for w, x, o in ((0, k, ko), (1, v, vo)):
        c, s = nvfp4_ref(x[keep], o, mode)
        codes[at, :, w, off], scales[at, :, w, off] = c, s
    return q.to(torch.bfloat16)


@gpu
@pytest.mark.parametrize("D,page,heads,qh,rot,interleaved,tokens", APPEND)
def test_append_bits(D, page, heads, qh, rot, interleaved, tokens):
    for mode in ("ieee", "cuda_eager"):
        qkv, slots, pos, cache, ko, vo, table = append_inputs(D, page, heads, qh, rot, tokens, seed=D + tokens)
        dev = qkv.cuda()
        got = cache.cuda()
        with Q.scalar_division(mode):
            q = Q.nvfp4_kv_append_cuda(dev[:, qh:qh + heads], dev[:, qh + heads:], got, slots.cuda(), ko.cuda(), vo.cuda(), positions=pos.cuda() if rot else None,
                                       cos_sin=table.cuda() if rot else None, interleaved=interleaved, q=dev[:, :qh] if qh else None)
        want = append_ref(qkv, qh, heads, slots, pos, cache, ko, vo, table, interleaved, mode)
        assert torch.equal(got.cpu(), cache), "cache"
        assert (q is None) == (qh == 0) and (q is None or torch.equal(q.cpu(), want)), "queries"
    assert L.device_error() == 0


@gpu
def test_append_casts_as_the_nvfp4_recipe():
    """Unrotated rows get the codes and block scales that nvfp4_gs_cuda gives them under the same outer scale."""
    g = torch.Generator().manual_seed(7)
    x = (torch.randn(32, 4, 128, generator=g) * 3).to(torch.bfloat16).cuda()
    outer = Q.nvfp4_gs_scale_cuda(x.reshape(-1, 128))
    cache = Q.nvfp4_kv_cache_cuda(2, 4, 16, 128)
    Q.nvfp4_kv_append_cuda(x, x, cache, torch.arange(32, device="cuda"), outer.reshape(1), outer.reshape(1))
    codes, scales = planes(cache, 128)
    qd, sc = Q.nvfp4_gs_cuda(x.reshape(-1, 128), outer)
    for w in range(2):
        assert torch.equal(codes[:, :, w].transpose(1, 2).reshape(128, 64), qd.view(torch.uint8))
        assert torch.equal(scales[:, :, w].transpose(1, 2).reshape(128, 8), sc.view(torch.uint8))


@gpu
def test_append_bad_numbers_are_not_followed():
    D, page, heads = 64, 16, 2
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 2 * heads + 1, D, generator=g).to(torch.bfloat16)
    before = torch.randint(0, 256, (2, heads, 2, page * 36), generator=g, dtype=torch.uint8)
    ko = vo = torch.tensor([0.004])
    table = rotation_table(8, 32)
    L.device_error()
    for slots, pos, code, row in (([3, 32, 5, 6], [0, 1, 2, 3], 20, 1), ([3, 4, 5, 6], [0, 1, 8, 3], 21, 2), ([3, 4, 5, 6], [-1, 1, 2, 3], 21, 0),
                                  ([3, 1 << 40, 5, 6], [0, 1, 2, 3], 20, 1)):
        got = before.cuda()
        dev = x.cuda()
        q = Q.nvfp4_kv_append_cuda(dev[:, 1:1 + heads], dev[:, 1 + heads:], got, torch.tensor(slots).cuda(), ko.cuda(), vo.cuda(), positions=torch.tensor(pos).cuda(),
                                   cos_sin=table.cuda(), q=dev[:, :1])
        assert L.device_error() == code and L.device_error() == 0
        want = before.clone()
        keep = [i for i in range(4) if i != row]
        append_ref(x[keep], 1, heads, torch.tensor(slots)[keep], torch.tensor(pos)[keep], want, ko, vo, table, False)
        assert torch.equal(got.cpu(), want)
        assert (code == 21) == bool((q[row] == 0).all())


@gpu
def test_append_nan_and_inf():
    D = 64
    x = torch.ones(3, 1, D, dtype=torch.bfloat16)
    x[0, 0, 17] = float("nan")
    x[1, 0, 40] = float("inf")
    cache = torch.zeros(1, 1, 2, 16 * 36, dtype=torch.uint8, device="cuda")
    o = torch.tensor([0.001], device="cuda")
    Q.nvfp4_kv_append_cuda(x.cuda(), x.cuda(), cache, torch.arange(3, device="cuda"), o, o)
    for t in Q.nvfp4_kv_gather_cuda(cache, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda"), 3, D, o, o):
        t = t.cpu().view(3, 4, 16)
        assert bool(torch.isnan(t[0, 1]).all()) and bool(torch.isfinite(t[0, [0, 2, 3]]).all())
        assert float(t[1, 2].max()) == float(torch.tensor(6 * 448 * 0.001).to(torch.bfloat16)) and bool(torch.isfinite(t[1:]).all())


@gpu
@pytest.mark.parametrize("D,page,heads,lens,extra", [(128, 16, 8, [0, 5, 0, 33, 16, 1, 0], 3), (64, 32, 1, [100], 0), (128, 128, 3, [129, 1], 1), (64, 64, 2, [0, 0], 2)])
def test_gather_bits(D, page, heads, lens, extra):
    g = torch.Generator().manual_seed(page)
    table, pages = batch(g, lens, page)
    cache, ko, vo = random_cache(g, pages, heads, page, D)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    total = sum(lens) + extra
    k, v = Q.nvfp4_kv_gather_cuda(cache.cuda(), table.cuda(), cu.cuda(), total, D, ko.cuda(), vo.cuda())
    x = values(cache, D).float()
    want = torch.zeros(2, total, heads, D)
    for b, n in enumerate(lens):
        for i in range(n):
            want[:, cu[b] + i] = x[table[b, i // page].long(), :, :, i % page].transpose(0, 1)
    assert torch.equal(k.cpu(), (want[0] * ko).to(torch.bfloat16)) and torch.equal(v.cpu(), (want[1] * vo).to(torch.bfloat16))
    assert L.device_error() == 0


@gpu
def test_gather_bad_pages_read_as_zeros():
    g = torch.Generator().manual_seed(0)
    cache, ko, vo = random_cache(g, 3, 1, 16, 64)
    for table, n, good in (([[0, 3]], 20, 16), ([[-1, 1]], 32, None), ([[2]], 20, 16)):
        L.device_error()
        k, _ = Q.nvfp4_kv_gather_cuda(cache.cuda(), torch.tensor(table, dtype=torch.int32).cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), n, 64, ko.cuda(), vo.cuda())
        assert L.device_error() == 20
        k = k.cpu()
        assert bool((k[good:] == 0).all()) and bool((k[:good] != 0).any()) if good else bool((k[:16] == 0).all()) and bool((k[16:] != 0).any())


# ------------------------------------------------------------------------------------------------ attention
def attention_ref(q, cache, table, lens, q_lens, ko, vo, scale):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits, see the module's docstring."""
    D, heads = q.shape[2], cache.shape[1]
    page = cache.shape[3] * 16 // (9 * D)
    grp = q.shape[1] // heads
    x = values(cache, D)
    x = x.transpose(1, 3)          # pages, page, 2, heads, D
    outs, lses, tols, ltols = [], [], [], []
    at = 0
    for b, n in enumerate(lens):
        m = q_lens[b]
        pages = -(-n // page)
        kv = x[table[b, :pages].long()].flatten(0, 1)[:n]
        k, v = kv[:, 0] * ko.double(), kv[:, 1] * vo.double()
        qb = q[at:at + m].double().view(m, heads, grp, D)
        at += m
        s = torch.einsum("mhgd,nhd->mhgn", qb, k) * scale
        big = torch.einsum("mhgd,nhd->mhgn", qb.abs(), k.abs()) * scale
        hidden = torch.arange(n)[None, :] > n - m + torch.arange(m)[:, None]
        s = s.masked_fill(hidden.view(m, 1, 1, n), -math.inf)
        some = (~hidden).any(1) if n else torch.zeros(m, dtype=torch.bool)
        lse = torch.logsumexp(s, -1) if n else torch.full((m, heads, grp), -math.inf, dtype=torch.float64)
        p = torch.where(some.view(m, 1, 1, 1), torch.exp(s - lse.unsqueeze(-1)), 0.0).nan_to_num(0.0) if n else s
        o = torch.einsum("mhgn,nhd->mhgd", p, v)
        A = torch.einsum("mhgn,nhd->mhgd", p, v.abs())
        e = D * 2.0 ** -23 * (big.masked_fill(hidden.view(m, 1, 1, n), 0).amax(-1) if n else torch.zeros(m, heads, grp, dtype=torch.float64))
        e = e + 2.0 ** -23 * (s.abs().masked_fill(hidden.view(m, 1, 1, n), 0).amax(-1) if n else 0)
        tol = (2 * e.unsqueeze(-1) + 2.0 ** -11 + (n + 64) * 2.0 ** -23) * A + n * 2.0 ** -25 * (v.abs().amax() if n else 0) + 2.0 ** -8 * o.abs()
        outs.append(o.reshape(m, heads * grp, D)), tols.append(tol.reshape(m, heads * grp, D) * 1.01)
        lses.append(lse.reshape(m, heads * grp)), ltols.append((e + (n + 64) * 2.0 ** -23 + 2.0 ** -22 * lse.abs().nan_to_num(0, 0, 0)).reshape(m, heads * grp) * 1.01)
    return torch.cat(outs), torch.cat(lses), torch.cat(tols), torch.cat(ltols)


def attention_case(D, page, hq, heads, lens, q_lens, seed=0, q_scale=1.0, poison=True):
    g = torch.Generator().manual_seed(seed)
    table, pages = batch(g, lens, page)
    cache, ko, vo = random_cache(g, pages, heads, page, D)
    rows = sum(q_lens)
    q = (torch.randn(rows, hq, D, generator=g) * q_scale).to(torch.bfloat16)
    dirty = cache.clone()
    if poison:     # slots that no sequence owns hold NaN scales and arbitrary codes
        owned = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                owned[table[b, i].long(), :min(page, n - i * page)] = True
        codes, scales = planes(dirty, D)
        scales.copy_(torch.where(owned.view(pages, 1, 1, page, 1), scales, torch.tensor(0x7F, dtype=torch.uint8)))
        codes.copy_(torch.where(owned.view(pages, 1, 1, page, 1), codes, torch.tensor(0xAB, dtype=torch.uint8)))
    return q, cache, dirty, table, ko, vo


def call(q, cache, table, lens, q_lens, ko, vo, scale=None, fn=None, decode=False):
    kw = {} if decode else dict(cu_q=torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).cuda(), max_q=max(q_lens + [1]))
    return (fn or Q.nvfp4_kv_attention_cuda)(q.cuda(), cache.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ko.cuda(), vo.cuda(), scale=scale, **kw)


def check_attention(D, page, hq, heads, lens, q_lens=None, scale=None, **kw):
    decode = q_lens is None
    q_lens = q_lens or [1] * len(lens)
    q, cache, dirty, table, ko, vo = attention_case(D, page, hq, heads, lens, q_lens, **kw)
    out, lse = call(q, dirty, table, lens, q_lens, ko, vo, scale, decode=decode)
    o, z, tol, ltol = attention_ref(q, cache, table, lens, q_lens, ko, vo, 1 / math.sqrt(D) if scale is None else scale)
    assert L.device_error() == 0
    err = (out.cpu().double() - o).abs()
    assert bool((err <= tol).all()), f"out: {float((err - tol).max())} above the tolerance"
    dead = torch.isinf(z)
    assert torch.equal(torch.isinf(lse.cpu()) & (lse.cpu() < 0), dead) and bool((out.cpu()[dead] == 0).all())
    lerr = (lse.cpu().double() - z)[~dead].abs()
    assert bool((lerr <= ltol[~dead]).all()), f"lse: {float((lerr - ltol[~dead]).max())} above the tolerance"
    return out, lse


EDGE = [0, 1, 2, 15, 16, 17, 31, 33, 63, 65, 127, 128, 129, 255, 257, 1000]


@gpu
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("D,hq,heads", [(128, 32, 8), (128, 8, 8), (128, 5, 1), (64, 12, 4), (64, 16, 1), (128, 24, 2), (64, 32, 1), (128, 64, 1)])
def test_decode(D, hq, heads, page):
    check_attention(D, page, hq, heads, EDGE, seed=page + D)


@gpu
@pytest.mark.parametrize("lens", [[0], [1], [0, 0, 0], [7000], [3, 5000, 0, 1200]])
def test_decode_batches(lens):
    check_attention(128, 16, 32, 8, lens, seed=11)
    check_attention(64, 64, 8, 8, lens, seed=12)


@gpu
def test_decode_many_sequences():
    lens = [(i * 37) % 300 for i in range(700)]
    check_attention(64, 32, 4, 2, lens, seed=13)


@gpu
def test_most_sequences_a_call_takes():
    lens = [(i * 37) % 40 for i in range(4096)]
    check_attention(64, 16, 2, 1, lens, seed=14)
    check_attention(64, 16, 40, 1, lens, [(i * 5) % 3 for i in range(4096)], seed=15)


@gpu
@pytest.mark.parametrize("page,D,hq,heads", [(16, 128, 8, 2), (128, 64, 6, 6), (32, 128, 16, 1), (64, 64, 40, 8)])
@pytest.mark.parametrize("lens,q_lens", [([5, 130, 0, 64], [2, 4, 3, 1]), ([300, 17], [7, 17]), ([3], [9]), ([400, 1, 129], [130, 1, 66]), ([700], [257])])
def test_several_queries(page, D, hq, heads, lens, q_lens):
    """Chunks of prompts and drafted tokens; some sequences have more queries than keys, whose first queries see nothing."""
    check_attention(D, page, hq, heads, lens, q_lens, seed=sum(lens))


@gpu
def test_sequences_without_queries():
    check_attention(128, 16, 8, 2, [40, 50, 60, 70], [0, 3, 0, 2], seed=4)


@gpu
@pytest.mark.parametrize("q_scale,scale", [(30.0, None), (1e-30, None), (1.0, 0.5), (3e4, 1e-5), (0.0, None)])
def test_score_ranges(q_scale, scale):
    """Sharp and flat softmaxes, queries far from fp16's range."""
    check_attention(128, 32, 8, 2, [500, 129], q_scale=q_scale, scale=scale, seed=21)
    check_attention(128, 32, 8, 2, [500, 129], [5, 70], q_scale=q_scale, scale=scale, seed=22)


@gpu
def test_rising_scores_move_the_maximum():
    """Keys that score higher and higher: the running maximum moves in every tile."""
    D, page, n = 128, 16, 1024
    cache, ko, vo = random_cache(torch.Generator().manual_seed(5), n // page, 1, page, D)
    _, scales = planes(cache, D)
    codes, _ = planes(cache, D)
    codes[:, :, 0] = 0x22                                    # key = 1.0 * scale in every element
    step = torch.arange(n).view(n // page, 1, page, 1) * 64 // n + 16
    scales[:, :, 0] = step.to(torch.uint8).expand(-1, -1, -1, D // 16)
    q = torch.ones(1, 4, D, dtype=torch.bfloat16)
    table = torch.arange(n // page, dtype=torch.int32).view(1, -1)
    out, lse = call(q, cache, table, [n], [1], ko, vo, 1.0, decode=True)
    o, z, tol, ltol = attention_ref(q, cache, table, [n], [1], ko, vo, 1.0)
    assert bool(((out.cpu().double() - o).abs() <= tol).all()) and bool(((lse.cpu().double() - z).abs() <= ltol).all())


@gpu
def test_nan_stays_with_its_query():
    q, cache, _, table, ko, vo = attention_case(128, 16, 8, 2, [200, 300], [3, 3], poison=False)
    want, wl = call(q, cache, table, [200, 300], [3, 3], ko, vo)
    q[4, 3, 70] = float("nan")
    out, lse = call(q, cache, table, [200, 300], [3, 3], ko, vo)
    assert bool(torch.isnan(out[4, 3]).all()) and bool(torch.isnan(lse[4, 3]))
    out[4, 3], lse[4, 3] = want[4, 3], wl[4, 3]
    assert torch.equal(out, want) and torch.equal(lse, wl)


@gpu
@pytest.mark.parametrize("D,page,hq,heads", [(128, 16, 8, 2), (64, 64, 4, 4)])
@pytest.mark.parametrize("lens,q_lens", [([200, 300], [2, 2]), ([200, 300], [4, 3]), ([90, 129], [8, 7]), ([200, 300], [33, 40]), ([257, 300], [257, 150])])
def test_nan_in_the_cache_reaches_the_queries_that_see_it(D, page, hq, heads, lens, q_lens):
    """One value block (its scale is NaN) and, in another call, one key of a late token: earlier queries do not see it."""
    q, cache, _, table, ko, vo = attention_case(D, page, hq, heads, lens, q_lens, poison=False)
    o, z, tol, ltol = attention_ref(q, cache, table, lens, q_lens, ko, vo, 1 / math.sqrt(D))
    for b in range(2):
        for back in {1, q_lens[b] // 2, q_lens[b]}:
            t, head, block = lens[b] - max(back, 1), heads - 1, D // 16 - 2
            first = sum(q_lens[:b]) + max(t - (lens[b] - q_lens[b]), 0)        # the first row that sees token t
            rows, hs = slice(first, sum(q_lens[:b + 1])), slice(head * hq // heads, (head + 1) * hq // heads)
            for w in (1, 0):
                dirty = cache.clone()
                planes(dirty, D)[1][table[b, t // page].long(), head, w, t % page, block] = 0xFF if b else 0x7F
                out, lse = (x.cpu() for x in call(q, dirty, table, lens, q_lens, ko, vo))
                hit = torch.zeros(out.shape, dtype=torch.bool)
                hit[rows, hs, block * 16:block * 16 + 16 if w else D] = True
                if w == 0:
                    hit[rows, hs] = True
                assert torch.equal(torch.isnan(out), hit), (b, back, w)
                assert bool(((out.double() - o).abs() <= tol)[~hit].all())
                assert torch.equal(torch.isnan(lse), hit[..., 0] if w == 0 else torch.zeros_like(lse, dtype=torch.bool))
                assert bool(((lse.double() - z).abs() <= ltol)[~torch.isnan(lse)].all())


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,q_lens", [([5000] * 40, [1] * 40), ([5000] * 40, [2] * 40), ([5000] * 40, [3] * 40), ([700, 3000, 90], [300, 70, 90])])
def test_workspace_is_what_it_says(D, lens, q_lens):
    """Partial sums of every CTA stay within the bytes that the size query returns: what lies behind them is untouched."""
    import ctypes
    lib = L.load()
    hq, heads, page = 16, 2, 64
    q, cache, _, table, ko, vo = attention_case(D, page, hq, heads, lens, q_lens, poison=False)
    want = call(q, cache, table, lens, q_lens, ko, vo)
    q, cache, table, ko, vo = (x.cuda() for x in (q, cache, table, ko, vo))
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32).cuda()
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    size = lib.qcc_nvfp4_kv_attention_workspace_bytes(q.shape[0], len(lens), max(q_lens), hq, heads, D)
    ws = torch.full((size + (1 << 22),), 0xA5, dtype=torch.uint8, device="cuda")
    p = lambda t: t.data_ptr()
    a = L.KvAttentionArgs(p(q), (ctypes.c_int64 * 2)(*q.stride()[:2]), q.shape[0], p(cache), cache.shape[0], p(table), table.stride(0), table.shape[1], p(n), p(cu),
                          len(lens), max(q_lens), p(ko), p(vo), 1 / math.sqrt(D), hq, heads, D, page, p(out), p(lse))
    assert lib.qcc_nvfp4_kv_attention(ctypes.byref(a), p(ws), size - 1, torch.cuda.current_stream().cuda_stream) == -4
    assert lib.qcc_nvfp4_kv_attention(ctypes.byref(a), p(ws), size, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert bool((ws[size:] == 0xA5).all()) and bool((ws[:size] != 0xA5).any())


@gpu
def test_strided_queries_and_table():
    lens = [100, 333]
    q, cache, _, table, ko, vo = attention_case(128, 16, 8, 2, lens, [1, 1])
    want = call(q, cache, table, lens, [1, 1], ko, vo, decode=True)
    wide = torch.zeros(2, 12, 256, dtype=torch.bfloat16)
    wide[:, 2:10, 64:192] = q
    t = torch.full((2, table.shape[1] + 5), -7, dtype=torch.int32)
    t[:, :table.shape[1]] = table
    got = Q.nvfp4_kv_attention_cuda(wide.cuda()[:, 2:10, 64:192], cache.cuda(), t.cuda()[:, :table.shape[1]], torch.tensor(lens, dtype=torch.int32).cuda(), ko.cuda(), vo.cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_same_bits_every_time_and_on_any_stream():
    for lens, q_lens in (([4000, 17, 900], None), ([600, 300], [200, 300])):
        ql = q_lens or [1] * len(lens)
        q, cache, _, table, ko, vo = attention_case(128, 32, 32, 8, lens, ql)
        want = call(q, cache, table, lens, ql, ko, vo, decode=q_lens is None)
        side = [torch.cuda.Stream() for _ in range(2)]
        for s in side:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(5):
            got = []
            for s in side:
                with torch.cuda.stream(s):
                    got.append(call(q, cache, table, lens, ql, ko, vo, decode=q_lens is None))
            torch.cuda.synchronize()
            for o, z in got:
                assert torch.equal(o, want[0]) and torch.equal(z, want[1])


@gpu
def test_graph_follows_lengths_and_table_on_the_device():
    """A captured decode step, padded to four sequences, is replayed as the sequences grow and leave."""
    D, page, hq, heads = 128, 16, 8, 2
    g = torch.Generator().manual_seed(8)
    full = [300, 41, 0, 160]
    q, cache, _, table, ko, vo = attention_case(D, page, hq, heads, full, [1] * 4, poison=False)
    dev = [t.cuda() for t in (q, cache, table, torch.tensor(full, dtype=torch.int32), ko, vo)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = Q.nvfp4_kv_attention_cuda(*dev)
        out2, lse2 = Q.nvfp4_kv_attention_cuda(*dev)
    for lens in ([300, 41, 0, 160], [1, 0, 0, 129], [0, 0, 0, 0], [299, 40, 0, 7]):
        dev[3].copy_(torch.tensor(lens, dtype=torch.int32))
        dev[0].copy_(torch.randn(4, hq, D, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        want = Q.nvfp4_kv_attention_cuda(*dev)
        for a, b in ((out, want[0]), (out2, want[0]), (lse, want[1]), (lse2, want[1])):
            assert torch.equal(a, b), lens


@gpu
def test_graph_follows_query_offsets_on_the_device():
    """A captured call for up to 300 rows of new tokens, replayed as they belong to other sequences; two share the pool of one graph."""
    D, page, hq, heads = 64, 32, 12, 4
    g = torch.Generator().manual_seed(9)
    q, cache, _, table, ko, vo = attention_case(D, page, hq, heads, [500, 140, 300], [300, 0, 0], poison=False)
    lens, cu = torch.tensor([500, 140, 300], dtype=torch.int32).cuda(), torch.tensor([0, 300, 300, 300], dtype=torch.int32).cuda()
    dev = [t.cuda() for t in (q, cache, table)] + [lens, ko.cuda(), vo.cuda()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = Q.nvfp4_kv_attention_cuda(*dev, cu_q=cu, max_q=300)
        again = Q.nvfp4_kv_attention_cuda(*dev, cu_q=cu, max_q=300)
    for n, offsets in (([500, 140, 300], [0, 300, 300, 300]), ([500, 140, 300], [0, 0, 140, 300]), ([0, 0, 0], [0, 0, 0, 0]), ([90, 0, 7], [0, 100, 130, 137]), ([1, 140, 300], [0, 1, 2, 300])):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        dev[0].copy_(torch.randn(300, hq, D, generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        want = Q.nvfp4_kv_attention_cuda(*dev, cu_q=cu, max_q=300)
        for a, b in zip(first + again, want + want):
            assert torch.equal(a, b), offsets
        o, z, tol, ltol = attention_ref(dev[0].cpu()[:offsets[-1]], cache, table, n, [b - a for a, b in zip(offsets, offsets[1:])], ko, vo, 1 / math.sqrt(D))
        assert bool(((want[0][:offsets[-1]].cpu().double() - o).abs() <= tol).all())
        assert bool((want[0][offsets[-1]:] == 0).all()) and bool((want[1][offsets[-1]:] == -math.inf).all())


@gpu
def test_many_queries_with_bad_numbers():
    """The form for many queries: a bad page, offsets and lengths outside their ranges are reported, and the other sequence is right."""
    D, page, hq, heads, lens, ql = 64, 16, 4, 2, [100, 130], [60, 70]
    q, cache, _, table, ko, vo = attention_case(D, page, hq, heads, lens, ql, poison=False)
    L.device_error()
    want = call(q, cache, table, lens, ql, ko, vo)
    assert L.device_error() == 0
    for n in (cache.shape[0], -1, 1 << 30):
        bad = table.clone()
        bad[0, 3] = n
        out, lse = call(q, cache, bad, lens, ql, ko, vo)
        assert L.device_error() == 20
        assert torch.equal(out[60:], want[0][60:]) and torch.equal(lse[60:], want[1][60:])
    call(q, cache, table, [100, 16 * table.shape[1] + 1], ql, ko, vo)
    assert L.device_error() == 20
    args = (q.cuda(), cache.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ko.cuda(), vo.cuda())
    for cu, mq in (([0, 60, 131], 70), ([0, 60, 50], 70), ([-1, 60, 130], 70), ([0, 60, 130], 69), ([0, 2 ** 31 - 1, -2 ** 31], 70)):
        Q.nvfp4_kv_attention_cuda(*args, cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), max_q=mq)
        assert L.device_error() == 22, cu
    out, lse = call(q, cache, table, lens, ql, ko, vo)
    assert L.device_error() == 0 and torch.equal(out, want[0]) and torch.equal(lse, want[1])


@gpu
def test_rows_behind_the_last_sequence():
    lens, q_lens = [100, 30], [3, 2]
    q, cache, _, table, ko, vo = attention_case(64, 16, 4, 2, lens, q_lens)
    want = call(q, cache, table, lens, q_lens, ko, vo)
    more = torch.cat([q, torch.full((77, 4, 64), float("nan"), dtype=torch.bfloat16)])
    out, lse = call(more, cache, table, lens, q_lens, ko, vo)
    assert torch.equal(out[:5], want[0]) and torch.equal(lse[:5], want[1])
    assert bool((out[5:] == 0).all()) and bool((lse[5:] == -math.inf).all())


@gpu
def test_bad_numbers_set_the_error_word():
    lens = [100, 30]
    q, cache, _, table, ko, vo = attention_case(64, 16, 4, 2, lens, [1, 1], poison=False)
    L.device_error()
    want = call(q, cache, table, lens, [1, 1], ko, vo, decode=True)
    bad = table.clone()
    bad[0, 2] = cache.shape[0]
    out, lse = call(q, cache, bad, lens, [1, 1], ko, vo, decode=True)
    assert L.device_error() == 20
    assert torch.equal(out[1], want[0][1]) and torch.equal(lse[1], want[1][1])
    call(q, cache, table, [100, 16 * table.shape[1] + 1], [1, 1], ko, vo, decode=True)      # longer than its row of the table
    assert L.device_error() == 20
    args = (q.cuda(), cache.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ko.cuda(), vo.cuda())
    for cu, mq in (([0, 1, 5], 2), ([0, 2, 1], 2), ([-1, 1, 2], 2), ([0, 0, 2], 1)):
        Q.nvfp4_kv_attention_cuda(*args, cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), max_q=mq)
        assert L.device_error() == 22, cu
    out, _ = call(q, cache, table, lens, [1, 1], ko, vo, decode=True)
    assert L.device_error() == 0 and torch.equal(out, want[0])


@gpu
def test_cache_beyond_4_gib():
    """Page offsets that pass 32 bits."""
    D, page, heads = 128, 16, 8
    pages = (1 << 32) // (heads * 2 * page * 72) + 9
    cache = torch.empty(pages, heads, 2, page * 72, dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, 2 * heads, D, generator=g).to(torch.bfloat16)
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32)
    at = torch.arange(40)
    slots = table[0, at // page].long() * page + at % page
    o = torch.tensor([0.003])
    dev = x.cuda()
    Q.nvfp4_kv_append_cuda(dev[:, :heads], dev[:, heads:], cache, slots.cuda(), o.cuda(), o.cuda())
    small = cache[table[0].long().cuda()].contiguous()
    t = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    q = torch.randn(1, 32, D, generator=g).to(torch.bfloat16)
    got = call(q, cache, table, [40], [1], o, o, decode=True)
    want = call(q, small, t, [40], [1], o, o, decode=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    cu = torch.tensor([0, 40], dtype=torch.int32).cuda()
    for a, b in zip(Q.nvfp4_kv_gather_cuda(cache, table.cuda(), cu, 40, D, o.cuda(), o.cuda()), Q.nvfp4_kv_gather_cuda(small, t.cuda(), cu, 40, D, o.cuda(), o.cuda())):
        assert torch.equal(a, b) and bool((a != 0).any())
    chunk = torch.randn(20, 32, D, generator=g).to(torch.bfloat16)
    for a, b in zip(call(chunk, cache, table, [40], [20], o, o), call(chunk, small, t, [40], [20], o, o)):
        assert torch.equal(a, b)
    ref = attention_ref(q, small.cpu(), t, [40], [1], o, o, 1 / math.sqrt(D))
    assert bool(((got[0].cpu().double() - ref[0]).abs() <= ref[2]).all())


@gpu
def test_refusals():
    q, cache, _, table, ko, vo = [t.cuda() for t in attention_case(64, 16, 4, 2, [100, 30], [1, 1])]
    lens = torch.tensor([100, 30], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    for bad in (lambda: Q.nvfp4_kv_attention_cuda(q[:1], cache, table, lens, ko, vo), lambda: Q.nvfp4_kv_attention_cuda(q, cache, table.long(), lens, ko, vo),
                lambda: Q.nvfp4_kv_attention_cuda(q, cache, table, lens[:1], ko, vo), lambda: Q.nvfp4_kv_attention_cuda(q.float(), cache, table, lens, ko, vo),
                lambda: Q.nvfp4_kv_attention_cuda(q, cache, table, lens, ko, vo, cu_q=cu), lambda: Q.nvfp4_kv_attention_cuda(q[:, :3], cache, table, lens, ko, vo),
                lambda: Q.nvfp4_kv_attention_cuda(q, cache[..., :100], table, lens, ko, vo), lambda: Q.nvfp4_kv_attention_cuda(q, cache, table, lens, ko.cpu(), vo),
                lambda: Q.nvfp4_kv_attention_cuda(q, cache, table, lens, ko, vo, scale=0.0), lambda: Q.nvfp4_kv_attention_cuda(q[:, :, :32], cache, table, lens, ko, vo),
                lambda: Q.nvfp4_kv_append_cuda(q, q, cache, torch.zeros(2, dtype=torch.int64).cuda(), ko, vo),
                lambda: Q.nvfp4_kv_append_cuda(q[:, :2], q[:, :2], cache, torch.zeros(2, dtype=torch.int32).cuda(), ko, vo),
                lambda: Q.nvfp4_kv_append_cuda(q[:, :2], q[:, :2], cache, torch.zeros(2, dtype=torch.int64).cuda(), ko, vo, cos_sin=torch.zeros(4, 48).cuda(), positions=torch.zeros(2, dtype=torch.int64).cuda()),
                lambda: Q.nvfp4_kv_append_cuda(q[:, :2], q[:, :2], cache, torch.zeros(2, dtype=torch.int64).cuda(), ko, vo, cos_sin=torch.zeros(4, 32).cuda())):
        with pytest.raises((AssertionError, ValueError)):
            bad()


@gpu
def test_empty_calls():
    q, cache, _, table, ko, vo = [t.cuda() for t in attention_case(64, 16, 4, 2, [100, 30], [1, 1])]
    none = torch.zeros(0, dtype=torch.int32).cuda()
    out, lse = Q.nvfp4_kv_attention_cuda(q[:0], cache, table[:0], none, ko, vo)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = Q.nvfp4_kv_attention_cuda(q, cache, table[:0], none, ko, vo, cu_q=torch.zeros(1, dtype=torch.int32).cuda(), max_q=1)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    before = cache.clone()
    assert Q.nvfp4_kv_append_cuda(q[:0, :2], q[:0, :2], cache, torch.zeros(0, dtype=torch.int64).cuda(), ko, vo, q=q[:0]).shape == (0, 4, 64)
    assert torch.equal(cache, before)
    k, v = Q.nvfp4_kv_gather_cuda(cache, table, torch.zeros(3, dtype=torch.int32).cuda(), 0, 64, ko, vo)
    assert k.shape == v.shape == (0, 2, 64)


@gpu
def test_native_operators_give_the_same_bits():
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops as N
    D, page, heads, qh = 128, 16, 2, 8
    qkv, slots, pos, cache, ko, vo, table = append_inputs(D, page, heads, qh, 64, 50, seed=1)
    dev, caches, outs = qkv.cuda(), [], []
    for fn in (Q.nvfp4_kv_append_cuda, N.nvfp4_kv_append_native):
        c = cache.cuda()
        outs.append(fn(dev[:, qh:qh + heads], dev[:, qh + heads:], c, slots.cuda(), ko.cuda(), vo.cuda(), positions=pos.cuda(), cos_sin=table.cuda(), interleaved=True, q=dev[:, :qh]))
        caches.append(c)
    assert torch.equal(*outs) and torch.equal(*caches)
    lens, q_lens = [100, 30], [3, 2]
    q, cache, _, table, ko, vo = attention_case(64, 16, 4, 2, lens, q_lens)
    for decode in (False, True):
        rows = q[:2] if decode else q
        a = call(rows, cache, table, lens, q_lens, ko, vo, decode=decode)
        b = call(rows, cache, table, lens, q_lens, ko, vo, decode=decode, fn=N.nvfp4_kv_attention_native)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    args = (cache.cuda(), table.cuda(), torch.tensor([0, 100, 130], dtype=torch.int32).cuda(), 130, 64, ko.cuda(), vo.cuda())
    for a, b in zip(Q.nvfp4_kv_gather_cuda(*args), N.nvfp4_kv_gather_native(*args)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        N.nvfp4_kv_attention_native(q.cuda(), cache.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), ko.cuda(), vo.cuda())


@gpu
def test_a_decoder_step():
    """The operators as a server chains them: int8 projection, append with rotation, attention over the cache, int8 projection.
    Each stage is held to its own definition in 64 bits on the stage's actual inputs; a prompt first, then two single tokens."""
    D, page, heads, qh, hidden = 128, 16, 2, 8, 512
    g = torch.Generator().manual_seed(0)
    wqkv, ws = Q.rowwise_int8_cuda((torch.randn((qh + 2 * heads) * D, hidden, generator=g) / math.sqrt(hidden)).to(torch.bfloat16).cuda())
    wo, wos = Q.rowwise_int8_cuda((torch.randn(hidden, qh * D, generator=g) / math.sqrt(qh * D)).to(torch.bfloat16).cuda())
    rope = rotation_table(200, D)
    cache = Q.nvfp4_kv_cache_cuda(12, heads, page, D)
    ko, vo = torch.tensor([6.0 / 2688]).cuda(), torch.tensor([5.0 / 2688]).cuda()
    table = torch.randperm(12, generator=g).to(torch.int32).view(2, 6)
    lens = [0, 0]
    for new in ([70, 33], [1, 1], [1, 1]):
        x = torch.randn(sum(new), hidden, generator=g).to(torch.bfloat16)
        pos = torch.cat([torch.arange(lens[b], lens[b] + new[b]) for b in range(2)])
        seq = torch.repeat_interleave(torch.arange(2), torch.tensor(new))
        slots = table[seq, pos // page].long() * page + pos % page
        lens = [lens[b] + new[b] for b in range(2)]
        xq, xs = Q.rowwise_int8_cuda(x.cuda())
        qkv = Q.int8_scaled_mm_cuda(xq, wqkv, xs, ws).view(-1, qh + 2 * heads, D)
        before = cache.cpu()
        q = Q.nvfp4_kv_append_cuda(qkv[:, qh:qh + heads], qkv[:, qh + heads:], cache, slots.cuda(), ko, vo, positions=pos.cuda(), cos_sin=rope.cuda(), q=qkv[:, :qh])
        want_q = append_ref(qkv.cpu(), qh, heads, slots, pos, before, ko.cpu(), vo.cpu(), rope, False)
        assert torch.equal(q.cpu(), want_q)
        written = [slots // page, slots % page]
        for a, b in zip(planes(cache.cpu(), D), planes(before, D)):
            assert torch.equal(a[written[0], :, :, written[1]], b[written[0], :, :, written[1]])
        out, lse = call(q, cache, table, lens, new, ko, vo, decode=max(new) == 1)
        o, z, tol, ltol = attention_ref(q.cpu(), cache.cpu(), table, lens, new, ko.cpu(), vo.cpu(), 1 / math.sqrt(D))
        assert bool(((out.cpu().double() - o).abs() <= tol).all()) and bool(((lse.cpu().double() - z).abs() <= ltol).all())
        oq, os_ = Q.rowwise_int8_cuda(out.view(-1, qh * D))
        y = Q.int8_scaled_mm_cuda(oq, wo, os_, wos, out_dtype=torch.float32)
        want = (oq.cpu().double() @ wo.cpu().double().T) * os_.cpu().double() * wos.cpu().double().T
        assert bool(((y.cpu().double() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs() + want.abs() * 2.0 ** -24).all())
    assert L.device_error() == 0


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hq,q_len", [(4, 1), (16, 1), (32, 1), (8, 10), (8, 40)])      # each form of the kernels
@pytest.mark.parametrize("every,ratio", [(32, 1.5 * 2.0 ** -24), (32, 1.3 * 2.0 ** -26), (32, 2.0 ** -19), (4096, 1.5 * 2.0 ** -24)])
def test_a_flat_tail_keeps_its_weight_beside_dominant_keys(D, hq, q_len, every, ratio):
    """Dominant keys, `every` tokens apart, whose values are zero, over a tail of keys of one score whose values are one: the output is the
    tail's share.  All keys of the tail are rounded alike, so nothing averages out.  A probability is rounded by half a step of fp16, 2^-11, or
    below fp16's normal numbers by half of 2^-24 where a dominant one is at least 2^7: 2^-32 of it.  Scores: see the module's docstring."""
    n, page = 4096, 64
    table = torch.randperm(n // page, generator=torch.Generator().manual_seed(D)).to(torch.int32).view(1, -1)
    cache = torch.zeros(n // page, 1, 2, page * 9 * D // 16, dtype=torch.uint8)
    codes, scales = planes(cache, D)
    scales.fill_(0x38)                                        # 1.0
    at = torch.arange(n)
    loud = at % every == 0
    codes[table[0, at // page].long(), 0, 0, at % page] = (loud * 0x22).to(torch.uint8).view(-1, 1).expand(-1, D // 2)
    codes[table[0, at // page].long(), 0, 1, at % page] = (~loud * 0x22).to(torch.uint8).view(-1, 1).expand(-1, D // 2)
    scale = float(torch.tensor(-math.log(ratio) / D))
    q, one = torch.ones(q_len, hq, D, dtype=torch.bfloat16), torch.ones(1)
    out, lse = call(q, cache, table, [n], [q_len], one, one, scale, decode=q_len == 1)
    o, z, _, ltol = attention_ref(q, cache, table, [n], [q_len], one, one, scale)
    e = (D + 2) * 2.0 ** -23 * scale * D
    tol = (2 * e + 2.0 ** -11 + (n + 64) * 2.0 ** -23 + 2.0 ** -8) * o + every * 2.0 ** -32
    err = (out.cpu().double() - o).abs()
    assert bool((err <= tol * 1.01).all()), f"off by {float((err / o).max())} of the tail, {float((tol / o).max())} allowed"
    assert bool(((lse.cpu().double() - z).abs() <= ltol).all()) and L.device_error() == 0


@pytest.mark.parametrize("name", ["int8.cu", "kv_cache.cuh", "kv_cache.cu", "kv_attention.cuh", "kv_attention.cu", "kv_prompt.cu"])
def test_overlapped_kernels_load_by_the_coherent_path(name):
    """These kernels start under their predecessor, which may still write what they read: no load that takes its data for constant."""
    import os
    import re
    with open(os.path.join(os.path.dirname(L.LIB_PATH), "..", "csrc", name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(r"__ldg\b|ld_nc_v4|\.nc\b|__restrict__", text)


@gpu
@pytest.mark.parametrize("captured", [False, True])
def test_steps_in_a_row_read_what_the_last_one_wrote(captured):
    """A projection into one buffer, an append to the same slots, a read-back and an attention, twelve times without a synchronisation
    between: each step sees the keys and values of its own."""
    D, page, heads, qh, tokens, steps = 128, 16, 2, 8, 48, 12
    g = torch.Generator().manual_seed(6)
    w, ws = Q.rowwise_int8_cuda(torch.randn((qh + 2 * heads) * D, 256, generator=g).to(torch.bfloat16).cuda())
    x = torch.randn(steps, tokens, 256, generator=g).to(torch.bfloat16).cuda()
    rope, slots, pos = rotation_table(tokens, D).cuda(), torch.randperm(tokens, generator=g).cuda(), torch.arange(tokens).cuda()
    one = torch.tensor([0.02]).cuda()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
    cu, n = torch.tensor([0, tokens], dtype=torch.int32).cuda(), torch.tensor([tokens], dtype=torch.int32).cuda()

    def run(cache, synchronise):
        got = []
        for i in range(steps):
            calls = []
            for call in range(5):
                if call == 0:
                    calls.append(Q.rowwise_int8_cuda(x[i]))
                elif call == 1:
                    calls.append(Q.int8_scaled_mm_cuda(calls[0][0], w, calls[0][1], ws).view(tokens, qh + 2 * heads, D))
                elif call == 2:
                    q, k, v = calls[1].split([qh, heads, heads], 1)
                    calls.append(Q.nvfp4_kv_append_cuda(k, v, cache, slots, one, one, positions=pos, cos_sin=rope, q=q))
                elif call == 3:
                    calls.append(Q.nvfp4_kv_gather_cuda(cache, table, cu, tokens, D, one, one))
                else:
                    calls.append(Q.nvfp4_kv_attention_cuda(calls[2], cache, table, n, one, one, cu_q=cu, max_q=tokens) if i % 2 else
                                 Q.nvfp4_kv_attention_cuda(calls[2][-1:], cache, table, n, one, one))
                if synchronise:
                    torch.cuda.synchronize()
            got += [calls[2], *calls[3], *calls[4]]
        return got
    want = run(torch.zeros(3, heads, 2, page * 72, dtype=torch.uint8, device="cuda"), True)
    cache = torch.zeros(3, heads, 2, page * 72, dtype=torch.uint8, device="cuda")
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(cache, False)
        graph.replay()
        graph.replay()
    else:
        got = run(cache, False)
    torch.cuda.synchronize()
    assert not any(torch.equal(a, b) for a, b in zip(got[:-5], got[5:]))        # the steps do differ
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert L.device_error() == 0


@pytest.mark.parametrize("device", ["meta", pytest.param("cuda", marks=gpu)])
def test_the_registered_operator_refuses_a_scale_that_is_not_positive(device):
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops  # noqa: F401  (loads the operators)
    op = torch.ops.quant_cast_cuda_native.nvfp4_kv_attention

    def zeros(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device=device)
    o = zeros(1, dtype=torch.float32) + 1
    args = (zeros(1, 4, 64), zeros(1, 2, 2, 16 * 36, dtype=torch.uint8), zeros(1, 1, dtype=torch.int32), zeros(1, dtype=torch.int32) + 3, o, o)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(RuntimeError, match="scale must be positive"):
            op(*args, scale=scale)
    assert all(a.shape == b.shape for a, b in zip(op(*args), op(*args, scale=0.125)))
    if device == "cuda":
        assert all(torch.equal(a, b) for a, b in zip(op(*args), op(*args, scale=0.125)))


@gpu
@pytest.mark.parametrize("lens,q_lens,hq", [([100, 30], None, 4), ([300] * 300, None, 4), ([5000, 20], None, 4), ([5000, 20], [8, 3], 4), ([200, 90], [70, 4], 4), ([200], None, 80)])
def test_launch_count_is_what_a_call_launches(lens, q_lens, hq):
    """The binding's counter against the kernels of the captured call: units dealt out whole, joined, many queries."""
    import ctypes
    ql = q_lens or [1] * len(lens)
    q, cache, _, table, ko, vo = (t.cuda() for t in attention_case(64, 16, hq, 2, lens, ql, poison=False))
    kw = {} if q_lens is None else dict(cu_q=torch.tensor([0] + ql).cumsum(0).to(torch.int32).cuda(), max_q=max(ql))
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    before = L.launch_count
    with torch.cuda.graph(graph):
        Q.nvfp4_kv_attention_cuda(q, cache, table, n, ko, vo, **kw)
    count = ctypes.c_size_t(0)
    assert ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(count)) == 0
    assert L.launch_count - before == count.value


@gpu
def test_overlapping_offsets_that_claim_more_rows_than_31_bits_number():
    """Every second sequence claims all rows of q, the others' offsets descend: 2048 times 2^20 and one blocks of 256 rows, which a 32-bit sum cannot
    hold.  The offsets are reported; all sequences are empty, so every row is zero."""
    rows, hq, D, seqs = (1 << 22) + 4, 64, 64, 4096
    assert seqs // 2 * -(-rows * hq // 256) > 1 << 31
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("36 GB of results")
    q = torch.zeros(1, 1, D, dtype=torch.bfloat16, device="cuda").expand(rows, hq, D)
    cache, one = Q.nvfp4_kv_cache_cuda(1, 1, 16, D), torch.ones(1, device="cuda")
    cu = (torch.arange(seqs + 1, device="cuda") % 2 * rows).to(torch.int32)
    L.device_error()
    out, lse = Q.nvfp4_kv_attention_cuda(q, cache, torch.zeros(seqs, 1, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                                         one, one, cu_q=cu, max_q=rows)
    assert L.device_error() == 22
    assert out.view(torch.int16).amax() == 0 and out.view(torch.int16).amin() == 0 and lse.amax() == -math.inf
    del out, lse
    torch.cuda.empty_cache()


@gpu
def test_max_q_may_be_any_bound():
    """max_q is at least the most queries of a sequence: numbers that a C int does not hold among them."""
    import sys
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops as N
    lens, q_lens = [100, 30], [30, 20]
    q, cache, _, table, ko, vo = (t.cuda() for t in attention_case(64, 16, 4, 2, lens, q_lens, poison=False))
    args = (q, cache, table, torch.tensor(lens, dtype=torch.int32).cuda(), ko, vo)
    cu = torch.tensor([0, 30, 50], dtype=torch.int32).cuda()
    want = Q.nvfp4_kv_attention_cuda(*args, cu_q=cu, max_q=30)
    for fn in (Q.nvfp4_kv_attention_cuda, N.nvfp4_kv_attention_native):
        for max_q in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 1, sys.maxsize):
            out, lse = fn(*args, cu_q=cu, max_q=max_q)
            assert L.device_error() == 0 and torch.equal(out, want[0]) and torch.equal(lse, want[1]), (fn, max_q)
    for max_q in (0, -5):
        with pytest.raises((AssertionError, RuntimeError)):
            Q.nvfp4_kv_attention_cuda(*args, cu_q=cu, max_q=max_q)
        with pytest.raises((AssertionError, RuntimeError)):
            N.nvfp4_kv_attention_native(*args, cu_q=cu, max_q=max_q)


@gpu
def test_empty_batches_and_caches():
    """A batch without sequences, and a cache without pages: tensors that have no address.  Rows without tokens are zeros, a slot is reported."""
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops as N
    D, one = 64, torch.ones(1, device="cuda")

    def ints(*v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")
    none, page = Q.nvfp4_kv_cache_cuda(0, 2, 16, D), Q.nvfp4_kv_cache_cuda(1, 2, 16, D)
    x = torch.ones(3, 2, D, dtype=torch.bfloat16, device="cuda")
    L.device_error()
    for gather, attention, append in ((Q.nvfp4_kv_gather_cuda, Q.nvfp4_kv_attention_cuda, Q.nvfp4_kv_append_cuda),
                                      (N.nvfp4_kv_gather_native, N.nvfp4_kv_attention_native, N.nvfp4_kv_append_native)):
        for cache in (none, page):
            empty = torch.empty(0, 4, dtype=torch.int32, device="cuda")
            for t in gather(cache, empty, ints(0), 5, D, one, one) + gather(cache, torch.empty(2, 0, dtype=torch.int32, device="cuda"), ints(0, 0, 0), 5, D, one, one):
                assert t.shape == (5, 2, D) and not t.any()
            for kw, lens in ((dict(), ints(0, 0, 0)), (dict(cu_q=ints(0, 2, 2), max_q=2), ints(0, 0)), (dict(cu_q=ints(0, 3), max_q=40), ints(0))):
                for width in (0, 2):
                    out, lse = attention(x, cache, torch.zeros(lens.shape[0], width, dtype=torch.int32, device="cuda"), lens, one, one, **kw)
                    assert not out.any() and bool((lse == -math.inf).all())
            assert append(x, x, cache, torch.full((3,), -1, device="cuda"), one, one, q=x).equal(x)
        assert L.device_error() == 0
        append(x, x, none, torch.tensor([-1, 0, -1], device="cuda"), one, one)
        assert L.device_error() == 20
        gather(none, ints(0).view(1, 1), ints(0, 3), 3, D, one, one)
        assert L.device_error() == 20
        attention(x[:1], none, ints(0).view(1, 1), ints(3), one, one)
        assert L.device_error() == 20
        attention(x, none, ints(0).view(1, 1), ints(3), one, one, cu_q=ints(0, 3), max_q=40)
        assert L.device_error() == 20


def test_c_takes_no_cache_without_pages():
    lib, p = L.load(), 1 << 20
    assert lib.qcc_nvfp4_kv_gather(None, 4, 2, 16, 64, p, 4, 4, p, 1, 4, p, p, p, p, None) == -3
    assert lib.qcc_nvfp4_kv_gather(p, 4, 2, 16, 64, None, 4, 4, p, 1, 4, p, p, p, p, None) == -3


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hq,q_len,longest", [(16, 1, 1000), (48, 1, 900), (8, 7, 1000), (80, 1, 500), (16, 8, 400)])      # 4, 12, 14, 20 and 32 rows
def test_many_short_units_are_dealt_out_whole(D, hq, q_len, longest):
    """Several whole units a CTA, one after the other; q of each in turn, where it is kept in shared memory, and idle slots between."""
    g = torch.Generator().manual_seed(hq)
    lens = [longest] + [0 if i % 16 == 3 else int(n) for i, n in enumerate(torch.randint(1, longest + 1, (169,), generator=g))]
    q_lens = None if q_len == 1 else [q_len if i % 3 else int(i % q_len) for i in range(170)]
    before = L.launch_count
    check_attention(D, 32, hq, 4, lens, q_lens, seed=hq + D)
    assert L.launch_count - before == 1


@gpu
def test_the_operators_trace_under_torch_compile():
    """A decoder step in one graph: the append writes the cache, an argument, and the reads behind it see that."""
    from quant_cast_bench_b200 import build as qbuild
    qbuild.build_torch_binding()
    from quant_cast_bench_b200.quant_cast_cuda import native_ops as N
    D, page, heads, qh, tokens = 64, 16, 2, 8, 20
    g = torch.Generator().manual_seed(3)
    w, ws = Q.rowwise_int8_cuda(torch.randn((qh + 2 * heads) * D, 256, generator=g).to(torch.bfloat16).cuda())
    x = torch.randn(tokens, 256, generator=g).to(torch.bfloat16).cuda()
    rope, slots, pos = rotation_table(tokens, D).cuda(), torch.arange(tokens).cuda(), torch.arange(tokens).cuda()
    one, table = torch.tensor([0.02]).cuda(), torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    cu, n = torch.tensor([0, tokens], dtype=torch.int32).cuda(), torch.tensor([tokens], dtype=torch.int32).cuda()

    def step(x, cache):
        a, s = N.rowwise_int8_native(x * 2.0)
        q, k, v = N.int8_scaled_mm_native(a, w, s, ws).view(tokens, qh + 2 * heads, D).split([qh, heads, heads], 1)
        q = N.nvfp4_kv_append_native(k, v, cache, slots, one, one, positions=pos, cos_sin=rope, q=q)
        kb, vb = N.nvfp4_kv_gather_native(cache, table, cu, tokens, D, one, one)
        out, lse = N.nvfp4_kv_attention_native(q, cache, table, n, one, one, cu_q=cu, max_q=tokens)
        last, last_lse = N.nvfp4_kv_attention_native(q[-1:], cache, table, n, one, one, scale=0.1)
        return q, kb, vb, out * 1.0, lse, last, last_lse

    caches = [torch.zeros(2, heads, 2, page * 36, dtype=torch.uint8, device="cuda") for _ in range(2)]
    slots = (table[0].long()[slots // page] * page + slots % page).contiguous()
    want = step(x, caches[0])
    got = torch.compile(step, fullgraph=True)(x, caches[1])
    assert torch.equal(*caches) and bool(caches[0].any())
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b)
    for op, args in ((N.ops.nvfp4_kv_append, (want[1], want[2], caches[0], slots, one, one)), (N.ops.int8_rowwise, (x,)),
                     (N.ops.int8_scaled_mm, (*N.rowwise_int8_native(x)[:1], w, N.rowwise_int8_native(x)[1], ws)),
                     (N.ops.nvfp4_kv_gather, (caches[0], table, cu, tokens, D, one, one)), (N.ops.nvfp4_kv_attention, (want[0][-1:], caches[0], table, n, one, one))):
        torch.library.opcheck(op.default, args, test_utils=("test_schema", "test_faketensor"))


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hq,q_len", [(4, 1), (16, 1), (32, 1), (8, 10), (8, 40)])      # each form of the kernels
def test_scores_that_leave_no_bits_for_a_difference(D, hq, q_len):
    """Keys of one score, up to 2^29 in log2 units, where fp32 numbers are 32 apart: each has the same weight all the same."""
    n, page = 200, 64
    cache = torch.zeros(4, 1, 2, page * 9 * D // 16, dtype=torch.uint8)
    codes, scales = planes(cache, D)
    scales.fill_(0x38)                                        # 1.0
    codes.fill_(0x22)                                         # 1.0 in every element of keys and values, but 37 twos in a key:
    codes[:, :, 0, :, :18], codes[:, :, 0, :, 18] = 0x44, 0x24      # a product of score and factor has more than 24 bits
    dot = D + 37
    table, one, q = torch.arange(4, dtype=torch.int32).view(1, 4), torch.ones(1), torch.ones(q_len, hq, D, dtype=torch.bfloat16)
    for log2 in [1.0, 1e3, 1e6] + [2.0 ** 27 * x for x in (1.1, 1.37, 1.73)] + [2.0 ** 28 * x for x in (1.03, 1.13, 1.27, 1.37, 1.49, 1.6, 1.72, 1.83, 1.91, 1.97)]:
        scale = float(torch.tensor(log2 * math.log(2) / dot))
        out, lse = call(q, cache, table, [n], [q_len], one, one, scale, decode=q_len == 1)
        assert bool(((out.cpu().double() - 1).abs() <= 2.0 ** -8 + 2.0 ** -11).all()), log2
        want = scale * dot + torch.log(torch.arange(n - q_len + 1, n + 1).double()).view(-1, 1)
        assert bool(((lse.cpu().double() - want).abs() <= 2.0 ** -21 * want).all()), log2
