"""Cases of the quantised serving operators: the 8-bit linear layer (int8 cast per token, int8 product with scales per token
and channel) and the paged nvfp4 key/value cache (append with position rotation, read back, attention).

`own` selects between the plain form of each operator (elementary torch operations in 32 bits) and the framework's calls.
The cache is one uint8 tensor (pages, kv heads, 2, page * 9 * head_dim / 16): for keys and for values of a page and head
the e2m1 codes of its tokens (page, head_dim / 2), the even element in the low nibble, then their e4m3 block scales
(page, head_dim / 16)."""
import math
import random

import torch

own = False

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a projection of a decoder layer: latency of two small launches
        {"name": "linear_one_token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "bias": False},
        # a prompt of 2000 tokens through a wide projection
        {"name": "linear_prompt", "op": "linear", "m": 2000, "n": 4096, "k": 7168, "bias": True},
        # a decode batch against a feed-forward weight: bound by reading the weight
        {"name": "mm_decode_batch", "op": "mm", "m": 64, "n": 14336, "k": 4096, "out": "bfloat16", "bias": False},
        # a large prefill product: bound by the tensor cores
        {"name": "mm_large", "op": "mm", "m": 8192, "n": 8192, "k": 8192, "out": "bfloat16", "bias": False},
        # nothing a multiple of a tile, 32-bit output (logits, a residual kept in fp32)
        {"name": "mm_odd", "op": "mm", "m": 1111, "n": 5003, "k": 2064, "out": "float32", "bias": True},
        # one new token for each of 64 sequences: the decode step's append
        {"name": "append_decode", "op": "append", "seqs": 64, "new": 1, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16,
         "rot": 128, "interleaved": False, "lens": 1},
        # prompts of up to 4096 tokens, four at a time
        {"name": "append_prompt", "op": "append", "seqs": 4, "new": 4096, "q_heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "rot": 128, "interleaved": False, "lens": 2},
        # narrow heads, one of them for all queries, half of each rotated in neighbouring pairs
        {"name": "append_narrow", "op": "append", "seqs": 7, "new": 333, "q_heads": 12, "kv_heads": 1, "head_dim": 64, "page": 32,
         "rot": 32, "interleaved": True, "lens": 3},
        # a single sequence of 1000 tokens, one query: the smallest decode
        {"name": "attn_one", "op": "attn", "seqs": 1, "q_len": 1, "ctx": 1000, "ragged": False, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "lens": 4},
        # 64 sequences of uneven length, some slots of the batch idle
        {"name": "attn_decode_batch", "op": "attn", "seqs": 64, "q_len": 1, "ctx": 16384, "ragged": True, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 32, "lens": 5},
        # two very long contexts
        {"name": "attn_long", "op": "attn", "seqs": 2, "q_len": 1, "ctx": 131072, "ragged": False, "q_heads": 64, "kv_heads": 8,
         "head_dim": 128, "page": 64, "lens": 6},
        # a chunk of a prompt over what the cache holds already
        {"name": "attn_prompt", "op": "attn", "seqs": 1, "q_len": 4096, "ctx": 12288, "ragged": False, "q_heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "lens": 7},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "mm", "append", "append", "attn", "attn", "attn"])
    while True:
        if op in ("linear", "mm"):
            c = {"op": op, "m": _log(rng, 1, 8192), "n": _log(rng, 200, 16384), "k": 16 * _log(rng, 8, 1024), "bias": rng.random() < 0.5}
            if op == "mm":
                c["out"] = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
            if c["m"] * c["n"] * c["k"] <= 8192 ** 3:
                return c
            continue
        kv = rng.choice([1, 2, 4, 8])
        c = {"op": op, "seqs": _log(rng, 1, 64), "q_heads": kv * rng.choice([1, 2, 4, 5, 8, 16]), "kv_heads": kv,
             "head_dim": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 128]), "lens": rng.randrange(1 << 30)}
        if op == "append":
            c |= {"new": 1 if rng.random() < 0.3 else _log(rng, 2, 4096), "interleaved": rng.random() < 0.3}
            c["rot"] = c["head_dim"] if rng.random() < 0.7 else c["head_dim"] // 2
            if c["seqs"] * c["new"] * (c["q_heads"] + 2 * kv) * c["head_dim"] <= 4 * 4096 * 48 * 128:
                return c
            continue
        c |= {"q_len": rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 17, 4096)]), "ctx": _log(rng, 2, 65536), "ragged": rng.random() < 0.7}
        c["q_len"] = min(c["q_len"], c["ctx"])
        scores = c["seqs"] * c["q_heads"] * c["q_len"] * c["ctx"]
        cached = c["seqs"] * kv * c["ctx"] * c["head_dim"]
        if scores <= 32 * 4096 * 12288 and cached <= 64 * 16384 * 8 * 128:
            return c


def _new_tokens(case):
    """append: for each sequence (tokens already on its first listed page, new tokens, position of the page's first token)."""
    r = random.Random(case["lens"])
    out = []
    for b in range(case["seqs"]):
        n = case["new"] if b == 0 else r.randint((case["new"] + 1) // 2, case["new"])
        out.append((r.randrange(case["page"]), n, case["page"] * r.randrange(65536 // case["page"])))
    return out


def _lengths(case):
    """attn: for each sequence (queries, cached tokens).  Ragged batches keep an idle slot: a query without any key."""
    r = random.Random(case["lens"])
    out = []
    for b in range(case["seqs"]):
        q, n = case["q_len"], case["ctx"]
        if case["ragged"]:
            q, n = (q, n) if b == 0 else (r.randint(1, q), r.randint(max(1, n // 8), n))
            n = 0 if b % 16 == 3 else n
        out.append((q, n))
    return out


def _visible(q, n):
    """Pairs of a query and a key that it sees: query i of q sees keys 0 .. n - q + i."""
    first = max(0, n - q + 1)          # keys of the first query
    rows = q if n >= q else n          # queries that see any
    return rows * first + rows * (rows - 1) // 2 if n >= q else rows * (rows + 1) // 2


def work(case):
    if case["op"] in ("linear", "mm"):
        m, n, k = case["m"], case["n"], case["k"]
        out = 4 if case.get("out") == "float32" else 2
        a = 2 * m * k if case["op"] == "linear" else m * k + 4 * m
        return {"bytes": a + n * k + 4 * n + out * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    d, kv, hq = case["head_dim"], case["kv_heads"], case["q_heads"]
    packed = 2 * kv * d * 9 // 16      # bytes of a cached token
    if case["op"] == "append":
        seqs = _new_tokens(case)
        new, kept = sum(n for _, n, _ in seqs), sum(p + n for p, n, _ in seqs)
        return {"bytes": new * (4 * hq * d + 4 * kv * d + 4 * case["rot"] + packed + 16) + kept * (packed + 4 * kv * d),
                "flops": new * (3 * (hq + kv) * case["rot"] + 8 * kv * d) + kept * 4 * kv * d}
    seqs = _lengths(case)
    rows = sum(q for q, _ in seqs)
    return {"bytes": sum(n for _, n in seqs) * packed + rows * hq * (4 * d + 4) + 4 * sum(-(-n // case["page"]) for _, n in seqs),
            "flops": 4 * hq * d * sum(_visible(q, n) for q, n in seqs)}


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, rows, cols):
    """Activations of a decoder: a few channels an order of magnitude louder than the rest."""
    x = _randn(g, rows, cols)
    loud = torch.rand(cols, device="cuda", generator=g) < 0.005
    return (x * torch.where(loud, 12.0, 1.0)).to(torch.bfloat16)


def _nvfp4(x, outer):
    """(e2m1 codes as whole numbers 0..15, e4m3 block scales) of x (..., d) in 32 bits; every division an IEEE division."""
    b = x.unflatten(-1, (-1, 16))
    amax = b.abs().amax(-1)
    inner = (amax / torch.full_like(amax, 6.0) / outer).clamp(0.015625, 448.0).to(torch.float8_e4m3fn)
    y = b * ((torch.ones_like(outer) / outer) / inner.float()).unsqueeze(-1)
    v = y.abs()
    code = ((v > 0.25).byte() + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0) + 8 * torch.signbit(y)).flatten(-2)
    return code.byte(), inner


def _planes(cache, d):
    """The codes (pages, heads, 2, page, d / 2) and scale bytes (pages, heads, 2, page, d / 16) of a cache, as views."""
    page = cache.shape[-1] * 16 // (9 * d)
    return cache[..., :page * d // 2].unflatten(-1, (page, d // 2)), cache[..., page * d // 2:].unflatten(-1, (page, d // 16))


def _pool(g, pages, kv, page, d):
    """A cache whose every slot holds quantised keys and values, and the outer scales of both."""
    channel = torch.exp(0.5 * _randn(g, 2, kv, 1, d)).transpose(0, 1)          # (kv, 2, 1, d)
    # a moving average of maxima, as calibration leaves it: a number of no special form
    outer = (torch.tensor([12.0, 9.0], device="cuda") * (1 + 0.2 * torch.rand(2, device="cuda", generator=g))) / 2688
    cache = torch.empty(pages, kv, 2, page * 9 * d // 16, dtype=torch.uint8, device="cuda")
    codes, scales = _planes(cache, d)
    step = max(1, (1 << 25) // (kv * 2 * page * d))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = _randn(g, n, kv, 2, page, d) * channel
        c, s = _nvfp4(x, outer.view(2, 1, 1))
        codes[at:at + n] = c[..., 0::2] + 16 * c[..., 1::2]
        scales[at:at + n] = s.view(torch.uint8)
    return cache, outer[:1].clone(), outer[1:].clone()


def _table(g, lens, page):
    """Pages of each sequence in the pool's shuffled order, and how many pages the pool has."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + max(2, sum(need) // 8)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).cpu()
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table.cuda(), pages


def _ends(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["op"] in ("linear", "mm"):
        m, n, k = case["m"], case["n"], case["k"]
        w = _randn(g, n, k) / math.sqrt(k)
        s["sb"] = w.abs().amax(1, keepdim=True) / 127.0
        s["b"] = (w / s["sb"]).round().to(torch.int8)
        del w
        s["bias"] = _randn(g, n).to(torch.bfloat16) if case["bias"] else None
        x = _activations(g, m, k)
        if case["op"] == "linear":
            s["x"] = x
            s["out"] = torch.bfloat16
        else:
            s["sa"] = x.float().abs().amax(1, keepdim=True) / 127.0
            s["a"] = (x.float() / s["sa"]).round().to(torch.int8)
            s["out"] = getattr(torch, case["out"])
        return s
    d, kv, hq, page = case["head_dim"], case["kv_heads"], case["q_heads"], case["page"]
    if case["op"] == "append":
        seqs = _new_tokens(case)
        kept = [p + n for p, n, _ in seqs]
        s["table"], pages = _table(g, kept, page)
        s["cache"], s["ko"], s["vo"] = _pool(g, pages, kv, page, d)
        host = s["table"].cpu()
        slots, positions = [], []
        for b, (p, n, base) in enumerate(seqs):
            at = torch.arange(p, p + n)
            slots.append(host[b, at // page].long() * page + at % page)
            positions.append(base + at)
        s["slots"], s["positions"] = torch.cat(slots).cuda(), torch.cat(positions).cuda()
        s["ends"], s["total"] = _ends(kept).cuda(), sum(kept)
        # the rows of a fused projection: queries, keys and values of a token side by side
        t = s["slots"].numel()
        qkv = _randn(g, t, hq + 2 * kv, d).to(torch.bfloat16)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + kv], qkv[:, hq + kv:]
        rate = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        angle = torch.arange(65536 + 4096 + 2 * page, device="cuda", dtype=torch.float64)[:, None] * rate
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        return s
    seqs = _lengths(case)
    s["table"], pages = _table(g, [n for _, n in seqs], page)
    s["cache"], s["ko"], s["vo"] = _pool(g, pages, kv, page, d)
    rows = sum(q for q, _ in seqs)
    s["q"] = _randn(g, rows, hq, d).to(torch.bfloat16)
    s["kv_lens"] = torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda")
    s["q_lens"] = torch.tensor([q for q, _ in seqs], dtype=torch.int32, device="cuda")
    s["cu_q"] = _ends([q for q, _ in seqs]).cuda()
    s["max_q"] = max(q for q, _ in seqs)
    # where each query row sits in the padded batch (sequence, place in the sequence)
    s["row_seq"] = torch.repeat_interleave(torch.arange(len(seqs)), torch.tensor([q for q, _ in seqs])).cuda()
    s["row_at"] = torch.cat([torch.arange(q) for q, _ in seqs]).cuda()
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _product(a, sa, b, sb, bias, out):
    y = (a.float() @ b.float().T) * sa * sb.view(1, -1)
    return (y if bias is None else y + bias.float()).to(out)


def _int8_cast(x):
    x = x.float()
    amax = x.abs().amax(1, keepdim=True).clamp_min(float(torch.tensor(1e-12, dtype=torch.bfloat16)))
    s = amax / torch.full_like(amax, 127.0)
    return (x * (torch.ones_like(s) / s)).round().clamp(-127, 127).to(torch.int8), s


def _rotate(x, cos, sin, interleaved):
    """x (t, heads, d) with its first 2 * cos.shape[-1] elements rotated; products and differences each rounded to 32 bits."""
    half = cos.shape[-1]
    x = x.float()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    ra, rb = a * c - b * s, b * c + a * s
    r = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([r, x[..., 2 * half:]], -1)


def _values(codes, scales):
    """32-bit values of packed codes (..., d / 2) under e4m3 scale bytes (..., d / 16), without the outer scale."""
    grid = torch.tensor(_GRID + tuple(-x for x in _GRID), device=codes.device)
    byte = torch.arange(256, device=codes.device)
    pair = torch.stack([grid[byte % 16], grid[byte // 16]], 1)
    v = pair[codes.int()].flatten(-2)
    return (v.unflatten(-1, (-1, 16)) * scales.contiguous().view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def _plain_append(s):
    case = s["case"]
    d, page = case["head_dim"], case["page"]
    cos, sin = s["cos_sin"][s["positions"]].chunk(2, 1)
    q = _rotate(s["q"], cos, sin, case["interleaved"]).to(torch.bfloat16)
    codes, scales = _planes(s["cache"], d)
    at, off = s["slots"] // page, s["slots"] % page
    x = torch.stack([_rotate(s["k"], cos, sin, case["interleaved"]), s["v"].float()], 2)          # (t, heads, 2, d)
    c, inner = _nvfp4(x, torch.cat([s["ko"], s["vo"]]).view(2, 1))
    codes[at, :, :, off] = c[..., 0::2] + 16 * c[..., 1::2]
    scales[at, :, :, off] = inner.view(torch.uint8)
    # read the sequences back: row r of sequence b is token r - ends[b] of it
    row = torch.arange(s["total"], device="cuda")
    b = torch.searchsorted(s["ends"], row, right=True) - 1
    i = row - s["ends"][b]
    p, o = s["table"][b, i // page].long(), i % page
    x = _values(codes[p, :, :, o], scales[p, :, :, o])
    return q, (x[:, :, 0] * s["ko"]).to(torch.bfloat16), (x[:, :, 1] * s["vo"]).to(torch.bfloat16)


def _plain_attention(s):
    case = s["case"]
    d, kv, hq, page, n = case["head_dim"], case["kv_heads"], case["q_heads"], case["page"], case["seqs"]
    codes, scales = _planes(s["cache"], d)
    t = s["table"].long()
    width = t.shape[1] * page

    def side(w):
        x = _values(codes[t, :, w], scales[t, :, w])                                 # (seqs, pages, heads, page, d)
        return x.transpose(1, 2).reshape(n, kv, width, d)

    q = torch.zeros(n, s["max_q"], hq, d, device="cuda")
    q[s["row_seq"], s["row_at"]] = s["q"].float()
    q = q.view(n, s["max_q"], kv, hq // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    score = (q @ side(0).transpose(2, 3)) * (s["ko"] / math.sqrt(d))
    score = score.view(n, kv, hq // kv, s["max_q"], width)
    last = (s["kv_lens"] - s["q_lens"]).view(n, 1) + torch.arange(s["max_q"], device="cuda")      # newest key that a query sees
    seen = torch.arange(width, device="cuda") <= last.unsqueeze(-1)                                # (seqs, max_q, width)
    score = score.masked_fill(~seen.view(n, 1, 1, s["max_q"], width), -math.inf)
    m = score.amax(-1, keepdim=True)
    score = (score - torch.where(m == -math.inf, 0.0, m)).exp()
    z = score.sum(-1, keepdim=True)
    o = (score.view(n, kv, -1, width) @ side(1)).view(n, kv, hq // kv, s["max_q"], d) * s["vo"] / torch.where(z == 0, 1.0, z)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s["max_q"], hq, d).to(torch.bfloat16)
    lse = (m + z.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(n, s["max_q"], hq)
    return o[s["row_seq"], s["row_at"]], lse[s["row_seq"], s["row_at"]]


def run(s):
    case = s["case"]
    if own:
        from quant_cast_bench_b200.quant_cast_cuda import native_ops as N
        if case["op"] == "linear":
            q, sa = N.rowwise_int8_native(s["x"])
            return N.int8_scaled_mm_native(q, s["b"], sa, s["sb"], bias=s["bias"])
        if case["op"] == "mm":
            return N.int8_scaled_mm_native(s["a"], s["b"], s["sa"], s["sb"], bias=s["bias"], out_dtype=s["out"])
        if case["op"] == "append":
            q = N.nvfp4_kv_append_native(s["k"], s["v"], s["cache"], s["slots"], s["ko"], s["vo"], positions=s["positions"],
                                         cos_sin=s["cos_sin"], interleaved=case["interleaved"], q=s["q"])
            k, v = N.nvfp4_kv_gather_native(s["cache"], s["table"], s["ends"], s["total"], case["head_dim"], s["ko"], s["vo"])
            return q, k, v
        if case["q_len"] == 1:
            return N.nvfp4_kv_attention_native(s["q"], s["cache"], s["table"], s["kv_lens"], s["ko"], s["vo"])
        return N.nvfp4_kv_attention_native(s["q"], s["cache"], s["table"], s["kv_lens"], s["ko"], s["vo"], cu_q=s["cu_q"], max_q=s["max_q"])
    if case["op"] == "linear":
        a, sa = _int8_cast(s["x"])
        return _product(a, sa, s["b"], s["sb"], s["bias"], s["out"])
    if case["op"] == "mm":
        return _product(s["a"], s["sa"], s["b"], s["sb"], s["bias"], s["out"])
    return _plain_append(s) if case["op"] == "append" else _plain_attention(s)


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_values(cache, d):
    """All values of a cache (pages, heads, 2, page, d) in 64 bits, read bit by bit, without the outer scales."""
    page = cache.shape[-1] * 16 // (9 * d)
    raw = cache[..., :page * d // 2].reshape(*cache.shape[:3], page, d // 2, 1).to(torch.int16)
    nib = torch.cat([raw & 15, raw >> 4], -1).flatten(-2)
    e, m = (nib >> 1) & 3, (nib & 1).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1)) * (1 - 2 * (nib >> 3)).double()
    sc = cache[..., page * d // 2:].reshape(*cache.shape[:3], page, d // 16).to(torch.int16)
    e, m = (sc >> 3) & 15, (sc & 7).double()
    w = torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.exp2(e.double() - 7))
    return v * w.repeat_interleave(16, -1)


def _exact_append(s):
    case = s["case"]
    d, rot, page = case["head_dim"], case["rot"], case["page"]
    pair = torch.arange(rot, device="cuda")
    if case["interleaved"]:
        other, freq, first = pair ^ 1, pair // 2, pair % 2 == 0
    else:
        other, freq, first = (pair + rot // 2) % rot, pair % (rot // 2), pair < rot // 2
    table = s["cos_sin"].double()[s["positions"]]
    cos, sin = table[:, freq].unsqueeze(1), table[:, rot // 2 + freq].unsqueeze(1)

    def turn(x):
        x = x.double().clone()
        x[..., :rot] = x[..., :rot] * cos + torch.where(first, -1.0, 1.0) * x[..., other] * sin
        return x

    def rounded(x, outer):
        """The nvfp4 value nearest to each element, without the outer scale."""
        outer = outer.double()
        b = x.unflatten(-1, (-1, 16))
        inner = (b.abs().amax(-1, keepdim=True) / 6 / outer).clamp(2.0 ** -6, 448)
        step = torch.exp2(torch.floor(torch.log2(inner)) - 3)          # distance of the e4m3 numbers around it (no subnormals from 2^-6 up)
        inner = (inner / step).round() * step
        y = b / outer / inner
        e = torch.exp2(torch.floor(torch.log2(y.abs().clamp(1.0, 6.0))) - 1)
        return ((y.abs().clamp(max=6.0) / e).round() * e * torch.where(y < 0, -1.0, 1.0) * inner).flatten(-2)

    cache = _exact_values(s["cache"], d)
    cache[s["slots"] // page, :, 0, s["slots"] % page] = rounded(turn(s["k"]), s["ko"])
    cache[s["slots"] // page, :, 1, s["slots"] % page] = rounded(s["v"].double(), s["vo"])
    lens = (s["ends"][1:] - s["ends"][:-1]).tolist()
    rows = [cache[s["table"][b].long()].transpose(1, 3)[:, :, :, :].flatten(0, 1)[:n] for b, n in enumerate(lens)]   # (page * pages, 2, heads, d)
    x = torch.cat(rows)
    return turn(s["q"]), x[:, 0] * s["ko"].double(), x[:, 1] * s["vo"].double()


def _exact_attention(s):
    case = s["case"]
    d, kv, g, page = case["head_dim"], case["kv_heads"], case["q_heads"] // case["kv_heads"], case["page"]
    out, lse = [], []
    cu, lens = s["cu_q"].tolist(), s["kv_lens"].tolist()
    for b, n in enumerate(lens):
        q = s["q"][cu[b]:cu[b + 1]].double()
        rows = q.shape[0]
        x = _exact_values(s["cache"][s["table"][b, :-(-n // page)].long()], d).permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n]
        k, v = x[:, 0] * s["ko"].double(), x[:, 1] * s["vo"].double()
        o = torch.zeros(rows, kv * g, d, dtype=torch.float64, device="cuda")
        z = torch.full((rows, kv * g), -math.inf, dtype=torch.float64, device="cuda")
        hidden = torch.arange(n, device="cuda") > n - rows + torch.arange(rows, device="cuda").unsqueeze(1)
        some = ~hidden.all(1) if n else torch.zeros(rows, dtype=torch.bool, device="cuda")
        for h in range(kv * g if n else 0):
            score = (q[:, h] @ k[h // g].T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            z[:, h] = torch.logsumexp(score, 1)
            o[some, h] = torch.exp(score[some] - z[some, h].unsqueeze(1)) @ v[h // g]
        out.append(o)
        lse.append(z)
    return torch.cat(out), torch.cat(lse)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("linear", "mm"):
        if case["op"] == "linear":
            x = s["x"].double()
            sa = x.abs().amax(1, keepdim=True).clamp_min(1e-12) / 127
            a = (x / sa).round()
        else:
            a, sa = s["a"].double(), s["sa"].double()
        y = torch.mm(a, s["b"].double().t()).mul_(sa).mul_(s["sb"].double().t())
        return y if s["bias"] is None else y + s["bias"].double()
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)
