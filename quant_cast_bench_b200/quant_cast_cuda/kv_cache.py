"""Paged nvfp4 key/value cache: append (with position rotation), read-back and attention.  No counterpart in the reference:
its nvfp4 cast with a cache's pages for destination, and the operators that read them.

    cache = nvfp4_kv_cache_cuda(num_pages, kv_heads, page, head_dim)
    q = nvfp4_kv_append_cuda(k, v, cache, slots, k_outer, v_outer, positions=pos, cos_sin=table, q=q)
    out, lse = nvfp4_kv_attention_cuda(q, cache, block_table, kv_lens, k_outer, v_outer)

The cache is one uint8 tensor (num_pages, kv_heads, 2, page * 9 * head_dim / 16); include/quant_cast_cuda.h has its layout.
Page, slot and position numbers live on the device and are checked there: one outside its range is not followed, and sets the
device error word (`_lib.device_error()`, codes 20 to 22; QCC_CHECK_DEVICE=1 raises).
"""
import ctypes
import math

import torch

from . import _lib as L
from .recipes import _on_device, _p, _stream

_PAGES = (16, 32, 64, 128)


def nvfp4_kv_cache_cuda(num_pages, kv_heads, page, head_dim, device="cuda"):
    """An uninitialised cache: a slot is read only once a sequence's length says that it holds a token."""
    assert head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}"
    assert page in _PAGES, f"page must be one of {_PAGES}, got {page}"
    assert kv_heads >= 1
    return torch.empty((num_pages, kv_heads, 2, page * 9 * head_dim // 16), dtype=torch.uint8, device=device)


def _check_cache(cache, head_dim):
    """(kv_heads, page) of a cache whose heads have head_dim elements."""
    if not (isinstance(cache, torch.Tensor) and cache.is_cuda):
        raise ValueError("cache must be a CUDA tensor (quant_cast_cuda has no CPU path)")
    assert cache.dtype == torch.uint8 and cache.dim() == 4 and cache.shape[2] == 2 and cache.is_contiguous(), (
        "cache: a contiguous uint8 tensor (pages, kv_heads, 2, page * 9 * head_dim / 16), see nvfp4_kv_cache_cuda")
    assert head_dim in (64, 128), f"head_dim must be 64 or 128, got {head_dim}"
    page, rest = divmod(cache.shape[3], 9 * head_dim // 16)
    assert rest == 0 and page in _PAGES, f"a page block of {cache.shape[3]} bytes is no page of {_PAGES} tokens of {head_dim} elements"
    return cache.shape[1], page


def _check_rows(t, name, cache, heads=None):
    assert t.device == cache.device and t.dtype == torch.bfloat16 and t.dim() == 3, f"{name} must be a 3-D bfloat16 tensor on the cache's device"
    assert t.stride(2) == 1 and (t.numel() == 0 or (t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0 and t.data_ptr() % 16 == 0)), (
        f"{name}: rows must be contiguous and 16-byte aligned")
    assert heads is None or t.shape[1] == heads, f"{name} has {t.shape[1]} heads, expected {heads}"


def _check_outer(k_outer, v_outer, cache):
    for t, name in ((k_outer, "k_outer"), (v_outer, "v_outer")):
        assert t.device == cache.device and t.dtype == torch.float32 and t.numel() == 1, f"{name}: one fp32 value on the cache's device"


def _check_numbers(t, name, dtype, shape, cache):
    assert t.device == cache.device and t.dtype == dtype and tuple(t.shape) == shape and t.is_contiguous(), (
        f"{name}: contiguous {dtype} of shape {shape} on the cache's device")


def _check_table(table, cache):
    assert table.device == cache.device and table.dtype == torch.int32 and table.dim() == 2 and (table.shape[1] <= 1 or table.stride(1) == 1) and table.stride(0) >= 0, (
        "block_table: int32 (seqs, pages) with contiguous rows on the cache's device")


def nvfp4_kv_append_cuda(k, v, cache, slots, k_outer, v_outer, positions=None, cos_sin=None, interleaved=False, q=None):
    """Append keys and values (tokens, kv_heads, head_dim) bf16 to the cache, in place.  slots (tokens) int64: page * page number + offset; a negative one
    skips the token; the others must differ.  With cos_sin (max_pos, rot) fp32, rot/2 cosines then rot/2 sines of a position, and
    positions (tokens) int64, the first rot elements of each key are rotated on the way: halves (i, i + rot/2), or neighbouring
    pairs if interleaved.  rot: a multiple of 32 up to head_dim.  k_outer, v_outer: the outer scales of the nvfp4 cast, as
    nvfp4_gs_scale_cuda gives them; > 0.  q (tokens, q_heads, head_dim), if given, is rotated the same way and returned
    contiguous; otherwise the result is None."""
    lib = L.load()
    if not (isinstance(k, torch.Tensor) and k.is_cuda):
        raise ValueError("k must be a CUDA tensor (quant_cast_cuda has no CPU path)")
    assert k.dim() == 3, "k must be (tokens, kv_heads, head_dim)"
    T, D = k.shape[0], k.shape[2]
    heads, page = _check_cache(cache, D)
    _check_rows(k, "k", cache, heads)
    _check_rows(v, "v", cache, heads)
    assert v.shape == k.shape, "k and v differ in shape"
    _check_outer(k_outer, v_outer, cache)
    _check_numbers(slots, "slots", torch.int64, (T,), cache)
    rot = 0
    if cos_sin is not None:
        assert cos_sin.device == cache.device and cos_sin.dtype == torch.float32 and cos_sin.dim() == 2 and cos_sin.is_contiguous(), (
            "cos_sin: contiguous fp32 (max_pos, rot) on the cache's device")
        rot = cos_sin.shape[1]
        assert 0 < rot <= D and rot % 32 == 0 and cos_sin.shape[0] > 0, f"rot must be a multiple of 32 up to {D}, got cos_sin {tuple(cos_sin.shape)}"
        assert positions is not None, "a rotation needs positions"
        _check_numbers(positions, "positions", torch.int64, (T,), cache)
    out = None
    if q is not None:
        _check_rows(q, "q", cache)
        assert q.shape[0] == T and q.shape[2] == D, "q must have k's tokens and head_dim"
        out = torch.empty((T, q.shape[1], D), dtype=torch.bfloat16, device=q.device)
    if T == 0:
        return out
    a = L.KvAppendArgs(_p(k), _p(v), _p(q), _p(out), (ctypes.c_int64 * 2)(*k.stride()[:2]), (ctypes.c_int64 * 2)(*v.stride()[:2]),
                       (ctypes.c_int64 * 2)(*(q.stride()[:2] if q is not None else (0, 0))), T, _p(cache), cache.shape[0], _p(slots),
                       _p(positions) if rot else None, _p(cos_sin), cos_sin.shape[0] if rot else 0, _p(k_outer), _p(v_outer), heads,
                       q.shape[1] if q is not None else 0, D, page, rot, (L.ROPE_INTERLEAVED if interleaved else 0) | L.div_flag())
    with _on_device(cache.device):
        L.check(lib.qcc_nvfp4_kv_append(ctypes.byref(a), _stream(cache)), "nvfp4_kv_append")
    L.launch_count += 1
    return out


def nvfp4_kv_gather_cuda(cache, block_table, cu_kv, total, head_dim, k_outer, v_outer):
    """Read sequences back: (k, v), each (total, kv_heads, head_dim) bf16 = code * scale * outer.  block_table (seqs, pages) int32;
    rows cu_kv[b] .. cu_kv[b + 1] - 1 (cu_kv: int32 (seqs + 1), ascending from 0) are the tokens of sequence b; rows from cu_kv[-1] on become zero."""
    lib = L.load()
    heads, page = _check_cache(cache, head_dim)
    _check_table(block_table, cache)
    _check_numbers(cu_kv, "cu_kv", torch.int32, (block_table.shape[0] + 1,), cache)
    _check_outer(k_outer, v_outer, cache)
    k = torch.empty((total, heads, head_dim), dtype=torch.bfloat16, device=cache.device)
    v = torch.empty_like(k)
    with _on_device(cache.device):
        L.check(lib.qcc_nvfp4_kv_gather(_p(cache), cache.shape[0], heads, page, head_dim, _p(block_table), block_table.stride(0), block_table.shape[1],
                                        _p(cu_kv), block_table.shape[0], total, _p(k_outer), _p(v_outer), _p(k), _p(v), _stream(cache)), "nvfp4_kv_gather")
    L.launch_count += 1
    return k, v


def nvfp4_kv_attention_cuda(q, cache, block_table, kv_lens, k_outer, v_outer, cu_q=None, max_q=None, scale=None):
    """Attention of q (rows, q_heads, head_dim) bf16, already rotated, over the cache: (out like q, lse (rows, q_heads) fp32).
    block_table (seqs, pages) int32, kv_lens (seqs) int32: the tokens that the cache holds of each sequence.  Without cu_q each sequence has one query;
    with cu_q (seqs + 1) int32, ascending from 0, rows cu_q[b] .. cu_q[b + 1] - 1 are the last tokens of sequence b and attend causally; max_q (a Python int) is at
    least the most queries of a sequence.  scale defaults to 1 / sqrt(head_dim).  q_heads must be a multiple of kv_heads.
    A query without keys, and a row behind the last sequence, gets zeros and lse -inf."""
    lib = L.load()
    if not (isinstance(q, torch.Tensor) and q.is_cuda):
        raise ValueError("q must be a CUDA tensor (quant_cast_cuda has no CPU path)")
    assert q.dim() == 3, "q must be (rows, q_heads, head_dim)"
    rows, hq, D = q.shape
    heads, page = _check_cache(cache, D)
    _check_rows(q, "q", cache)
    assert hq >= heads and hq % heads == 0, f"{hq} query heads do not divide among {heads} kv heads"
    _check_table(block_table, cache)
    seqs = block_table.shape[0]
    _check_numbers(kv_lens, "kv_lens", torch.int32, (seqs,), cache)
    _check_outer(k_outer, v_outer, cache)
    if cu_q is None:
        assert rows == seqs, f"{rows} query rows for {seqs} sequences: several queries a sequence need cu_q"
        max_q = 1
    else:
        _check_numbers(cu_q, "cu_q", torch.int32, (seqs + 1,), cache)
        assert max_q is not None and max_q >= 1, "cu_q needs max_q"
        max_q = min(max_q, 0x7FFFFFFF)      # (more rows than that there are not; a C int)
    if scale is not None and not scale > 0:
        raise ValueError(f"scale must be positive, got {scale}")
    out = torch.empty((rows, hq, D), dtype=torch.bfloat16, device=q.device)
    lse = torch.empty((rows, hq), dtype=torch.float32, device=q.device)
    if rows == 0 or seqs == 0:
        return out.zero_(), lse.fill_(-math.inf)
    a = L.KvAttentionArgs(_p(q), (ctypes.c_int64 * 2)(*q.stride()[:2]), rows, _p(cache), cache.shape[0], _p(block_table), block_table.stride(0),
                          block_table.shape[1], _p(kv_lens), _p(cu_q), seqs, max_q, _p(k_outer), _p(v_outer),
                          1.0 / math.sqrt(D) if scale is None else scale, hq, heads, D, page, _p(out), _p(lse))
    with _on_device(q.device):
        nws = lib.qcc_nvfp4_kv_attention_workspace_bytes(rows, seqs, max_q, hq, heads, D)
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device)
        L.check(lib.qcc_nvfp4_kv_attention(ctypes.byref(a), _p(ws), nws, _stream(q)), "nvfp4_kv_attention")
        L.launch_count += lib.qcc_nvfp4_kv_attention_launches(ctypes.byref(a))
    return out, lse
