"""Paged KV caches: rows of K and V written into pages, in bf16 or rounded to 8 bits with one scale for each token and head, read back, and
attention of one new token of each sequence over them.

As in ``functional``, every function has two bodies: CUDA tensors go to the hand-written sm_100a kernels (head dimension 64 or 128), CPU
tensors take a plain torch restatement (fp32, or fp64 for fp64 inputs).

    cache = paged_cache(pages, KVH, page, D, device, "int8")              # one per layer; a table serves all of them
    paged_append(k, v, cache, table, seq, pos, cos, sin)                  # prompts: any tokens of any sequences
    o = paged_attn_append(kqv, cache, table, lens, QH, KVH, cos, sin)     # one new token of each sequence
    paged_read(cache, table, lens, kcache, vcache)                        # out into contiguous caches, for ``tree_attn_append``

``table`` int32 [B, width] names the pages of each sequence: token t stands in row t % page of page table[b, t // page]. An entry that is
no page of the pool is one that is not there: what would be written to it is left out, what would be read from it is not seen. Sequences
may share pages that are only read.

In 8 bits a row x of one token and head is held as round(x / scale), scale = max(largest |x| (1 / L), 2^-80), with L = 127 (int8) or 448
(e4m3) and 1 / L rounded to fp32. Rows have to be finite.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import functional as F
from . import native
from .masked_attn import _modifier, _scale, _softmax_reference, _scores_reference, _work_dtype

_f = ctypes.c_float
_ll = ctypes.c_longlong
KINDS = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
HELD = {torch.bfloat16: 0, torch.int8: 1, torch.float8_e4m3fn: 2}
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
LEAST_SCALE = 2.0 ** -80
HEAD_DIMS = (64, 128)                                        # that there are CUDA kernels for
PAGES = (32, 64, 128, 256, 512, 1024)


class PagedCache(NamedTuple):
    """The pool of one layer: ``k``, ``v`` [pages, KV heads, page, D]; ``k_scale``, ``v_scale`` fp32 [pages, KV heads, page] for int8 and
    e4m3 (float8_e4m3fn) rows, None for rows in floating point (bf16; on the CPU fp32 and fp64 too)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: Optional[torch.Tensor] = None
    v_scale: Optional[torch.Tensor] = None


def paged_cache(pages: int, KVH: int, page: int, D: int, device, kind: str = "bf16", dtype=None) -> PagedCache:
    """An empty pool. ``kind``: "bf16", "int8" or "e4m3"; ``dtype`` replaces the type of "bf16" (CPU: fp32, fp64)."""
    if kind not in KINDS:
        raise ValueError(f"paged_cache: kind is one of {', '.join(KINDS)}")
    if pages < 1 or KVH < 1 or D < 1 or page not in PAGES:
        raise ValueError(f"paged_cache: at least one page and KV head, pages of one of {PAGES} tokens")
    dt = KINDS[kind] if kind != "bf16" or dtype is None else dtype
    k, v = (torch.zeros((pages, KVH, page, D), dtype=dt, device=device) for _ in range(2))
    if dt not in LARGEST:
        return PagedCache(k, v)
    return PagedCache(k, v, *(torch.zeros((pages, KVH, page), dtype=torch.float32, device=device) for _ in range(2)))


def _check_cache(name: str, cache: PagedCache, table, B: int | None = None) -> None:
    k, v, ks, vs = cache
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.shape[2] not in PAGES or 0 in k.shape:
        raise ValueError(f"{name}: k and v of the cache are [pages, KV heads, page, D] of one type, pages of one of {PAGES} tokens")
    if k.dtype not in HELD and k.is_cuda or not (k.dtype in LARGEST or k.dtype.is_floating_point):
        raise TypeError(f"{name}: rows are held in bf16, int8 or float8_e4m3fn")
    if (k.dtype in LARGEST) != (ks is not None) or (ks is None) != (vs is None):
        raise ValueError(f"{name}: int8 and e4m3 rows have scales, others have none")
    if ks is not None and (ks.shape != k.shape[:3] or vs.shape != ks.shape or ks.dtype != torch.float32 or vs.dtype != torch.float32):
        raise ValueError(f"{name}: scales are float32 [pages, KV heads, page]")
    if any(t is not None and not t.is_contiguous() for t in cache):
        raise ValueError(f"{name}: the cache is contiguous")
    if table.dim() != 2 or table.dtype != torch.int32 or table.shape[1] < 1 or (B is not None and table.shape[0] != B):
        raise ValueError(f"{name}: table is int32 [B, width]")
    if table.shape[1] * k.shape[2] >= 1 << 31:
        raise ValueError(f"{name}: a table holds fewer than 2^31 tokens a sequence")
    if any(t is not None and t.device != k.device for t in (v, ks, vs, table)):
        raise ValueError(f"{name}: all tensors are on one device")


def _check_int32(name: str, n: int, like, **vectors) -> None:
    for what, t in vectors.items():
        if tuple(t.shape) != (n,) or t.dtype != torch.int32:
            raise ValueError(f"{name}: {what} is int32 [{n}]")
        if t.device != like.device:
            raise ValueError(f"{name}: all tensors are on one device")


def _check_tables(name: str, cos, sin, D: int, like) -> None:
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[0] < 1 or cos.shape[1] != D // 2:
        raise ValueError(f"{name}: rotary tables are [positions, D / 2]")
    if cos.device != like.device or sin.device != like.device:
        raise ValueError(f"{name}: all tensors are on one device")


def _cuda_only(name: str, cache: PagedCache) -> None:
    if cache.k.shape[3] not in HEAD_DIMS:
        raise ValueError(f"{name}: CUDA kernels exist for a head dimension of 64 or 128")
    if any(t is not None and t.data_ptr() % 16 for t in cache):
        raise ValueError(f"{name}: rows and scales of the cache start on 16-byte boundaries")


def _on_16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _pool_args(cache: PagedCache):
    return tuple(native.ptr(t) for t in cache)


def _log_page(cache: PagedCache) -> int:
    return cache.k.shape[2].bit_length() - 1


# --------------------------------------------------------------------------- plain forms
def _hold(x, dtype):
    """fp rows as they are held: (rows, scales)."""
    if dtype not in LARGEST:
        return x.to(dtype), None
    s = (x.abs().amax(-1) * torch.tensor(1.0 / LARGEST[dtype], dtype=torch.float32).to(x)).clamp_min(LEAST_SCALE)
    y = x / s[..., None]
    return (torch.round(y).to(dtype) if dtype == torch.int8 else y.float().to(dtype)), s.float()


def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _pages_of(cache, table, seq, pos):
    """Pages and rows of (sequence, position), and which of them are there."""
    page = cache.k.shape[2]
    ok = (seq >= 0) & (seq < table.shape[0]) & (pos >= 0) & (pos < table.shape[1] * page)
    s, t = torch.where(ok, seq, 0).long(), torch.where(ok, pos, 0).long()
    at = table[s, t // page].long()
    ok = ok & (at >= 0) & (at < cache.k.shape[0])
    return torch.where(ok, at, 0), t % page, ok


def _bytes(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _put_reference(cache, table, k, v, seq, pos, ok):
    at, off, there = _pages_of(cache, table, seq, pos)
    keep = there & ok
    at, off = at[keep], off[keep]
    for x, rows, scales in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        y, s = _hold(x[keep], rows.dtype)
        _bytes(rows)[at, :, off] = _bytes(y)
        if scales is not None:
            scales[at, :, off] = s


def _get_reference(cache, table, T, dt):
    """Tokens 0 .. T of every sequence [B, T, KVH, D] in ``dt`` (K, V), and which are there [B, T]."""
    B = table.shape[0]
    t = torch.arange(T, device=table.device)
    at, off, ok = _pages_of(cache, table, torch.arange(B, device=table.device)[:, None].expand(B, T), t.expand(B, T))
    out = []
    for rows, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = _bytes(rows)[at, :, off].view(rows.dtype).to(dt)
        out.append(x if scales is None else x * scales[at, :, off][..., None].to(dt))
    return out[0], out[1], ok


# --------------------------------------------------------------------------- writing and reading
def paged_append(k, v, cache: PagedCache, table, seq, pos, cos=None, sin=None) -> None:
    """Rows ``k``, ``v`` [M, KV heads, D] (a slice of the packed projection, for one) into the pages of sequence ``seq`` [M] at position
    ``pos`` [M] (int32). With ``cos``, ``sin`` [positions, D / 2] K is rotated to its position first; it is not rounded in between. A
    row whose sequence is none of the table's (-1: padding), or whose position lies behind the table's pages, or behind the rotary
    tables, is left out. No two rows go to one place."""
    if (cos is None) != (sin is None):
        raise ValueError("paged_append: cos and sin, or neither")
    if native.host is not None:
        if native.host.paged_append(k, v, *cache, table, seq, pos, cos, sin):
            native.bump()
            return
    _check_cache("paged_append", cache, table)
    pages, KVH, page, D = cache.k.shape
    if k.dim() != 3 or k.shape != v.shape or tuple(k.shape[1:]) != (KVH, D) or k.dtype != v.dtype or not k.dtype.is_floating_point:
        raise ValueError("paged_append: k and v are [M, KV heads, D] of one floating type")
    M = k.shape[0]
    _check_int32("paged_append", M, k, seq=seq, pos=pos)
    if k.device != cache.k.device or v.device != k.device:
        raise ValueError("paged_append: all tensors are on one device")
    if cos is not None:
        _check_tables("paged_append", cos, sin, D, k)
    if not k.is_cuda:
        dt = _work_dtype(k)
        x, ok = k.to(dt), torch.ones_like(seq, dtype=torch.bool)
        if cos is not None:
            ok = pos < cos.shape[0]
            t = pos.long().clamp(0, cos.shape[0] - 1)
            x = _rotate(x, cos[t][:, None].to(dt), sin[t][:, None].to(dt))
        _put_reference(cache, table, x, v.to(dt), seq, pos, ok)
        return
    F._bf16(k, v)
    _cuda_only("paged_append", cache)
    if cos is not None and (cos.dtype != torch.float32 or sin.dtype != torch.float32):
        raise TypeError("paged_append: rotary tables are float32")
    if M == 0 or table.shape[0] == 0:
        return
    with torch.cuda.device(k.device):
        k, v = (t if t.stride()[1:] == (D, 1) and (M == 1 or t.stride(0) % 8 == 0 and t.stride(0) > 0) and t.data_ptr() % 16 == 0
                else t.clone(memory_format=torch.contiguous_format) for t in (k, v))
        if cos is not None:
            cos, sin = _on_16(cos), _on_16(sin)
        table, seq, pos = table.contiguous(), seq.contiguous(), pos.contiguous()
        ldk, ldv = (t.stride(0) if M > 1 else KVH * D for t in (k, v))
        native.check(F._lib().b200_paged_append(
            native.ptr(k), native.ptr(v), *_pool_args(cache), native.ptr(table), native.ptr(seq), native.ptr(pos), native.ptr(cos),
            native.ptr(sin), 0 if cos is None else cos.shape[0], _ll(M), _ll(ldk), _ll(ldv), table.shape[0], table.shape[1], pages, KVH,
            _log_page(cache), D, HELD[cache.k.dtype], native.stream_ptr()), "paged_append")
    native.bump()


def paged_read(cache: PagedCache, table, lens, kcache, vcache, start=None):
    """Tokens ``start[b]`` (None: 0) up to ``lens[b]`` (int32 [B]) of every sequence into rows 0, 1, ... of ``kcache``, ``vcache``
    [B, KV heads, Tmax, D], as the values that they stand for, rounded once. Rows behind them, rows of tokens whose page is not there and
    tokens that Tmax has no room for are left as they are. Returns the two."""
    if native.host is not None:
        if native.host.paged_read(*cache, table, lens, kcache, vcache, start):
            native.bump()
            return kcache, vcache
    _check_cache("paged_read", cache, table)
    pages, KVH, page, D = cache.k.shape
    B = table.shape[0]
    if kcache.dim() != 4 or kcache.shape != vcache.shape or kcache.shape[0] != B or kcache.shape[1] != KVH or kcache.shape[3] != D:
        raise ValueError("paged_read: kcache and vcache are [B, KV heads, Tmax, D]")
    if kcache.dtype != vcache.dtype or not kcache.dtype.is_floating_point:
        raise TypeError("paged_read: kcache and vcache are of one floating type")
    if any(t.device != cache.k.device for t in (kcache, vcache)):
        raise ValueError("paged_read: all tensors are on one device")
    _check_int32("paged_read", B, cache.k, lens=lens, **({} if start is None else dict(start=start)))
    Tmax = kcache.shape[2]
    if not kcache.is_cuda:
        T = table.shape[1] * page
        first = torch.zeros_like(lens) if start is None else start.clamp_min(0)
        dt = _work_dtype(kcache)
        kx, vx, ok = _get_reference(cache, table, T, dt)
        t = first[:, None].long() + torch.arange(Tmax)
        there = (t < lens[:, None].long().clamp_max(T))
        t = t.clamp_max(T - 1)
        there &= torch.gather(ok, 1, t)
        for dst, x in ((kcache, kx), (vcache, vx)):
            x = torch.gather(x, 1, t[:, :, None, None].expand(B, Tmax, KVH, D)).transpose(1, 2).to(dst.dtype)
            dst.copy_(torch.where(there[:, None, :, None], x, dst))
        return kcache, vcache
    F._bf16(kcache, vcache)
    _cuda_only("paged_read", cache)
    if not (kcache.is_contiguous() and vcache.is_contiguous()) or (kcache.data_ptr() | vcache.data_ptr()) % 16:
        raise ValueError("paged_read: kcache and vcache are contiguous and start on a 16-byte boundary")
    if B == 0 or Tmax == 0:
        return kcache, vcache
    if B > 32767 or KVH > 65535:
        raise ValueError("paged_read: at most 32767 sequences and 65535 KV heads a call")
    with torch.cuda.device(kcache.device):
        table, lens, start = table.contiguous(), lens.contiguous(), None if start is None else start.contiguous()
        native.check(F._lib().b200_paged_read(
            *_pool_args(cache), native.ptr(table), native.ptr(start), native.ptr(lens), native.ptr(kcache), native.ptr(vcache), Tmax, B,
            table.shape[1], pages, KVH, _log_page(cache), D, HELD[cache.k.dtype], native.stream_ptr()), "paged_read")
    native.bump()
    return kcache, vcache


# --------------------------------------------------------------------------- attention of one new token
def paged_attn_append(kqv, cache: PagedCache, table, lens, QH: int, KVH: int, cos, sin, *, scale: float | None = None,
                      softcap: float = 0.0, slopes=None):
    """Attention of one new token of each of ``B`` sequences over its pages. ``kqv`` [B, (2 KVH + QH) * D]: the packed projection
    K | Q | V, un-rotated; ``lens`` int32 [B]: cached tokens, the new one's position; ``cos``, ``sin`` fp32 [positions, D / 2].

    K (rotated) and V of the new token are written to its page, and it sees the cached tokens and itself, its own row as it is held. One
    that would stand behind the table's pages or the rotary tables, or whose page is not there, is not kept and not seen. A sequence of
    fewer than 0 tokens is none (a padded batch): nothing is written for it, and its result is 0, as it is where nothing is seen.
    ``softcap`` > 0 caps the scores (c tanh(s / c)); ``slopes`` fp32 [QH]: scores lose slope[head] * distance. Pages that are written
    belong to one sequence. Elements of Q go to the products off by at most 2^-17 of themselves over bf16 rows, 2^-30 of their head's
    largest over int8 rows, 2^-23 of themselves or 2^-35 of the largest, whichever is more, over e4m3 rows; weights off by 2^-17 of
    themselves over bf16 rows, else 2^-23 of themselves or 2^-39 of the largest. Returns [B, QH, D]."""
    if native.host is not None:
        out = native.host.paged_attn(kqv, *cache, table, lens, QH, KVH, cos, sin, 0.0 if scale is None else scale or -1.0, softcap, slopes)
        if out is not None:
            native.bump()
            return out
    _check_cache("paged_attn_append", cache, table)
    pages, heads, page, D = cache.k.shape
    B = table.shape[0]
    if KVH != heads or QH <= 0 or QH % KVH != 0 or kqv.dim() != 2 or tuple(kqv.shape) != (B, (2 * KVH + QH) * D):
        raise ValueError("paged_attn_append: sizes of kqv, cache and table do not go together")
    if not kqv.dtype.is_floating_point or kqv.device != cache.k.device:
        raise ValueError("paged_attn_append: all tensors are on one device, kqv in floating point")
    _check_int32("paged_attn_append", B, kqv, lens=lens)
    _check_tables("paged_attn_append", cos, sin, D, kqv)
    _modifier("paged_attn_append", QH, softcap, slopes, kqv.device)
    scale = _scale(scale, D)
    if not kqv.is_cuda:
        return _attn_reference(kqv, cache, table, lens, QH, KVH, cos, sin, scale, softcap, slopes)
    F._bf16(kqv)
    _cuda_only("paged_attn_append", cache)
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("paged_attn_append: rotary tables are float32")
    if B > 65535 or KVH * ((QH // KVH + 3) // 4) > 65535:
        raise ValueError("paged_attn_append: at most 65535 sequences, and KV heads (once for every 4 query heads), a call")
    with torch.cuda.device(kqv.device):
        out = torch.empty((B, QH, D), dtype=torch.bfloat16, device=kqv.device)
        if B == 0:
            return out
        if kqv.stride(1) != 1 or (B > 1 and (kqv.stride(0) % 8 or kqv.stride(0) <= 0)) or kqv.data_ptr() % 16:
            kqv = kqv.clone(memory_format=torch.contiguous_format)
        cos, sin, table, lens = _on_16(cos), _on_16(sin), table.contiguous(), lens.contiguous()
        slopes = slopes if slopes is None else slopes.contiguous()
        lib = F._lib()
        lib.b200_paged_attn_workspace.restype = _ll
        size = lib.b200_paged_attn_workspace(B, QH, KVH, table.shape[1], _log_page(cache), D)
        ws = torch.empty(size, dtype=torch.uint8, device=kqv.device) if size else None
        native.check(lib.b200_paged_attn_append(
            native.ptr(kqv), *_pool_args(cache), native.ptr(table), native.ptr(lens), native.ptr(cos), native.ptr(sin), native.ptr(slopes),
            native.ptr(out), native.ptr(ws), cos.shape[0], _ll(kqv.stride(0) if B > 1 else kqv.shape[1]), B, table.shape[1], pages, QH, KVH,
            _log_page(cache), D, HELD[cache.k.dtype], _f(scale), _f(softcap), native.stream_ptr()), "paged_attn_append")
    native.bump()
    return out


def _attn_reference(kqv, cache, table, lens, QH, KVH, cos, sin, scale, softcap, slopes):
    B, D = table.shape[0], cache.k.shape[3]
    dt = _work_dtype(kqv)
    T = table.shape[1] * cache.k.shape[2]
    k, q, v = kqv.to(dt).split([KVH * D, QH * D, KVH * D], dim=1)
    pos = lens.long().clamp(0, cos.shape[0] - 1)
    c, s = (x.to(dt)[pos][:, None] for x in (cos, sin))
    q = _rotate(q.reshape(B, QH, D), c, s)
    seq = torch.arange(B)
    _put_reference(cache, table, _rotate(k.reshape(B, KVH, D), c, s), v.reshape(B, KVH, D), seq, lens, (lens >= 0) & (lens < cos.shape[0]))
    kx, vx, ok = _get_reference(cache, table, T, dt)
    t = torch.arange(T)
    upto = torch.where(lens < cos.shape[0], lens, lens - 1)              # a token that is not kept is not seen
    seen = ok & (t <= upto[:, None]) & (lens >= 0)[:, None]
    kx, vx = (torch.where(seen[:, :, None, None], x, torch.zeros((), dtype=dt)) for x in (kx, vx))
    x, _ = _scores_reference(q[:, None], kx, seen[:, None], scale, softcap, slopes, (lens[:, None] - t).abs()[:, None, None])
    p, _ = _softmax_reference(x)
    return torch.einsum("bhts,bshd->bthd", p, vx.repeat_interleave(QH // KVH, dim=2))[:, 0].to(kqv.dtype).contiguous()
