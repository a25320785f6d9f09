"""Attention beyond one causal sequence per row: packed documents, prefixes and padding (span masks), scores that are capped by
a tanh or get a bias that grows with the distance, and trees of drafted tokens over a KV cache.

As in ``functional``, every function has two bodies: CUDA tensors go to the hand-written sm_100a kernels (bf16 storage, fp32
scores, softmax statistics and sums), CPU tensors take a plain torch restatement (fp32, or fp64 for fp64 inputs).

Training and scoring:

    mask = span_mask(B, T, device, docs=ids)                   # once per batch, for all layers
    o, lse = span_attn_fwd(q, k, v, mask, softcap=50.0)
    dq, dk, dv = span_attn_bwd(dout, q, k, v, o, lse, mask, softcap=50.0)

Serving, ``n`` drafted tokens of each sequence (n = 1: the decoded token):

    o = tree_attn_append(kqv, kcache, vcache, lens, tree_mask(parents, device), QH, KVH, cos, sin, softcap=50.0)

A cap c makes c tanh(s / c) of every scaled score s; a bias takes slope[head] * |query position - key position| from it.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import functional as F
from . import native

_f = ctypes.c_float
_i = ctypes.c_int
# Caps and scales that the kernels' arithmetic has room for: a cap's square, and the quotient of the two, are fp32 numbers.
LEAST, MOST = 1e-18, 1e18


# --------------------------------------------------------------------------- span masks
class SpanMask:
    """Which keys each query of a [B, T] batch sees: positions [lo, hi) per query, and (CUDA) the tables of tiles of 128 tokens
    that the kernels walk by. Made by ``span_mask`` or ``SpanMask.from_spans``; one serves any number of layers and heads."""

    def __init__(self, buf: torch.Tensor, B: int, T: int):
        # CUDA: [B, nt, 4] key tiles of every query tile, [B, nt, 2] query tiles of every key tile, the spans [B, T, 2] (lo, hi), and
        # the orders, those with most to do first: [B, nt] query tiles, [B, (nt + 1) / 2] pairs of them, [B, nt] key tiles. What has the
        # wider entries comes first. CPU: the spans alone.
        self.buf, self.B, self.T = buf, B, T

    @property
    def device(self):
        return self.buf.device

    @property
    def spans(self) -> torch.Tensor:
        """int32 [B, T, 2]: lo, hi."""
        n = self.B * self.T * 2
        at = 6 * self.B * ((self.T + 127) // 128) if self.buf.is_cuda else 0
        return self.buf[at:at + n].view(self.B, self.T, 2)

    def _ptrs(self, b0: int = 0):
        """Addresses of spans, query-tile and key-tile table from batch element ``b0`` on (CUDA)."""
        nt, p = (self.T + 127) // 128, self.buf.data_ptr()
        return (native.c_void_p(p + 4 * (6 * self.B * nt + 2 * b0 * self.T)), native.c_void_p(p + 16 * b0 * nt),
                native.c_void_p(p + 4 * (4 * self.B * nt + 2 * b0 * nt)))

    def _orders(self, b0: int = 0):
        """Addresses of the orders of query tiles and of key tiles (CUDA); those of pairs stand between them."""
        nt = (self.T + 127) // 128
        pairs, p = (nt + 1) // 2, self.buf.data_ptr() + 4 * self.B * (6 * nt + 2 * self.T)
        return native.c_void_p(p + 4 * b0 * nt), native.c_void_p(p + 4 * (self.B * (nt + pairs) + b0 * nt))

    @classmethod
    def from_spans(cls, lo: torch.Tensor, hi: torch.Tensor) -> "SpanMask":
        """Query t of row b sees keys lo[b, t] <= s < hi[b, t] (int32 [B, T]; cut to [0, T), nothing where hi <= lo)."""
        if lo.dim() != 2 or lo.shape != hi.shape or lo.dtype != torch.int32 or hi.dtype != torch.int32 or lo.device != hi.device:
            raise ValueError("SpanMask.from_spans: lo and hi are int32 [B, T] on one device")
        return _make_mask(*lo.shape, lo.device, lo=lo.contiguous(), hi=hi.contiguous())

    def dense(self) -> torch.Tensor:
        """bool [B, T, T]: query t (second) sees key s (third). For verification and small sizes."""
        s, spans = torch.arange(self.T, device=self.device), self.spans
        return (s >= spans[..., :1]) & (s < spans[..., 1:])


def _make_mask(B, T, device, docs=None, prefix=None, valid_len=None, lo=None, hi=None) -> SpanMask:
    if torch.device(device).type != "cuda":
        if lo is None:
            lo, hi = _spans_reference(B, T, docs, prefix, valid_len)
        lo, hi = lo.clamp_min(0), hi.clamp_max(T)
        none = hi <= lo
        return SpanMask(torch.stack([lo.masked_fill(none, 0), hi.masked_fill(none, 0)], -1).to(torch.int32).reshape(-1), B, T)
    nt = (T + 127) // 128
    mask = SpanMask(torch.empty(B * (8 * nt + (nt + 1) // 2 + 2 * T), dtype=torch.int32, device=device), B, T)
    native.check(F._lib().b200_span_mask(native.ptr(docs), native.ptr(prefix), native.ptr(valid_len), native.ptr(lo), native.ptr(hi),
                                         *mask._ptrs(), mask._orders()[0], B, T, native.stream_ptr()), "span_mask")
    native.bump()
    return mask


def _spans_reference(B, T, docs, prefix, valid_len):
    t = torch.arange(T)[None].expand(B, T)
    docs = torch.zeros(B, T, dtype=torch.int32) if docs is None else docs
    start = torch.ones(B, T, dtype=torch.bool)
    start[:, 1:] = docs[:, 1:] != docs[:, :-1]
    lo = torch.cummax(torch.where(start, t, 0), 1).values
    hi = t + 1
    if prefix is not None:
        plain = torch.cummax(torch.where(prefix, -1, t), 1).values           # the last token that is not flagged
        stop = torch.where(start | ~prefix, t, T)
        nxt = torch.full((B, T), T)
        nxt[:, :-1] = torch.flip(torch.cummin(torch.flip(stop[:, 1:], [1]), 1).values, [1])
        hi = torch.where(prefix & (plain < lo), nxt, hi)
    vlen = torch.full((B, 1), T) if valid_len is None else valid_len[:, None].long().clamp(0, T)
    hi = torch.minimum(hi, vlen)
    return lo, torch.where((docs < 0) | (t >= vlen), torch.zeros_like(hi), hi)


def _is_device(x: torch.Tensor, device) -> bool:
    """Whether ``x`` is on ``device``: a GPU without a number is the current one."""
    d = torch.device(device)
    return x.device.type == d.type and (d.type != "cuda" or x.device.index == (torch.cuda.current_device() if d.index is None else d.index))


def span_mask(B: int, T: int, device, docs=None, prefix=None, valid_len=None) -> SpanMask:
    """Mask of ``B`` rows of ``T`` tokens. ``docs`` int32 [B, T]: which document a token belongs to; a change of the number
    starts the next one, a negative one is padding, which sees nothing and is not seen. ``prefix`` bool [B, T]: a document's leading
    flagged tokens see one another whichever comes first; every other token sees its document up to itself. ``valid_len``
    int32 [B]: tokens from there on are padding too. Without any of them: plain causal rows."""
    if native.host is not None:
        buf = native.host.span_mask(B, T, docs, prefix, valid_len)      # (on the current device, as docs, prefix and valid_len are)
        if buf is not None and (device == "cuda" or _is_device(buf, device)):
            native.bump()
            return SpanMask(buf, B, T)
    if B < 0 or T < 0:
        raise ValueError("span_mask: negative size")
    for name, x, dt, shape in (("docs", docs, torch.int32, (B, T)), ("prefix", prefix, torch.bool, (B, T)),
                               ("valid_len", valid_len, torch.int32, (B,))):
        if x is not None and (x.dtype != dt or tuple(x.shape) != shape):
            raise ValueError(f"span_mask: {name} is {dt} {list(shape)}")
        if x is not None and not _is_device(x, device):
            raise ValueError(f"span_mask: {name} is not on {device}")
    if T > 512000:
        raise ValueError("span_mask: more than 512000 tokens in a row")
    docs, prefix, valid_len = (x if x is None else x.contiguous() for x in (docs, prefix, valid_len))
    return _make_mask(B, T, device, docs, prefix, valid_len)


# --------------------------------------------------------------------------- span attention
def _heads(name: str, q, k, v):
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"{name}: q is [B, T, query heads, D], k and v are [B, T, KV heads, D]")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2] != 0:
        raise ValueError(f"{name}: the query heads are a multiple of the KV heads")
    _same_device(name, q, k, v)


def _same_device(name: str, first, *others) -> None:
    if any(t.device != first.device for t in others):
        raise ValueError(f"{name}: all tensors are on one device")


def _modifier(name: str, q_heads: int, softcap: float, slopes, device) -> None:
    if softcap != 0.0 and not LEAST <= softcap <= MOST:
        raise ValueError(f"{name}: softcap is 0 (none) or a number from {LEAST} to {MOST}")
    if slopes is None:
        return
    if softcap > 0.0:
        raise ValueError(f"{name}: scores are capped or biased, not both")
    if slopes.dtype != torch.float32 or tuple(slopes.shape) != (q_heads,) or slopes.device != device:
        raise ValueError(f"{name}: slopes is float32 [query heads] on the device of q")


def _check_mask(name: str, mask: SpanMask, q) -> None:
    if not isinstance(mask, SpanMask):
        raise TypeError(f"{name}: mask is a SpanMask")
    if (mask.B, mask.T) != tuple(q.shape[:2]) or mask.device != q.device:
        raise ValueError(f"{name}: the mask is of {mask.B} x {mask.T} tokens on {mask.device}, "
                         f"q of {q.shape[0]} x {q.shape[1]} on {q.device}")


def _scale(scale, D: int) -> float:
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not LEAST <= scale <= MOST:
        raise ValueError(f"attention: scale is a number from {LEAST} to {MOST}")
    return scale


def _tile_view(t: torch.Tensor) -> torch.Tensor:
    """``t`` [B, T, heads, D] if tiles can be copied from it as it lies (16-byte rows), else a copy."""
    s, n = t.stride(), t.shape
    ok = s[3] == 1 and t.data_ptr() % 16 == 0 and all(n[i] == 1 or (s[i] % 8 == 0 and s[i] > 0) for i in range(3))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _strides3(t: torch.Tensor) -> list[int]:
    """(batch, token, head) strides; of a dimension of one, which is never stepped along, one that a tile copy can have."""
    return [t.stride(i) if t.shape[i] > 1 else 16 for i in range(3)]


def _work_dtype(x):
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def _scores_reference(q, k, mask_bool, scale, softcap, slopes, dist):
    """(modified scores [B, QH, n, S] with -inf where ``mask_bool`` [B, n, S] is False, 1 - tanh^2 or None)."""
    dt = _work_dtype(q)
    kx = k.to(dt).repeat_interleave(q.shape[2] // k.shape[2], dim=2)
    x = torch.einsum("bthd,bshd->bhts", q.to(dt), kx) * scale
    slope = None
    if softcap > 0.0:
        th = torch.tanh(x / softcap)
        x, slope = softcap * th, 1 - th * th
    if slopes is not None:
        x = x - slopes.to(dt)[None, :, None, None] * dist.to(dt)
    return x.masked_fill(~mask_bool[:, None], float("-inf")), slope


def _softmax_reference(x):
    m = x.amax(-1, keepdim=True) if x.shape[-1] else x.new_full((*x.shape[:-1], 1), float("-inf"))
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total), (m + torch.log(total))[..., 0]


def _span_reference(q, k, v, mask, scale, softcap, slopes):
    T = q.shape[1]
    t = torch.arange(T, device=q.device)
    x, slope = _scores_reference(q, k, mask.dense(), scale, softcap, slopes, (t[:, None] - t[None, :]).abs())
    p, lse = _softmax_reference(x)
    vx = v.to(p.dtype).repeat_interleave(q.shape[2] // k.shape[2], dim=2)
    return torch.einsum("bhts,bshd->bthd", p, vx), lse, p, slope


def span_attn_fwd(q, k, v, mask: SpanMask, *, scale: float | None = None, softcap: float = 0.0, slopes=None):
    """Attention of q [B, T, QH, D] over k, v [B, T, KVH, D] (already rotated; any strides) under ``mask``. CUDA: bf16, D 64 or
    128. Returns (o [B, T, QH, D] contiguous, lse [B, QH, T] fp32); a query that sees nothing gets zeros and -inf.

    For every two neighbouring tiles of 128 queries the tiles of 128 keys from the first to the last that one of them sees are read, gaps
    between spans included. All that is read has to be finite, padding too: a value that is masked goes through the tensor core with
    weight 0. Weights are rounded to bf16 for the tensor core (sums and statistics are fp32): with the result's own rounding 1.8 to
    2.2e-3 of the result, root mean square."""
    if native.host is not None and type(mask) is SpanMask:
        r = native.host.span_fwd(q, k, v, mask.buf, mask.B, mask.T, 0.0 if scale is None else scale or -1.0, softcap, slopes)
        if r is not None:
            native.bump()
            return r
    _heads("span_attn_fwd", q, k, v)
    _check_mask("span_attn_fwd", mask, q)
    B, T, QH, D = q.shape
    KVH = k.shape[2]
    _modifier("span_attn_fwd", QH, softcap, slopes, q.device)
    scale = _scale(scale, D)
    if not q.is_cuda:
        o, lse, _, _ = _span_reference(q, k, v, mask, scale, softcap, slopes)
        return o.to(q.dtype).contiguous(), lse
    F._bf16(q, k, v)
    if D not in (64, 128):
        raise ValueError("span_attn_fwd: CUDA kernels exist for a head dimension of 64 or 128")
    q, k, v = _tile_view(q), _tile_view(k), _tile_view(v)
    o = torch.empty((B, T, QH, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, QH, T), dtype=torch.float32, device=q.device)
    arr = (ctypes.c_longlong * 12)(*_strides3(q), *_strides3(k), *_strides3(v), *_strides3(o))
    slopes = slopes if slopes is None else slopes.contiguous()
    native.check(F._lib().b200_flash_fwd_span(native.ptr(q), native.ptr(k), native.ptr(v), native.ptr(o), native.ptr(lse),
                                              *mask._ptrs()[:2], mask._orders()[0], arr, B, T, QH, KVH, D, _f(scale),
                                              _f(softcap), native.ptr(slopes), native.stream_ptr()), "flash_fwd_span")
    native.bump()
    return o, lse


def span_attn_bwd(dout, q, k, v, o, lse, mask: SpanMask, *, scale: float | None = None, softcap: float = 0.0, slopes=None, out=None,
                  unrotate=None, delta=None):
    """Gradients (dq, dk, dv) of ``span_attn_fwd`` with its results ``o``, ``lse``. ``out``: three [B, T, heads, D] views to
    write into; ``unrotate`` = (cos, sin) tables [>= T, D / 2]: dq and dk leave as gradients of the un-rotated q and k; ``delta``
    [B, QH, T] fp32, sum over D of dout * o, where the caller has it (``gemm.gemm_delta``). The
    kernels keep dS^T of as many batch elements or KV heads at a time as ``functional.FLASH_DQ_GEMM_MAX_BYTES`` holds, of one KV
    head at least, whatever its spans: 2 T^2 bytes for each of its query heads. That is where one GPU ends: 34 GB at 65536 tokens and four
    of them, 137 GB at 131072. Deterministic: no atomics.

    All inputs have to be finite, also where nothing is seen. dq and dk are 2.6 to 3.3e-3 (root mean square) from exact ones, dv
    2.3e-3, where the rounding of a bf16 result alone is 1.7e-3: P and dS are bf16 for the tensor core, and ``delta`` comes from an ``o``
    that is bf16."""
    if native.host is not None and type(mask) is SpanMask and out is None and unrotate is None and delta is None:
        r = native.host.span_bwd(dout, q, k, v, o, lse, mask.buf, mask.B, mask.T, 0.0 if scale is None else scale or -1.0, softcap, slopes,
                                 F.FLASH_DQ_GEMM_MAX_BYTES)
        if r is not None:
            native.bump(3)
            return r
    _heads("span_attn_bwd", q, k, v)
    _check_mask("span_attn_bwd", mask, q)
    B, T, QH, D = q.shape
    KVH = k.shape[2]
    if dout.shape != q.shape or o.shape != q.shape or tuple(lse.shape) != (B, QH, T):
        raise ValueError("span_attn_bwd: dout and o are like q, lse is [B, query heads, T]")
    _modifier("span_attn_bwd", QH, softcap, slopes, q.device)
    if unrotate is not None and any(x.dim() != 2 or x.shape[0] < T or x.shape[1] != D // 2 for x in unrotate):
        raise ValueError("span_attn_bwd: rotary tables are [>= T, D / 2]")
    if out is not None and [x.shape for x in out] != [q.shape, k.shape, v.shape]:
        raise ValueError("span_attn_bwd: out has the shapes of q, k and v")
    if delta is not None and tuple(delta.shape) != (B, QH, T):
        raise ValueError("span_attn_bwd: delta is [B, query heads, T]")
    _same_device("span_attn_bwd", q, dout, o, lse, *(unrotate or ()), *(out or ()), *(() if delta is None else (delta,)))
    scale = _scale(scale, D)
    if not q.is_cuda:
        return _span_bwd_reference(dout, q, k, v, o, mask, scale, softcap, slopes, out, unrotate)
    F._bf16(dout, q, k, v, o)
    if D not in (64, 128):
        raise ValueError("span_attn_bwd: CUDA kernels exist for a head dimension of 64 or 128")
    if any(x.dtype != torch.float32 for x in (lse, *(unrotate or ()))):
        raise TypeError("span_attn_bwd: lse and the rotary tables are float32")
    q, k, v, dout, o = (_tile_view(t) for t in (q, k, v, dout, o))
    lse = lse.contiguous()
    if out is None:
        dq = torch.empty((B, T, QH, D), dtype=q.dtype, device=q.device)
        dk, dv = torch.empty((B, T, KVH, D), dtype=q.dtype, device=q.device), torch.empty((B, T, KVH, D), dtype=q.dtype, device=q.device)
    else:
        dq, dk, dv = out
        F._bf16(dq, dk, dv)
        if any(_tile_view(t) is not t for t in out):
            raise ValueError("span_attn_bwd: out needs rows on 16-byte boundaries")
    if B == 0 or T == 0:
        return dq, dk, dv
    if delta is None:
        delta = F.flash_delta(o, dout, torch.empty((B, QH, T), dtype=torch.float32, device=q.device))
    elif delta.dtype != torch.float32 or not delta.is_contiguous():
        raise ValueError("span_attn_bwd: delta is float32 [B, query heads, T], contiguous")
    ucos = usin = None
    if unrotate is not None:
        from .gemm import rope_tables_transposed
        ucos, usin = rope_tables_transposed(unrotate[0].contiguous(), unrotate[1].contiguous())[:2]
    uld = ucos.shape[1] if ucos is not None else 0
    slopes = slopes if slopes is None else slopes.contiguous()
    R = QH // KVH
    arr = (ctypes.c_longlong * 21)(*_strides3(q), *_strides3(k), *_strides3(v), *_strides3(dout), *_strides3(dq), *_strides3(dk),
                                   *_strides3(dv))
    tp = (T + 127) // 128 * 128
    bc = F._ds_batch_chunk(B, QH, T)
    if bc >= 1:
        ws = torch.empty(bc * QH * tp * tp, dtype=torch.bfloat16, device=q.device)
        chunks = [(b0, min(b0 + bc, B), 0, KVH) for b0 in range(0, B, bc)]
    else:                                                  # KV heads of one batch element, with their query heads
        kc = max(1, min(KVH, F._ds_batch_chunk(KVH, R, T)))
        ws = torch.empty(kc * R * tp * tp, dtype=torch.bfloat16, device=q.device)
        chunks = [(b0, b0 + 1, g0, min(g0 + kc, KVH)) for b0 in range(B) for g0 in range(0, KVH, kc)]
    for b0, b1, g0, g1 in chunks:                          # slices along batch and heads keep every stride
        def qs(t):
            return native.ptr(t[b0:b1, :, g0 * R:g1 * R])

        def ks(t):
            return native.ptr(t[b0:b1, :, g0:g1])

        def rows(t):
            return native.ptr(t[b0:b1, g0 * R:g1 * R])     # contiguous: head slices only come with one batch element
        native.check(F._lib().b200_flash_bwd_span(
            qs(q), ks(k), ks(v), qs(dout), rows(lse), rows(delta), qs(dq), ks(dk), ks(dv), *mask._ptrs(b0), mask._orders(b0)[1],
            mask._orders(b0)[0], arr, b1 - b0, T, (g1 - g0) * R, g1 - g0, D, _f(scale), _f(softcap),
            native.ptr(slopes if slopes is None else slopes[g0 * R:g1 * R]), native.ptr(ws), native.ptr(ucos), native.ptr(usin), uld,
            native.stream_ptr()), "flash_bwd_span")
    native.bump(2 * len(chunks))
    return dq, dk, dv


def _span_bwd_reference(dout, q, k, v, o, mask, scale, softcap, slopes, out, unrotate):
    R = q.shape[2] // k.shape[2]
    B, T, KVH, D = k.shape
    _, _, p, slope = _span_reference(q, k, v, mask, scale, softcap, slopes)
    dt = p.dtype
    do = dout.to(dt)
    vx, kx = (x.to(dt).repeat_interleave(R, dim=2) for x in (v, k))
    dp = torch.einsum("bthd,bshd->bhts", do, vx)
    delta = (do * o.to(dt)).sum(-1).permute(0, 2, 1)
    ds = p * (dp - delta[..., None]) * scale
    if slope is not None:
        ds = ds * slope
    dq = torch.einsum("bhts,bshd->bthd", ds, kx)
    dk = torch.einsum("bhts,bthd->bshd", ds, q.to(dt)).reshape(B, T, KVH, R, D).sum(3)
    dv = torch.einsum("bhts,bthd->bshd", p, do).reshape(B, T, KVH, R, D).sum(3)
    if unrotate is not None:
        c, s = (x[:T].to(dt)[None, :, None] for x in unrotate)

        def back(x):
            y1, y2 = x[..., :D // 2], x[..., D // 2:]
            return torch.cat([y1 * c + y2 * s, y2 * c - y1 * s], -1)
        dq, dk = back(dq), back(dk)
    res = (dq.to(q.dtype), dk.to(q.dtype), dv.to(q.dtype))
    if out is not None:
        for dst, src in zip(out, res):
            dst.copy_(src)
        return tuple(out)
    return res


# --------------------------------------------------------------------------- drafted tokens over a KV cache
def tree_mask(parents, device) -> torch.Tensor:
    """int64 [B, n] masks for ``tree_attn_append`` from ``parents`` [B, n] (lists, or an integer tensor; read on the host):
    the draft that each draft continues, which stands before it in its row, or -1 for the cached text. Bit j of an entry is set
    when the draft sees draft j: its ancestors and itself. n is at most 64."""
    rows = parents.tolist() if isinstance(parents, torch.Tensor) else parents
    out = []
    for row in rows:
        if len(row) > 64:
            raise ValueError("tree_mask: more than 64 drafts")
        bits = []
        for i, par in enumerate(row):
            if not -1 <= par < i:
                raise ValueError("tree_mask: a draft's parent stands before it")
            bits.append((1 << i) | (bits[par] if par >= 0 else 0))
        out.append([x - (1 << 64) if x >> 63 else x for x in bits])
    return torch.tensor(out, dtype=torch.int64, device=device)


def tree_attn_append(kqv, kcache, vcache, lens, tree, QH: int, KVH: int, cos, sin, *, scale: float | None = None,
                     softcap: float = 0.0, slopes=None):
    """Attention of ``n`` drafted tokens of each of ``B`` sequences over their KV caches. ``kqv`` [B * n, (2 KVH + QH) * D]: the packed
    projection K | Q | V, un-rotated; ``kcache``, ``vcache`` [B, KVH, Tmax, D] (K rotated); ``lens`` int32 [B]: cached tokens;
    ``tree`` int64 [B, n] (``tree_mask``); ``cos``, ``sin`` fp32 [>= Tmax, D / 2].

    Draft i stands at position lens + its depth, sees the cached tokens and the drafts of its mask, and its K (rotated) and V
    are appended to the caches at lens + i. One that would stand behind the end of the cache is not kept, and no draft sees it, itself
    included: its own result is that of the cached tokens and of its ancestors that were kept. n = 1 with mask 1 is a decoded token.
    Weights are rounded to bf16 for the tensor core; the rotated Q goes in as two bf16 parts.
    Returns [B, n, QH, D]. A mask of 0 leaves the cached tokens alone; with none of them the result is 0. Cache rows from
    lens + n on may hold anything; the cached ones and all drafts have to be finite (a value that a draft does not see has weight 0)."""
    if native.host is not None:
        out = native.host.tree_attn(kqv, kcache, vcache, lens, tree, QH, KVH, cos, sin, 0.0 if scale is None else scale or -1.0, softcap,
                                    slopes)
        if out is not None:
            native.bump(3)
            return out
    if kcache.dim() != 4 or kcache.shape != vcache.shape or tree.dim() != 2 or kqv.dim() != 2:
        raise ValueError("tree_attn_append: caches are [B, KV heads, Tmax, D], tree is [B, n], kqv [B * n, columns]")
    B, n = tree.shape
    Tmax, D = kcache.shape[2:]
    if KVH <= 0 or QH <= 0 or QH % KVH != 0 or kcache.shape[:2] != (B, KVH) or tuple(kqv.shape) != (B * n, (2 * KVH + QH) * D):
        raise ValueError("tree_attn_append: sizes of kqv, caches and tree do not go together")
    if not 1 <= n <= 64 or QH // KVH > 128 or Tmax == 0:
        raise ValueError("tree_attn_append: 1 to 64 drafts, up to 128 query heads to a KV head, caches of at least one position")
    if tuple(lens.shape) != (B,) or lens.dtype != torch.int32 or tree.dtype != torch.int64:
        raise ValueError("tree_attn_append: lens is int32 [B], tree int64 [B, n]")
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[0] < Tmax or cos.shape[1] != D // 2:
        raise ValueError("tree_attn_append: rotary tables are [>= Tmax, D / 2]")
    if any(t.device != kqv.device for t in (kcache, vcache, lens, tree, cos, sin)):
        raise ValueError("tree_attn_append: all tensors are on one device")
    _modifier("tree_attn_append", QH, softcap, slopes, kqv.device)
    scale = _scale(scale, D)
    if not kqv.is_cuda:
        return _tree_reference(kqv, kcache, vcache, lens, tree, QH, KVH, cos, sin, scale, softcap, slopes)
    F._bf16(kqv, kcache, vcache)
    if D not in (64, 128):
        raise ValueError("tree_attn_append: CUDA kernels exist for a head dimension of 64 or 128")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError("tree_attn_append: rotary tables are float32")
    if not (kcache.is_contiguous() and vcache.is_contiguous()) or (kcache.data_ptr() | vcache.data_ptr()) % 16:
        raise ValueError("tree_attn_append: caches are contiguous and start on a 16-byte boundary")
    if kqv.stride(1) != 1 or (B * n > 1 and kqv.stride(0) % 8) or kqv.data_ptr() % 16:
        kqv = kqv.clone(memory_format=torch.contiguous_format)
    cos, sin, lens, tree = cos.contiguous(), sin.contiguous(), lens.contiguous(), tree.contiguous()
    cos, sin = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (cos, sin))
    slopes = slopes if slopes is None else slopes.contiguous()
    out = torch.empty((B, n, QH, D), dtype=torch.bfloat16, device=kqv.device)
    if B == 0:
        return out
    lib = F._lib()
    lib.b200_tree_attn_workspace.restype = ctypes.c_longlong
    ws = torch.empty(lib.b200_tree_attn_workspace(B, n, QH, KVH, Tmax, D), dtype=torch.uint8, device=kqv.device)
    native.check(lib.b200_tree_attn_append(
        native.ptr(kqv), native.ptr(kcache), native.ptr(vcache), native.ptr(out), native.ptr(lens), native.ptr(tree), native.ptr(cos),
        native.ptr(sin), native.ptr(slopes), native.ptr(ws), B, n, QH, KVH, Tmax, D, cos.shape[0],
        ctypes.c_longlong(kqv.stride(0) if B * n > 1 else kqv.shape[1]), _f(scale), _f(softcap), native.stream_ptr()), "tree_attn_append")
    native.bump(3)
    return out


def _tree_reference(kqv, kcache, vcache, lens, tree, QH, KVH, cos, sin, scale, softcap, slopes):
    B, n = tree.shape
    Tmax, D = kcache.shape[2:]
    j = torch.arange(n, device=kqv.device)
    sees = ((tree[:, :, None] >> j) & 1).bool()
    depth = (sees.sum(-1) - 1).clamp_min(0)
    lens = lens.long().clamp(0, Tmax)
    pos = lens[:, None] + depth
    dt = _work_dtype(kqv)
    k, q, v = kqv.to(dt).view(B, n, kqv.shape[1]).split([KVH * D, QH * D, KVH * D], dim=2)
    c, s = (x.to(dt)[pos.clamp_max(x.shape[0] - 1)][:, :, None] for x in (cos, sin))

    def rot(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1)
    q, k = rot(q.reshape(B, n, QH, D)), rot(k.reshape(B, n, KVH, D)).to(kcache.dtype)
    v = v.reshape(B, n, KVH, D)
    t = torch.arange(Tmax, device=kqv.device)
    for b in range(B):
        keep = min(n, Tmax - int(lens[b]))
        at = int(lens[b])
        kcache[b, :, at:at + keep] = k[b, :keep].transpose(0, 1)
        vcache[b, :, at:at + keep] = v[b, :keep].transpose(0, 1).to(vcache.dtype)
    off = t - lens[:, None]                                   # which draft a position is
    draft = off.clamp(0, n - 1)
    seen = (off < 0)[:, None] | (((off >= 0) & (off < n))[:, None] & torch.gather(sees, 2, draft[:, None].expand(B, n, Tmax)))
    kpos = torch.where(off < 0, t, lens[:, None] + torch.gather(depth, 1, draft))
    dist = (pos[:, :, None] - kpos[:, None, :]).abs()[:, None]
    used = (off < n)[:, None, :, None]                         # rows behind the drafts may hold anything
    kc, vc = (torch.where(used, x.to(dt), torch.zeros((), dtype=dt, device=x.device)).transpose(1, 2) for x in (kcache, vcache))
    x, _ = _scores_reference(q, kc, seen, scale, softcap, slopes, dist)
    p, _ = _softmax_reference(x)
    return torch.einsum("bhts,bshd->bthd", p, vc.repeat_interleave(QH // KVH, dim=2)).to(kqv.dtype).contiguous()
