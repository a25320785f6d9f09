"""What the paged cache and the verification of drafted tokens are measured on.

Four operators, with sizes of the benchmark configurations (125M: 12 / 4 heads of 64, context 1024; 1.3B: 16 / 4 heads of 128,
context 2048; 7B: 32 / 8 heads of 128, context 4096; vocabulary 32000) and their neighbours:

  write   K and V of packed projections go into the pages of their sequences: K rotated to its position, both rounded to 8 bits
          (integers, or e4m3) with one scale for each token and head, or kept in bf16. What was written is read back, as the
          values that it stands for.
  read    the cached tokens of each sequence out of their pages, as contiguous bf16 caches.
  token   attention of one new token of each sequence over its pages, with the token's rotation and append.
  verify  drafted tokens against the target's probabilities (temperature, nucleus) from given random numbers: which path of each
          sequence's tree is kept, and the token behind it; with the probabilities that the drafts were drawn with, or without.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
ROPE_BASE = 10000.0
HEADS = {"125m": (12, 4, 64), "1.3b": (16, 4, 128), "7b": (32, 8, 128)}
VOCAB = 32000
KINDS = {"bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
LEAST_SCALE = 2.0 ** -80


# ------------------------------------------------------------------------------------------- the cases
def _cache(kind, model, store, B, lo, hi, page, **more):
    """``B`` sequences of ``lo`` to ``hi`` tokens in pages of ``page``, held as ``store``."""
    QH, KVH, D = HEADS[model]
    return dict(kind=kind, store=store, B=B, lo=lo, hi=hi, page=page, QH=QH, KVH=KVH, D=D, **more)


def _token(model, store, B, lo, hi, page, cap=0.0, bias=False):
    return _cache("token", model, store, B, lo, hi, page, cap=cap, bias=bias)


def _verify(B, n, width, V, temp, top, drawn):
    """``n`` nodes with at most ``width`` children each; ``drawn``: the drafts' probabilities are known."""
    return dict(kind="verify", B=B, n=n, width=width, V=V, temp=temp, top=top, drawn=drawn)


def listed():
    return [
        # short prompts of odd lengths, a new batch for the 125M model
        dict(_cache("write", "125m", "e4m3", 3, 37, 301, 32), name="write_prompts"),
        # one 7B context that is put into the cache at once
        dict(_cache("write", "7b", "int8", 1, 4096, 4096, 64), name="write_7b"),
        # one idle 125M conversation that goes on
        dict(_cache("read", "125m", "int8", 1, 777, 777, 32), name="read_125m"),
        # sequences of a 7B batch that go on in contiguous caches
        dict(_cache("read", "7b", "e4m3", 8, 2000, 4000, 128), name="read_7b"),
        # one sequence of a small model, the latency of a token
        dict(_token("125m", "int8", 1, 500, 500, 32), name="token_125m"),
        # a batch of the 1.3B model with capped scores, an empty sequence among very different lengths
        dict(_token("1.3b", "e4m3", 32, 0, 1980, 64, cap=50.0), name="token_ragged"),
        # a full serving batch of the 7B model
        dict(_token("7b", "int8", 64, 1500, 4000, 64), name="token_7b"),
        # one long context of the 7B model
        dict(_token("7b", "int8", 1, 60001, 60001, 128), name="token_long"),
        # a batch whose cache stays in bf16, scores with a distance bias
        dict(_token("1.3b", "bf16", 16, 900, 2047, 32, bias=True), name="token_bf16"),
        # a chain from a small draft model, one sequence
        dict(_verify(1, 6, 1, VOCAB, 0.7, 0.9, True), name="verify_chain"),
        # trees from the draft model's probabilities, a batch
        dict(_verify(8, 24, 3, VOCAB, 1.0, 1.0, True), name="verify_trees"),
        # large trees of looked-up drafts, a large batch
        dict(_verify(16, 63, 4, VOCAB, 0.7, 0.9, False), name="verify_large"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "token", "token", "verify"])
    if kind == "verify":
        V = rng.choice([VOCAB, _log(rng, 512, 80000)])
        drawn = rng.random() < 0.5
        n = _log(rng, 1, 64)
        most = 24_000_000 // (2 if drawn else 1)
        B = max(1, min(64, _log(rng, 1, 64), most // (n * V)))
        return _verify(B, n, rng.choice([1, 1, 2, 4]), V, rng.choice([0.0, 0.7, 1.0, 1.3]), rng.choice([1.0, 0.9, 0.5]), drawn)
    model, store, page = rng.choice(sorted(HEADS)), rng.choice(sorted(KINDS)), rng.choice([32, 64, 128])
    hi = _log(rng, 1, 16000 if kind == "read" else 4000 if kind == "write" else 60000)
    B = max(1, min(64, _log(rng, 1, 64), (90000 if kind == "token" else 4000 if kind == "write" else 16000) // hi))
    lo = rng.choice([hi, hi // 2, 0 if kind == "token" else 1]) if B > 1 else hi
    lo = max(lo, 0 if kind == "token" else 1)
    if kind != "token":
        return _cache(kind, model, store, B, lo, hi, page)
    mod = rng.choice(["", "", "cap", "bias"])
    return _token(model, store, B, lo, hi, page, cap=float(rng.choice([20, 30, 50])) if mod == "cap" else 0.0, bias=mod == "bias")


# ------------------------------------------------------------------------------------------- inputs
def _lens(c):
    B = c["B"]
    return [c["hi"] if B == 1 else c["lo"] + (c["hi"] - c["lo"]) * i // (B - 1) for i in range(B)]


def _rounded(x, store):
    """What ``store`` holds of fp32 rows, and their scales."""
    if store == "bf16":
        return x.to(torch.bfloat16), None
    s = (x.abs().amax(-1) / LARGEST[store]).clamp_min(LEAST_SCALE)
    y = x / s[..., None]
    return (torch.round(y).to(torch.int8) if store == "int8" else y.to(torch.float8_e4m3fn)), s


def _tables(n, D):
    freq = ROPE_BASE ** (-2.0 * torch.arange(D // 2, device=DEV, dtype=torch.float64) / D)
    ang = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "verify":
        return _prepare_verify(case, rng, g)
    QH, KVH, D, B, page = case["QH"], case["KVH"], case["D"], case["B"], case["page"]
    lens = _lens(case)
    rng.shuffle(lens)
    need = [(n + page) // page for n in lens]                                # room for one more token
    width = max(need)
    pages = list(range(sum(need) + 3))
    rng.shuffle(pages)
    table = torch.zeros((B, width), dtype=torch.int32)
    for b in range(B):
        for i in range(need[b]):
            table[b, i] = pages.pop()
    n_pages = sum(need) + 3

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=DEV, generator=g) * std

    s = dict(case=case, table=table.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    if case["kind"] == "write":
        M = sum(lens)
        dt = KINDS[case["store"]]
        s.update(k=torch.zeros((n_pages, KVH, page, D), device=DEV).to(dt), v=torch.zeros((n_pages, KVH, page, D), device=DEV).to(dt))
        for x in ("k_scale", "v_scale"):
            s[x] = torch.zeros((n_pages, KVH, page), device=DEV) if case["store"] != "bf16" else None
        # [K | Q | V] columns of the packed projection, sequence after sequence
        s["kqv"] = normal(M, (2 * KVH + QH) * D, std=1.5).to(torch.bfloat16)
        s["seq"] = torch.cat([torch.full((n,), b, dtype=torch.int32) for b, n in enumerate(lens)]).to(DEV)
        s["pos"] = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(DEV)
    else:
        s["k"], s["k_scale"] = _rounded(normal(n_pages, KVH, page, D, std=1.5), case["store"])
        s["v"], s["v_scale"] = _rounded(normal(n_pages, KVH, page, D), case["store"])
    if case["kind"] == "token":
        s["kqv"] = normal(B, (2 * KVH + QH) * D, std=1.5).to(torch.bfloat16)
        s["slopes"] = (torch.tensor([2.0 ** (-8.0 * (h + 1) / QH) for h in range(QH)], dtype=torch.float32, device=DEV)
                       if case["bias"] else None)
        s["start"], s["more"], rows = s["lens"], s["lens"] + 1, 1
    else:
        s["start"], s["more"], rows = torch.zeros_like(s["lens"]), s["lens"], case["hi"]
    # contiguous caches: of the whole sequences, or of the new tokens
    s["kc"], s["vc"] = (torch.zeros((B, KVH, rows, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    s["cos"], s["sin"] = _tables(case["hi"] + 1, D)
    return s


def _logits(rows, V, g):
    """Rows of logits whose probabilities fall off with a power of the rank, as those of text do."""
    rank = torch.rand(rows, V, device=DEV, generator=g) * V
    return -1.3 * torch.log1p(rank) + 0.4 * torch.randn(rows, V, device=DEV, generator=g)


def _prepare_verify(c, rng, g):
    B, n, width, V = c["B"], c["n"], c["width"], c["V"]
    parents = []
    for _ in range(B):
        row, kids = [-1], [0]
        for _ in range(1, n):
            free = [i for i, k in enumerate(kids) if k < width]
            p = free[-1] if rng.random() < 0.5 else rng.choice(free)
            kids[p] += 1
            row.append(p)
            kids.append(0)
        parents.append(row)
    rank = [[sum(q == p for q in row[:i]) for i, p in enumerate(row)] for row in parents]    # which child of its parent
    parents, rank = torch.tensor(parents, dtype=torch.int32, device=DEV), torch.tensor(rank, device=DEV)
    logits = _logits(B * n, V, g)
    near = logits + 0.5 * torch.randn(B * n, V, device=DEV, generator=g)
    if c["drawn"]:
        probs = torch.softmax(near / max(c["temp"], 0.5), -1)
        choice = torch.multinomial(probs, width, replacement=True, generator=g)
    else:
        probs, choice = None, torch.topk(near, width, -1).indices
    up = parents.clamp_min(0).long()
    tokens = choice.view(B, n, width)[torch.arange(B, device=DEV)[:, None], up, rank].to(torch.int32)
    return dict(case=c, logits=logits.view(B, n, V), tokens=tokens, parents=parents, probs=None if probs is None else probs.view(B, n, V),
                u=torch.rand(B, n, device=DEV, generator=g), accept=torch.rand(B, n, device=DEV, generator=g))


# ------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        from create_llm_by_cupy_b200.ops import drafts, paged
        if c["kind"] == "verify":
            tokens, path, count = drafts.verify_drafts(s["logits"], s["tokens"], s["parents"], s["u"], temp=c["temp"], top=c["top"],
                                                       draft_probs=s["probs"], accept=s["accept"] if c["drawn"] else None)
            return {"tokens": tokens, "path": path, "count": count}
        cache = paged.PagedCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        out = {}
        if c["kind"] == "write":
            KVH, QH, D = c["KVH"], c["QH"], c["D"]
            k, v = s["kqv"][:, :KVH * D].unflatten(1, (KVH, D)), s["kqv"][:, (KVH + QH) * D:].unflatten(1, (KVH, D))
            paged.paged_append(k, v, cache, s["table"], s["seq"], s["pos"], s["cos"], s["sin"])
        elif c["kind"] == "token":
            out["o"] = paged.paged_attn_append(s["kqv"], cache, s["table"], s["lens"], c["QH"], c["KVH"], s["cos"], s["sin"],
                                               softcap=c["cap"], slopes=s["slopes"])
        paged.paged_read(cache, s["table"], s["more"], s["kc"], s["vc"], start=s["start"])
        return _with_state(s, out)
    if c["kind"] == "verify":
        return _plain_verify(s, c)
    out = {}
    if c["kind"] == "write":
        _plain_write(s, c)
    elif c["kind"] == "token":
        out["o"] = _plain_token(s, c)
    _plain_read(s, c)
    return _with_state(s, out)


def _with_state(s, out):
    """What the pass wrote: pages of bf16, or scales, where they stand, and the rows as the values that they stand for."""
    out.update(kc=s["kc"], vc=s["vc"])
    if s["case"]["kind"] != "read":
        for x in ("k", "v"):
            name = x if s["k_scale"] is None else x + "_scale"
            out[name] = s[name]
    return out


def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _put(s, c, k, v, seq, pos):
    """fp32 rows [M, KVH, D] into the pages of (sequence, position)."""
    at = s["table"][seq, pos // c["page"]].long()
    off = pos % c["page"]
    for x, name in ((k, "k"), (v, "v")):
        y, scale = _rounded(x, c["store"])
        if c["store"] == "e4m3":                                             # indexed as bytes
            s[name].view(torch.uint8)[at, :, off] = y.view(torch.uint8)
        else:
            s[name][at, :, off] = y
        if scale is not None:
            s[name + "_scale"][at, :, off] = scale


def _plain_write(s, c):
    KVH, QH, D = c["KVH"], c["QH"], c["D"]
    k, _, v = s["kqv"].float().split([KVH * D, QH * D, KVH * D], dim=1)
    seq, pos = s["seq"].long(), s["pos"].long()
    k = _rotate(k.unflatten(1, (KVH, D)), s["cos"][pos][:, None], s["sin"][pos][:, None])
    _put(s, c, k, v.unflatten(1, (KVH, D)), seq, pos)


def _values(s, name, at, off):
    """fp32 values of tokens: [..., KVH, D] at page ``at``, row ``off``."""
    x = s[name]
    x = x.view(torch.uint8)[at, :, off].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[at, :, off]
    scale = s[name + "_scale"]
    return x.float() if scale is None else x.float() * scale[at, :, off][..., None]


def _plain_read(s, c):
    rows = s["kc"].shape[2]
    t = s["start"].long()[:, None] + torch.arange(rows, device=DEV)
    there = (t < s["more"][:, None])[:, None, :, None]
    t = t.clamp_max(s["table"].shape[1] * c["page"] - 1)
    at, off = torch.gather(s["table"].long(), 1, t // c["page"]), t % c["page"]
    for name, to in (("k", "kc"), ("v", "vc")):
        x = _values(s, name, at, off).transpose(1, 2).to(torch.bfloat16)
        s[to].copy_(torch.where(there, x, s[to]))


def _plain_token(s, c):
    B, KVH, QH, D, page = c["B"], c["KVH"], c["QH"], c["D"], c["page"]
    R, cap = QH // KVH, c["cap"]
    lens = s["lens"].long()
    k, q, v = s["kqv"].float().split([KVH * D, QH * D, KVH * D], dim=1)
    cos, sin = s["cos"][lens][:, None], s["sin"][lens][:, None]
    _put(s, c, _rotate(k.unflatten(1, (KVH, D)), cos, sin), v.unflatten(1, (KVH, D)), torch.arange(B, device=DEV), lens)
    q = _rotate(q.unflatten(1, (QH, D)), cos, sin).view(B, KVH, R, D)
    at = s["table"].long()
    T = at.shape[1] * page

    def rows(name):                                                          # [B, KVH, T, D]
        x = s[name]
        x = x.view(torch.uint8)[at].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[at]
        x = x.float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][at][..., None]
        return x.transpose(1, 2).reshape(B, KVH, T, D)

    x = (q @ rows("k").transpose(-1, -2)) / math.sqrt(D)
    if cap:
        x = cap * torch.tanh(x / cap)
    t = torch.arange(T, device=DEV)
    if c["bias"]:
        x = x - s["slopes"].view(KVH, R, 1) * (lens[:, None] - t).abs().float()[:, None, None]
    x = x.masked_fill((t > lens[:, None])[:, None, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    o = (x @ rows("v")) / x.sum(-1, keepdim=True)
    return o.view(B, QH, D).to(torch.bfloat16)


def _plain_verify(s, c):
    """In 64 bits: which token a number falls on depends on sums over the whole vocabulary."""
    B, n, V = c["B"], c["n"], c["V"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    if c["temp"] > 0:
        w = torch.exp((x - top) / c["temp"])
        if c["top"] < 1:
            ranked, order = torch.sort(w, dim=-1, descending=True, stable=True)
            below = torch.cumsum(ranked, -1) - ranked                        # mass in front of each
            ranked = torch.where(below < c["top"] * ranked.sum(-1, keepdim=True), ranked, torch.zeros_like(ranked))
            w = torch.zeros_like(w).scatter_(-1, order, ranked)
    else:
        w = torch.zeros_like(x).scatter_(-1, x.argmax(-1, keepdim=True), 1.0)
    p = w / w.sum(-1, keepdim=True)
    parents = s["parents"].long()
    kid = (parents[:, None, :] == torch.arange(n, device=DEV)[:, None])      # [B, i, j]: j is a child of i
    child = torch.full((B, n), -1, device=DEV)
    if c["drawn"]:
        q = s["probs"].double()
        nth = torch.cumsum(kid, -1) * kid
        used, mass = (torch.full((B, n), z, dtype=torch.float64, device=DEV) for z in (0.0, 1.0))
        for k in range(c["width"]):
            j = (nth == k + 1)
            there, j = j.any(-1) & (child < 0), j.int().argmax(-1)
            tok = torch.gather(s["tokens"].long(), 1, j)[..., None]
            px, qx = torch.gather(p, -1, tok)[..., 0], torch.gather(q, -1, tok)[..., 0]
            yes = there & (torch.gather(s["accept"], 1, j).double() * qx * mass < (px - used * qx).clamp_min(0))
            child = torch.where(yes, j, child)
            no = there & ~yes
            used = torch.where(no, used + mass, used)
            mass = torch.where(no, (p - used[..., None] * q).clamp_min(0).sum(-1), mass)
        left = (p - used[..., None] * q).clamp_min(0)
        p = torch.where((mass > 0)[..., None], left, p)
    cum = torch.cumsum(p, -1)
    tok = (cum <= s["u"].double()[..., None] * cum[..., -1:]).sum(-1).clamp_max(V - 1)
    if not c["drawn"]:
        hit = kid & (s["tokens"][:, None, :] == tok[..., None])
        child = torch.where(hit.any(-1), hit.int().argmax(-1), child)
    # a node is reached when each node on the way to it is its parent's choice
    chosen = torch.gather(child, 1, parents.clamp_min(0)) == torch.arange(n, device=DEV)
    chosen[:, 0] = True
    way = (kid.transpose(1, 2) | torch.eye(n, dtype=torch.bool, device=DEV)).float()
    for _ in range(max(1, (n - 1).bit_length())):
        way = ((way @ way) > 0).float()                                      # [B, j, i]: i is j or in front of it
    on = ((way > 0) <= chosen[:, None, :]).all(-1)
    count = on.sum(-1) - 1
    depth = (way > 0).sum(-1) - 1
    last = torch.where(on, depth, -1).argmax(-1, keepdim=True)
    path = torch.full((B, n + 1), -1, device=DEV)
    path.scatter_(1, torch.where(on & (depth > 0), depth - 1, n), torch.arange(n, device=DEV).expand(B, n))
    path = path[:, :n]
    tokens = torch.where(path >= 0, torch.gather(s["tokens"].long(), 1, path.clamp_min(0)), -1)
    tokens.scatter_(1, count[:, None], torch.gather(tok, 1, last))
    return {"tokens": tokens.to(torch.int32), "path": path.to(torch.int32), "count": count.to(torch.int32)}


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "verify":
        size = case["B"] * case["n"] * case["V"]
        return {"bytes": 4 * size * (2 if case["drawn"] else 1), "flops": 4 * size}
    KVH, QH, D, B = case["KVH"], case["QH"], case["D"], case["B"]
    tok = sum(_lens(case))
    held = KVH * (4 * D if case["store"] == "bf16" else 2 * D + 8)           # of one token
    if case["kind"] == "write":                                              # projection in, rows written and read, values out
        return {"bytes": tok * (4 * KVH * D + 4 * D + 2 * held + 4 * KVH * D), "flops": 10 * tok * KVH * D}
    if case["kind"] == "read":
        return {"bytes": tok * (held + 4 * KVH * D), "flops": 2 * tok * KVH * D}
    return {"bytes": tok * held + B * (2 * D * (2 * KVH + 2 * QH) + 2 * held + 4 * KVH * D), "flops": 4 * D * QH * (tok + B)}


# ------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_verify(s, case) if case["kind"] == "verify" else _exact_cache(s, case)


def _held(x, store):
    """fp64 rows as ``store`` holds them: values, and scales."""
    if store == "bf16":
        return x.to(torch.bfloat16).double(), None
    s = torch.maximum(x.abs().max(-1).values / LARGEST[store], torch.tensor(LEAST_SCALE, dtype=torch.float64, device=x.device))
    y = x / s.unsqueeze(-1)
    y = y.round() if store == "int8" else y.float().to(torch.float8_e4m3fn).double()
    return y * s.unsqueeze(-1), s


def _turned(x, pos, D):
    freq = ROPE_BASE ** (-2.0 * torch.arange(D // 2, device=DEV, dtype=torch.float64) / D)
    ang = (pos[:, None] * freq)[:, None]
    z = torch.view_as_real(torch.complex(x[..., :D // 2], x[..., D // 2:]) * torch.polar(torch.ones_like(ang), ang))
    return torch.cat([z[..., 0], z[..., 1]], -1)


def _exact_cache(s, c):
    """Sequence by sequence."""
    KVH, QH, D, B, page = c["KVH"], c["QH"], c["D"], c["B"], c["page"]
    table, lens = s["table"].tolist(), s["lens"].tolist()
    kc, vc = (torch.zeros(s["kc"].shape, dtype=torch.float64, device=DEV) for _ in range(2))
    bf16 = c["store"] == "bf16"
    ks, vs = (s[x if bf16 else x + "_scale"].double() for x in ("k", "v"))   # what is returned of the state
    o = torch.zeros(B, QH, D, dtype=torch.float64, device=DEV)
    first = 0
    for b, n in enumerate(lens):
        def cached(name):                                                    # [KVH, n, D] of the pages, in order
            rows = []
            for i in range((n + page - 1) // page):
                x = s[name][table[b][i]].double()
                rows.append(x if s[name + "_scale"] is None else x * s[name + "_scale"][table[b][i]].double().unsqueeze(-1))
            return torch.cat(rows, 1)[:, :n] if rows else torch.zeros(KVH, 0, D, dtype=torch.float64, device=DEV)

        if c["kind"] == "read":
            kc[b, :, :n], vc[b, :, :n] = cached("k"), cached("v")
            continue
        m = n if c["kind"] == "write" else 1
        x = s["kqv"][first:first + m].double().view(m, 2 * KVH + QH, D)
        first += m
        pos = torch.arange(n - m, n, dtype=torch.float64, device=DEV) + (0 if c["kind"] == "write" else 1)
        (k, k_s), (v, v_s) = _held(_turned(x[:, :KVH], pos, D), c["store"]), _held(x[:, KVH + QH:], c["store"])
        kc[b, :, :m], vc[b, :, :m] = k.transpose(0, 1), v.transpose(0, 1)
        where = pos.long().tolist()
        at = torch.tensor([table[b][t // page] for t in where], device=DEV)
        off = torch.tensor([t % page for t in where], device=DEV)
        ks[at, :, off], vs[at, :, off] = (k, v) if bf16 else (k_s, v_s)
        if c["kind"] == "token":
            keys = torch.cat([cached("k"), k.transpose(0, 1)], 1)
            vals = torch.cat([cached("v"), v.transpose(0, 1)], 1)
            q = _turned(x[:, KVH:KVH + QH], pos, D)[0].view(KVH, QH // KVH, D)
            x = torch.einsum("grd,gtd->grt", q, keys) * D ** -0.5
            x = c["cap"] * torch.tanh(x / c["cap"]) if c["cap"] else x
            if c["bias"]:
                far = n - torch.arange(n + 1, dtype=torch.float64, device=DEV)
                x = x - s["slopes"].double().view(KVH, -1, 1) * far
            o[b] = torch.einsum("grt,gtd->grd", torch.softmax(x, -1), vals).reshape(QH, D)
    out = {"kc": kc, "vc": vc}
    if c["kind"] == "token":
        out["o"] = o
    if c["kind"] != "read":
        out.update(dict(k=ks, v=vs) if bf16 else dict(k_scale=ks, v_scale=vs))
    return out


def _exact_verify(s, c):
    """Sequence by sequence, down its tree."""
    B, n = c["B"], c["n"]
    tokens, path = (torch.full((B, n), -1, dtype=torch.int32) for _ in range(2))
    count = torch.zeros(B, dtype=torch.int32)
    parents, drafts = s["parents"].tolist(), s["tokens"].tolist()
    u, accept = s["u"].double().tolist(), s["accept"].double().tolist()
    for b in range(B):
        node = 0
        while True:
            x = s["logits"][b, node].double()
            if c["temp"] == 0:
                p = torch.zeros_like(x)
                p[int((x == x.max()).nonzero()[0])] = 1.0
            else:
                p = torch.softmax(x / c["temp"], 0)
                if c["top"] < 1:
                    order = torch.sort(p, dim=0, descending=True, stable=True).indices
                    sums = torch.cumsum(p[order], 0)
                    kept = order[:int((sums < c["top"] * sums[-1]).sum()) + 1]
                    cut = torch.zeros_like(p)
                    cut[kept] = p[kept]
                    p = cut / cut.sum()
            kids, go = [j for j in range(1, n) if parents[b][j] == node], None
            if c["drawn"]:
                rest, q = p, s["probs"][b, node].double()
                for j in kids:
                    t = drafts[b][j]
                    if accept[b][j] * float(q[t]) < float(rest[t]):
                        go = j
                        break
                    rest = (rest - q).clamp_min(0)
                    rest = rest / rest.sum()
                p = rest if bool(torch.isfinite(rest).all()) else p
            if go is None:
                sums = torch.cumsum(p, 0)
                t = min(int(torch.searchsorted(sums, u[b][node] * sums[-1], right=True)), c["V"] - 1)
                if not c["drawn"]:
                    go = next((j for j in kids if drafts[b][j] == t), None)
            if go is None:
                tokens[b, count[b]] = t
                break
            tokens[b, count[b]], path[b, count[b]] = drafts[b][go], go
            count[b] += 1
            node = go
    return {"tokens": tokens, "path": path, "count": count}
