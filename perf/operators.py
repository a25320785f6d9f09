"""What the masked and the drafted-token attention are measured on.

Two operators, with sizes of the benchmark configurations (125M: 12 / 4 heads of 64, context 1024; 1.3B: 16 / 4 heads of
128, context 2048; 7B: 32 / 8 heads of 128, context 4096) and their neighbours:

  span   attention of packed sequences: every query sees a run of keys, given by the documents that are packed into its
         row (causal inside each; a document's leading prefix sees itself whole; padding sees nothing), with scores that
         are capped by a tanh or get a bias that grows with the distance. ``train``: forward and backward.
  tree   attention of n drafted tokens per sequence over its KV cache: K | Q | V of the drafts come packed from the
         projection, K and Q are rotated to their depth in the tree, K and V appended behind the cached tokens, and each
         draft sees the cached tokens, its ancestors and itself. n = 1 is the plain decoded token.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
ROPE_BASE = 10000.0
HEADS = {"125m": (12, 4, 64), "1.3b": (16, 4, 128), "7b": (32, 8, 128)}


# ------------------------------------------------------------------------------------------- the cases
def _span(model, B, T, doc, *, prefix=0.0, pad=0, cap=0.0, bias=False, train=False):
    """``doc``: mean length of a document (0: one per row); ``prefix``: share of a document's tokens that are its
    prefix; ``pad``: padding at the end of every row."""
    QH, KVH, D = HEADS[model]
    return dict(kind="span", B=B, T=T, QH=QH, KVH=KVH, D=D, doc=doc, prefix=prefix, pad=pad, cap=cap, bias=bias, train=train)


def _tree(model, B, n, lo, hi, ctx, *, cap=0.0, bias=False):
    """Sequences of ``lo`` to ``hi`` cached tokens in caches of ``ctx`` positions, ``n`` drafts each."""
    QH, KVH, D = HEADS[model]
    return dict(kind="tree", B=B, n=n, lo=lo, hi=hi, ctx=ctx, QH=QH, KVH=KVH, D=D, cap=cap, bias=bias)


def listed():
    return [
        # a short prompt that is scored: one row, a prefix that sees itself, capped scores
        dict(_span("125m", 1, 100, 0, prefix=0.5, cap=30.0), name="score_short"),
        # a 7B context of instruction and answer pairs that is scored
        dict(_span("7b", 1, 4096, 700, prefix=0.4), name="score_7b"),
        # small fine-tuning batch: prefix documents of an odd length
        dict(_span("125m", 2, 301, 90, prefix=0.3, train=True), name="train_prefix"),
        # rows of documents and padding with a distance bias, a length that is no multiple of a tile
        dict(_span("125m", 3, 777, 260, pad=70, bias=True, train=True), name="train_bias"),
        # pre-training of the 125M model on packed documents
        dict(_span("125m", 8, 1024, 200, train=True), name="train_125m"),
        # pre-training of the 1.3B model on packed documents, capped scores
        dict(_span("1.3b", 4, 2048, 600, cap=50.0, train=True), name="train_1.3b"),
        # context extension of the 1.3B model: one document of 8192 tokens, capped scores
        dict(_span("1.3b", 1, 8192, 0, cap=50.0, train=True), name="train_long"),
        # one decoded token of one sequence of a model with capped scores
        dict(_tree("1.3b", 1, 1, 1801, 1801, 2048, cap=50.0), name="token_1.3b"),
        # a small draft tree of one sequence
        dict(_tree("125m", 1, 16, 500, 500, 1024), name="tree_125m"),
        # draft trees of a batch of 7B sequences of about the same length
        dict(_tree("7b", 8, 24, 2800, 3200, 4096), name="tree_7b"),
        # large trees over sequences of very different lengths, an empty one among them
        dict(_tree("1.3b", 16, 63, 0, 1980, 2048, cap=50.0), name="tree_ragged"),
        # a draft tree at the end of one long context
        dict(_tree("7b", 1, 32, 60001, 60001, 65536), name="tree_long"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    model = rng.choice(sorted(HEADS))
    mod = rng.choice(["", "", "cap", "bias"])
    cap = float(rng.choice([20, 30, 50])) if mod == "cap" else 0.0
    if rng.random() < 0.5:
        prefix = rng.choice([0.0, 0.0, 0.3, 0.6])
        T = _log(rng, 64, 5900 if prefix else 8192)
        tokens = 8192 * (1 if T > 4096 or prefix else 2)
        if model == "7b":
            tokens //= 2
            T = min(T, 4900)
        B = max(1, min(8, tokens // T, _log(rng, 1, 8)))
        doc = rng.choice([0, _log(rng, 40, 1500)])
        return _span(model, B, T, doc, prefix=prefix, pad=rng.choice([0, 0, T // 9]), cap=cap,
                     bias=mod == "bias", train=rng.random() < 0.7)
    n = _log(rng, 1, 64)
    hi = _log(rng, 64, 60000)
    B = max(1, min(16, 60000 // hi, _log(rng, 1, 16)))
    lo = rng.choice([hi, hi, 0, hi // 2]) if B > 1 else hi
    return _tree(model, B, n, lo, hi, hi + n + rng.randrange(0, 200), cap=cap, bias=mod == "bias")


# ------------------------------------------------------------------------------------------- inputs
def _documents(case):
    """(length, prefix length) of the documents of each row: fixed by the case, so that its work is."""
    rng = random.Random(1000003 * case["T"] + 7 * case["doc"] + case["B"])
    rows = []
    for _ in range(case["B"]):
        left, row = case["T"] - case["pad"], []
        while left > 0:
            n = left if case["doc"] == 0 else max(2, int(rng.expovariate(1.0 / case["doc"])))
            n = left if left - n < 2 else n
            row.append((n, int(n * case["prefix"])))
            left -= n
        rows.append(row)
    return rows


def _lens(case):
    B = case["B"]
    return [case["hi"] if B == 1 else case["lo"] + (case["hi"] - case["lo"]) * i // (B - 1) for i in range(B)]


def _slopes(QH):
    """Slopes of the distance bias, a geometric row from 2^-(8 / heads) down to 2^-8."""
    return [2.0 ** (-8.0 * (h + 1) / QH) for h in range(QH)]


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * std).to(torch.bfloat16)

    QH, KVH, D, B = case["QH"], case["KVH"], case["D"], case["B"]
    s = dict(case=case, slopes=torch.tensor(_slopes(QH), dtype=torch.float32, device=DEV) if case["bias"] else None)
    if case["kind"] == "span":
        T = case["T"]
        docs = torch.full((B, T), -1, dtype=torch.int32)
        prefix = torch.zeros((B, T), dtype=torch.bool)
        for b, row in enumerate(_documents(case)):
            rng.shuffle(row)
            at = 0
            for i, (n, pre) in enumerate(row):
                docs[b, at:at + n] = i
                prefix[b, at:at + pre] = True
                at += n
        # one packed projection as the layer has it: [K | Q | V] columns
        kqv = normal(B, T, (2 * KVH + QH) * D, std=1.5)
        k, q, v = kqv.split([KVH * D, QH * D, KVH * D], dim=2)
        s.update(q=q.unflatten(2, (QH, D)), k=k.unflatten(2, (KVH, D)), v=v.unflatten(2, (KVH, D)),
                 docs=docs.to(DEV), prefix=prefix.to(DEV) if case["prefix"] else None)
        if case["train"]:
            s["dout"] = normal(B, T, QH, D)
        return s
    n, ctx = case["n"], case["ctx"]
    lens = _lens(case)
    rng.shuffle(lens)
    parents = [[-1] + [rng.choice([i - 1, rng.randrange(-1, i)]) for i in range(1, n)] for _ in range(B)]
    bits = torch.zeros((B, n), dtype=torch.int64)
    for b in range(B):
        for i, p in enumerate(parents[b]):
            m = (1 << i) | (int(bits[b, p]) if p >= 0 else 0)
            bits[b, i] = m - (1 << 64) if m >= 1 << 63 else m
    freq = ROPE_BASE ** (-2.0 * torch.arange(D // 2, device=DEV, dtype=torch.float64) / D)
    ang = torch.arange(ctx, device=DEV, dtype=torch.float64)[:, None] * freq
    s.update(kqv=normal(B * n, (2 * KVH + QH) * D, std=1.5), k=normal(B, KVH, ctx, D, std=1.5), v=normal(B, KVH, ctx, D),
             lens=torch.tensor(lens, dtype=torch.int32, device=DEV), tree=bits.to(DEV), cos=ang.cos().float(), sin=ang.sin().float())
    return s


# ------------------------------------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    if own:
        from create_llm_by_cupy_b200.ops import masked_attn as A
        mod = dict(softcap=c["cap"], slopes=s["slopes"])
        if c["kind"] == "tree":
            o = A.tree_attn_append(s["kqv"], s["k"], s["v"], s["lens"], s["tree"], c["QH"], c["KVH"], s["cos"], s["sin"], **mod)
            return {"o": o, "k": s["k"], "v": s["v"]}
        mask = A.span_mask(c["B"], c["T"], DEV, docs=s["docs"], prefix=s["prefix"])
        o, lse = A.span_attn_fwd(s["q"], s["k"], s["v"], mask, **mod)
        if not c["train"]:
            return {"o": o, "lse": lse}
        dq, dk, dv = A.span_attn_bwd(s["dout"], s["q"], s["k"], s["v"], o, lse, mask, **mod)
        return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    return _plain_tree(s, c) if c["kind"] == "tree" else _plain_span(s, c)


def _seen(docs, prefix):
    """[B, T, T]: which keys (last) a query sees."""
    T = docs.shape[1]
    t = torch.arange(T, device=docs.device)
    same = (docs[:, :, None] == docs[:, None, :]) & (docs >= 0)[:, :, None]
    ok = t[:, None] >= t[None, :]
    if prefix is not None:
        ok = ok | (prefix[:, :, None] & prefix[:, None, :])
    return same & ok


def _plain_span(s, c):
    scale, cap = 1.0 / math.sqrt(c["D"]), c["cap"]
    B, T, QH, KVH, D = c["B"], c["T"], c["QH"], c["KVH"], c["D"]
    R = QH // KVH
    q = s["q"].float().reshape(B, T, KVH, R, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, R * T, D)
    k = s["k"].float().transpose(1, 2)
    v = s["v"].float().transpose(1, 2)
    seen = _seen(s["docs"], s["prefix"])[:, None]
    x = ((q @ k.transpose(-1, -2)) * scale).view(B, QH, T, T)
    if cap:
        x = torch.tanh(x / cap)
        th, x = x, x * cap
    if c["bias"]:
        t = torch.arange(T, device=x.device, dtype=torch.float32)
        x = x - s["slopes"][:, None, None] * (t[:, None] - t[None, :]).abs()
    x = x.masked_fill(~seen, float("-inf"))
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    x = torch.exp(x - m)
    l = x.sum(-1, keepdim=True)
    lse = (m + torch.log(l))[..., 0]
    p = x / torch.where(l > 0, l, torch.ones_like(l))
    del x, seen
    of = p.view(B, KVH, R * T, T) @ v
    o = of.view(B, KVH, R, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, QH, D).to(torch.bfloat16)
    if not c["train"]:
        return {"o": o, "lse": lse}
    do = s["dout"].float().reshape(B, T, KVH, R, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, R * T, D)
    dv = p.view(B, KVH, R * T, T).transpose(-1, -2) @ do
    ds = (do @ v.transpose(-1, -2) - (do * of).sum(-1, keepdim=True)).view(B, QH, T, T)
    ds = p * ds * scale
    del p
    if cap:
        ds = ds * (1 - th * th)
        del th
    ds = ds.view(B, KVH, R * T, T)
    dq = (ds @ k).view(B, KVH, R, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, QH, D)
    dk = (ds.transpose(-1, -2) @ q).transpose(1, 2)
    return {"o": o, "lse": lse, "dq": dq.to(torch.bfloat16), "dk": dk.to(torch.bfloat16).contiguous(),
            "dv": dv.transpose(1, 2).to(torch.bfloat16).contiguous()}


def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_tree(s, c):
    B, n, QH, KVH, D, ctx = c["B"], c["n"], c["QH"], c["KVH"], c["D"], c["ctx"]
    R, scale, cap = QH // KVH, 1.0 / math.sqrt(c["D"]), c["cap"]
    j = torch.arange(n, device=DEV)
    sees = (s["tree"][:, :, None] >> j) & 1                                  # [B, n, n]
    depth = sees.sum(-1) - 1
    pos = s["lens"].long()[:, None] + depth                                  # [B, n]
    at = s["lens"].long()[:, None] + j                                       # where a draft is kept
    k, q, v = s["kqv"].float().view(B, n, -1).split([KVH * D, QH * D, KVH * D], dim=2)
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    k = _rotate(k.reshape(B, n, KVH, D), cos, sin).to(torch.bfloat16)
    q = _rotate(q.reshape(B, n, QH, D), cos, sin)
    b = torch.arange(B, device=DEV)[:, None]
    s["k"][b, :, at] = k
    s["v"][b, :, at] = v.reshape(B, n, KVH, D).to(torch.bfloat16)
    q = q.reshape(B, n, KVH, R, D).permute(0, 2, 3, 1, 4).reshape(B, KVH, R * n, D)
    x = ((q @ s["k"].float().transpose(-1, -2)) * scale).view(B, QH, n, ctx)
    if cap:
        x = cap * torch.tanh(x / cap)
    t = torch.arange(ctx, device=DEV)
    off = t - s["lens"][:, None]                                             # [B, ctx]: which draft a key is
    bit = torch.gather(sees, 2, off.clamp(0, n - 1)[:, None].expand(B, n, ctx))
    seen = (off < 0)[:, None] | ((off < n)[:, None] & (bit > 0))
    if c["bias"]:
        kpos = torch.where(off < 0, t, s["lens"][:, None] + torch.gather(depth, 1, off.clamp(0, n - 1)))
        x = x - (s["slopes"][:, None, None] * (pos[:, :, None] - kpos[:, None, :]).abs().float()[:, None])
    x = x.masked_fill(~seen[:, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    p = x / x.sum(-1, keepdim=True)
    o = (p.view(B, KVH, R * n, ctx) @ s["v"].float()).view(B, KVH, R, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, QH, D)
    return {"o": o.to(torch.bfloat16), "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    QH, KVH, D, B = case["QH"], case["KVH"], case["D"], case["B"]
    if case["kind"] == "span":
        pairs = sum(n * (n + 1) // 2 + p * (p - 1) // 2 for row in _documents(case) for n, p in row)
        tok = B * case["T"]
        nbytes = tok * (2 * D * (2 * QH + 2 * KVH) + 4 * QH + 4)
        if case["train"]:
            nbytes += tok * 2 * D * (2 * QH + 2 * KVH)
        return {"bytes": nbytes, "flops": (14 if case["train"] else 4) * D * QH * pairs}
    n, lens = case["n"], _lens(case)
    # cached rows are read, the drafts' rows read with their projection and written
    nbytes = sum(lens) * KVH * D * 4 + B * n * (2 * D * (2 * KVH + 2 * QH) + 4 * KVH * D + 8)
    return {"bytes": nbytes, "flops": 4 * D * QH * sum(n * (x + 1) for x in lens)}


# ------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_tree(s, case) if case["kind"] == "tree" else _exact_span(s, case)


def _softmax_of(x, cap, slope, dist, seen):
    if cap:
        x = cap * torch.tanh(x / cap)
    if slope is not None:
        x = x - slope * dist
    return x.masked_fill(~seen, float("-inf"))


def _exact_span(s, c):
    """Document by document and head by head; gradients by reverse differentiation of that."""
    B, T, QH, KVH, D = c["B"], c["T"], c["QH"], c["KVH"], c["D"]
    R = QH // KVH
    q, k, v = (s[x].detach().double() for x in "qkv")
    o = torch.zeros(B, T, QH, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, QH, T), float("-inf"), dtype=torch.float64, device=DEV)
    dq, dk, dv = (torch.zeros(*x.shape, dtype=torch.float64, device=DEV) for x in (q, k, v))
    docs = s["docs"].cpu()
    for b in range(B):
        ids, sizes = torch.unique_consecutive(docs[b], return_counts=True)
        a = 0
        for i, size in zip(ids.tolist(), sizes.tolist()):
            e = a + size
            if i < 0:
                a = e
                continue
            pre = 0 if s["prefix"] is None else int(s["prefix"][b, a:e].sum())
            r = torch.arange(size, device=DEV)
            seen = (r[None, :] <= r[:, None]) | ((r[None, :] < pre) & (r[:, None] < pre))
            dist = (r[None, :] - r[:, None]).abs().double()
            for h in range(QH):
                leaf = [x[b, a:e, y].clone().requires_grad_(c["train"]) for x, y in ((q, h), (k, h // R), (v, h // R))]
                x = _softmax_of(leaf[0] @ leaf[1].T / math.sqrt(D), c["cap"], float(s["slopes"][h]) if c["bias"] else None, dist, seen)
                out = torch.softmax(x, -1) @ leaf[2]
                o[b, a:e, h] = out.detach()
                lse[b, h, a:e] = torch.logsumexp(x.detach(), -1)
                if c["train"]:
                    gq, gk, gv = torch.autograd.grad(out, leaf, s["dout"][b, a:e, h].double())
                    dq[b, a:e, h] += gq
                    dk[b, a:e, h // R] += gk
                    dv[b, a:e, h // R] += gv
            a = e
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv} if c["train"] else {"o": o, "lse": lse}


def _exact_tree(s, c):
    """Sequence by sequence, with the tree walked draft by draft. The caches hold bfloat16: the appended rows are rounded."""
    B, n, QH, KVH, D = c["B"], c["n"], c["QH"], c["KVH"], c["D"]
    R = QH // KVH
    kc, vc = s["k"].double(), s["v"].double()
    o = torch.zeros(B, n, QH, D, dtype=torch.float64, device=DEV)
    tree, lens = s["tree"].tolist(), s["lens"].tolist()
    freq = ROPE_BASE ** (-2.0 * torch.arange(D // 2, device=DEV, dtype=torch.float64) / D)
    rows = s["kqv"].double().view(B, n, 2 * KVH + QH, D)
    for b in range(B):
        L = lens[b]
        anc = [[j for j in range(n) if (tree[b][i] >> j) & 1] for i in range(n)]
        depth = torch.tensor([len(x) - 1 for x in anc], dtype=torch.float64, device=DEV)
        ang = (L + depth)[:, None, None] * freq
        turned = torch.view_as_real(torch.complex(rows[b, ..., :D // 2], rows[b, ..., D // 2:]) * torch.polar(torch.ones_like(ang), ang))
        turned = torch.cat([turned[..., 0], turned[..., 1]], -1)
        knew, vnew = turned[:, :KVH], rows[b, :, KVH + QH:]
        kc[b, :, L:L + n] = knew.transpose(0, 1)
        vc[b, :, L:L + n] = vnew.transpose(0, 1)
        keys = torch.cat([kc[b, :, :L], knew.transpose(0, 1).to(torch.bfloat16).double()], 1)
        vals = vc[b, :, :L + n]
        seen = torch.zeros(n, L + n, dtype=torch.bool, device=DEV)
        seen[:, :L] = True
        for i in range(n):
            seen[i, [L + j for j in anc[i]]] = True
        kpos = torch.cat([torch.arange(L, device=DEV, dtype=torch.float64), L + depth])
        dist = ((L + depth)[:, None] - kpos[None, :]).abs()
        for h in range(QH):
            x = _softmax_of(turned[:, KVH + h] @ keys[h // R].T / math.sqrt(D), c["cap"], float(s["slopes"][h]) if c["bias"] else None,
                            dist, seen)
            o[b, :, h] = torch.softmax(x, -1) @ vals[h // R]
    return {"o": o, "k": kc, "v": vc}
