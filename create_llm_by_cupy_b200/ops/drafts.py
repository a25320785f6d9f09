"""Verification of drafted tokens against the target's probabilities: which of them a sampled text keeps, and the token behind them.

    tokens, path, count = verify_drafts(logits, drafts, parents, u, temp=0.7, top=0.9)                         # looked-up drafts
    tokens, path, count = verify_drafts(logits, drafts, parents, u, draft_probs=q, accept=a)                   # drawn from a draft model

What is kept is distributed as if the target alone had drawn it, whatever the drafts are. As in ``functional``, CUDA tensors go to the
hand-written sm_100a kernels, CPU tensors take a plain torch restatement in fp64. The kernels' weights are fp64, off by at most 3e-13 of
themselves, and are summed as whole numbers of 2^-(62 - b) of the row's largest, b the bits of the vocabulary's size (2^-47 at 32000 tokens,
2^-43 at the most), which add up to the same in any order: the two forms differ where a number falls that close to a border.
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import functional as F
from . import native

MOST_NODES = 64
MOST_TOKENS = 8 * 376 * 128


def verify_drafts(logits, tokens, parents, u, *, temp: float = 1.0, top: float = 1.0, draft_probs=None, accept=None):
    """Each of ``B`` sequences has ``n`` nodes (1 to 64): node 0 is its last token, the others are drafts. ``logits`` [B, n, V] (fp32 or
    bf16): the target's, of the token behind each node; ``tokens`` int32 [B, n]: what the drafts are (node 0's is not read); ``parents``
    int32 [B, n]: the node that each draft continues, which stands before it. A draft whose parent does not (-1) is not there: batches
    may be ragged. ``u`` fp32 [B, n]: numbers from [0, 1), for the draw behind each node.

    A node's probabilities p are the softmax of its logits / ``temp`` over its nucleus, the fewest tokens, by falling probability and
    rising index, whose mass reaches ``top``. ``temp`` is from 1e-6 to 1e6, or 0, which leaves the largest logit, of several the one of the
    lowest index. Logits of -infinity and NaN count for nothing, +infinity for the largest number.

    Without ``draft_probs`` the token behind a node is the first whose sum of probabilities, in the order of the tokens, exceeds u; if a
    child holds it (of several the first) the text goes on there. With ``draft_probs`` fp32 [B, n, V] - row i: the distribution q that
    the children of node i were drawn from, independently - and ``accept`` fp32 [B, n], a number from [0, 1) for each draft, the children
    are tried in their order: one that holds x is kept if accept q(x) < p(x), and if not, p becomes max(p - q, 0) over its sum for those
    behind it (p itself, should nothing be left). If none is kept, the token behind the node is drawn from what p has become. A draft
    whose token is not of the vocabulary is not tried.

    Returns int32 (tokens [B, n]: the kept drafts' and the one behind them, then -1; path [B, n]: the kept nodes, then -1; count [B]: how
    many are kept). A node all of whose logits are -infinity ends the text with -1."""
    if native.host is not None:
        r = native.host.verify_drafts(logits, tokens, parents, u, temp, top, draft_probs, accept)
        if r is not None:
            native.bump(2)
            return r
    if logits.dim() != 3 or 0 in logits.shape[1:] or logits.shape[1] > MOST_NODES:
        raise ValueError(f"verify_drafts: logits are [B, n, V], with 1 to {MOST_NODES} nodes")
    B, n, V = logits.shape
    if V > MOST_TOKENS:
        raise ValueError(f"verify_drafts: vocabularies of up to {MOST_TOKENS} tokens")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("verify_drafts: logits are float32 or bfloat16")
    for what, t, dt in (("tokens", tokens, torch.int32), ("parents", parents, torch.int32), ("u", u, torch.float32)):
        if tuple(t.shape) != (B, n) or t.dtype != dt:
            raise ValueError(f"verify_drafts: {what} is {str(dt).removeprefix('torch.')} [B, n]")
    if (draft_probs is None) != (accept is None):
        raise ValueError("verify_drafts: draft_probs and accept, or neither")
    if draft_probs is not None and (draft_probs.shape != logits.shape or draft_probs.dtype != torch.float32 or
                                    tuple(accept.shape) != (B, n) or accept.dtype != torch.float32):
        raise ValueError("verify_drafts: draft_probs is float32 [B, n, V], accept float32 [B, n]")
    temp, top = float(temp), float(top)
    if not (temp == 0.0 or 1e-6 <= temp <= 1e6) or not top > 0.0:
        raise ValueError("verify_drafts: temp is 0 or from 1e-6 to 1e6, top is more than 0")
    if any(t is not None and t.device != logits.device for t in (tokens, parents, u, draft_probs, accept)):
        raise ValueError("verify_drafts: all tensors are on one device")
    if not logits.is_cuda:
        return _reference(logits, tokens, parents, u, temp, top, draft_probs, accept)
    with torch.cuda.device(logits.device):
        out, path = (torch.empty((B, n), dtype=torch.int32, device=logits.device) for _ in range(2))
        count = torch.empty(B, dtype=torch.int32, device=logits.device)
        if B == 0:
            return out, path, count
        logits, tokens, parents, u = logits.contiguous(), tokens.contiguous(), parents.contiguous(), u.contiguous()
        if draft_probs is not None:
            draft_probs, accept = draft_probs.contiguous(), accept.contiguous()
        ws = torch.empty(2 * B * n, dtype=torch.int32, device=logits.device)
        native.check(F._lib().b200_verify_drafts(
            native.ptr(logits), native.ptr(draft_probs), native.ptr(tokens), native.ptr(parents), native.ptr(u), native.ptr(accept),
            native.ptr(out), native.ptr(path), native.ptr(count), native.ptr(ws), int(logits.dtype == torch.bfloat16), B, n, V,
            ctypes.c_double(temp), ctypes.c_double(top), native.stream_ptr()), "verify_drafts")
    native.bump(2)
    return out, path, count


def target_probs(logits, temp: float, top: float):
    """fp64 probabilities of rows of logits [..., V] as ``verify_drafts`` takes them; a row of which nothing is left is 0."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x).clamp_max(torch.finfo(torch.float32).max)
    most = x.amax(-1, keepdim=True)
    if temp == 0.0:
        w = torch.zeros_like(x).scatter_(-1, (x == most).int().argmax(-1, keepdim=True), 1.0)
    else:
        w = torch.exp((x - torch.where(most == -math.inf, 0.0, most)) / temp)
        if top < 1.0:
            ranked, order = torch.sort(w, dim=-1, descending=True, stable=True)
            front = torch.cumsum(ranked, -1) - ranked
            ranked = torch.where(front < top * ranked.sum(-1, keepdim=True), ranked, 0.0)
            w = torch.zeros_like(w).scatter_(-1, order, ranked)
    w = torch.where(most == -math.inf, 0.0, w)
    total = w.sum(-1, keepdim=True)
    return w / torch.where(total > 0, total, 1.0)


def _reference(logits, tokens, parents, u, temp, top, draft_probs, accept):
    B, n, V = logits.shape
    out, path = (torch.full((B, n), -1, dtype=torch.int32) for _ in range(2))
    count = torch.zeros(B, dtype=torch.int32)
    par, tok = parents.tolist(), tokens.tolist()
    for b in range(B):
        node = 0
        while True:
            p = target_probs(logits[b, node], temp, top)
            if not bool(p.sum() > 0):
                break
            kids, go, t = [j for j in range(node + 1, n) if par[b][j] == node], -1, -1
            if draft_probs is not None:
                q, used, mass = draft_probs[b, node].double(), 0.0, 1.0
                for j in kids:
                    if not 0 <= tok[b][j] < V:
                        continue
                    px, qx = float(p[tok[b][j]]), float(q[tok[b][j]])
                    if float(accept[b, j]) * qx * mass < max(px - used * qx, 0.0):
                        go = j
                        break
                    used += mass
                    mass = float((p - used * q).clamp_min(0.0).sum())
                if go < 0 and used > 0.0 and mass > 0.0:
                    p = (p - used * q).clamp_min(0.0)
            if go < 0:
                sums = torch.cumsum(p, 0)
                t = int((sums <= float(u[b, node]) * sums[-1]).sum())
                t = min(t, int(p.nonzero()[-1]))
                if draft_probs is None:
                    go = next((j for j in kids if tok[b][j] == t), -1)
            out[b, count[b]] = tok[b][go] if go >= 0 else t
            if go < 0:
                break
            path[b, count[b]] = go
            count[b] += 1
            node = go
    return out, path, count
