"""Several continuations of one prompt in 64 bits, the plain restatement the tests check
against: attention behind a shared prefix, the beams' selection, the caches' move.

The reference has no counterpart (its ``generate`` keeps a copy of the prompt per
sequence, ``kempnerforge/model/generate.py:60-131``); the attention is the decode of
``kempnerforge/model/attention.py:165-175,229-231`` over the prefix and the sequence's
own rows.
"""

from __future__ import annotations

import torch

from oracle.spec_ref import _rotate


def rotated(x, starts, cos, sin, counts, row_offset=0, norm=None, eps=1e-5):
    """``x [B, N, H, D]`` (RMS-normalised first with ``norm``), token i of sequence b
    rotated at position ``starts[b] + i``, in 64 bits; unused tokens are left zero."""
    y = torch.zeros(x.shape, dtype=torch.float64)
    for b in range(x.shape[0]):
        for i in range(counts[b]):
            r = x[b, i].double()
            if norm is not None:
                r = r / (r.pow(2).mean(-1, keepdim=True) + eps).sqrt() * norm.double()
            at = starts[b] + i - row_offset
            y[b, i] = _rotate(r, cos[at], sin[at])
    return y


def branch_attention(q, kp, vp, plens, kc, vc, lens, counts):
    """out (float64) of rotated queries ``q [B, N, Hq, D]`` over prefixes and caches that
    hold the new tokens' rows, and per output element the sum of p |v|."""
    B, N, Hq, D = q.shape
    G, Hkv = kp.shape[:2]
    out = torch.zeros(B, N, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        g = b // (B // G)
        for i in range(counts[b]):
            n = lens[b] + i + 1
            kk = torch.cat([kp[g, :, :plens[g]], kc[b, :, :n]], dim=1).double()
            vv = torch.cat([vp[g, :, :plens[g]], vc[b, :, :n]], dim=1).double()
            p = torch.softmax(
                (q[b, i].double().view(Hkv, -1, D) @ kk.transpose(1, 2)) * D ** -0.5, dim=-1)
            out[b, i] = (p @ vv).view(Hq, D)
            mag[b, i] = (p @ vv.abs()).view(Hq, D)
    return out, mag


def totals(logits, scores):
    """``[G, W, V]`` in 64 bits: what the selection orders; -inf where there is no
    candidate."""
    x, s = logits.double(), scores.double()
    ok = torch.isfinite(s) & torch.isfinite(x.amax(-1))  # (NaN is the maximum of any row)
    x = torch.where(ok[..., None], x, 0.0)
    t = torch.where(ok, s, 0.0)[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))
    return torch.where(ok[..., None], t, -torch.inf)


def select(logits, scores, K):
    """scores (float64), parents and tokens of the K best, equals by the lowest beam, then
    token; -inf, -1, -1 behind the last candidate."""
    G, W, V = logits.shape
    t = totals(logits, scores).view(G, W * V)
    best, at = t.sort(dim=-1, descending=True, stable=True)
    if W * V < K:
        best = torch.nn.functional.pad(best, (0, K - W * V), value=-torch.inf)
        at = torch.nn.functional.pad(at, (0, K - W * V))
    best, at = best[:, :K], at[:, :K]
    none = torch.isinf(best)
    return best, torch.where(none, -1, at // V).int(), torch.where(none, -1, at % V)


def reorder(cache, lens, parents):
    """The cache after the move (``parents``: a list of lists)."""
    out = cache.clone()
    W = len(parents[0])
    for g, row in enumerate(parents):
        for w, p in enumerate(row):
            if 0 <= p < W and 0 <= lens[g * W + p] <= cache.shape[2]:
                n = lens[g * W + p]
                out[g * W + w, :, :n] = cache[g * W + p, :, :n]
    return out
