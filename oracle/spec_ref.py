"""Speculative decoding in 64 bits, the plain restatement the tests check against.

The reference has no counterpart (its ``generate`` decodes one token per step,
``kempnerforge/model/generate.py:60-131``); the attention it restates is the decode
of ``kempnerforge/model/attention.py:165-175,229-231`` with a mask among the new
tokens.
"""

from __future__ import annotations

import torch


def ancestors(parents: list[int]) -> list[list[int]]:
    """For each node, itself and its ancestors (parents come before children)."""
    out: list[list[int]] = []
    for i, p in enumerate(parents):
        assert -1 <= p < i
        out.append(([] if p < 0 else out[p]) + [i])
    return out


def _rotate(x, cos, sin):
    """Half-split RoPE of ``x [..., D]`` by one row of the tables, in 64 bits."""
    half = x.shape[-1] // 2
    c, s = cos.double(), sin.double()
    x1, x2 = x[..., :half], x[..., half:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def rotated(x, lens, cos, sin, parents, counts=None, row_offset=0, norm=None, eps=1e-5):
    """``x [B, N, H, D]`` (RMS-normalised first with ``norm``) rotated at each
    node's position, in 64 bits; unused nodes are left zero."""
    y = torch.zeros(x.shape, dtype=torch.float64)
    for b in range(x.shape[0]):
        n = x.shape[1] if counts is None else int(counts[b])
        for i, anc in enumerate(ancestors(parents[b][:n])):
            r = x[b, i].double()
            if norm is not None:
                r = r / (r.pow(2).mean(-1, keepdim=True) + eps).sqrt() * norm.double()
            at = int(lens[b]) + len(anc) - 1 - row_offset
            y[b, i] = _rotate(r, cos[at], sin[at])
    return y


def tree_attention(q, kc, vc, lens, parents, counts=None):
    """out (float64) of rotated queries ``q [B, N, Hq, D]`` over caches that hold the
    nodes' rows behind the prefix, and per output element the sum of p |v| (what
    errors of the probabilities multiply).  Unused nodes: zeros."""
    B, N, Hq, D = q.shape
    Hkv = kc.shape[1]
    rep = Hq // Hkv
    out = torch.zeros(B, N, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        n = N if counts is None else int(counts[b])
        L = int(lens[b])
        for i, anc in enumerate(ancestors(parents[b][:n])):
            rows = list(range(L)) + [L + j for j in anc]
            kk, vv = kc[b][:, rows].double(), vc[b][:, rows].double()
            p = torch.softmax(
                (q[b, i].double().view(Hkv, rep, D) @ kk.transpose(1, 2)) * D ** -0.5, dim=-1)
            out[b, i] = (p @ vv).view(Hq, D)
            mag[b, i] = (p @ vv.abs()).view(Hq, D)
    return out, mag


def verify(logits, tokens, uniforms, temperature, parents, counts=None, draft_logits=None):
    """path, kept, token as lists, walking one sequence at a time.  ``parents``: one
    list per sequence."""
    B, N, V = logits.shape
    paths, kepts, nexts = [], [], []

    def dist(row):
        e = ((row.double() - row.double().max()) / temperature).exp()
        return e / e.sum()

    for b in range(B):
        n = N if counts is None else int(counts[b])
        par, path, nxt = parents[b], [], -1
        if n > 0:
            cur, w = 0, None
            while True:
                path.append(cur)
                row = logits[b, cur]
                if temperature == 0:
                    if not torch.isfinite(row.max()):  # (NaN is the maximum of any row)
                        best = -1
                        break
                    best = int((row == row.max()).nonzero()[0])
                else:
                    w = dist(row)
                    if torch.isnan(w).any():
                        w = None
                        break
                step = None
                for i in range(cur + 1, n):
                    if par[i] != cur:
                        continue
                    c, u = int(tokens[b, i]), float(uniforms[b, i])
                    known = 0 <= c < V
                    if temperature == 0:
                        if c == best:
                            step = i
                            break
                    elif draft_logits is not None:
                        q = dist(draft_logits[b, cur])
                        if known and u * float(q[c]) < float(w[c]):
                            step = i
                            break
                        w = (w - q).clamp_min(0.0)
                    elif known and float(w[c]) > 0:
                        if u * float(w.sum()) < float(w[c]):
                            step = i
                            break
                        w[c] = 0.0
                if step is None:
                    break
                cur = step
            if temperature == 0:
                nxt = best
            elif w is not None:
                cum = w.cumsum(0)
                nxt = min(V - 1, int((cum <= float(uniforms[b, 0]) * cum[-1]).sum()))
        paths.append(path + [-1] * (N - len(path)))
        kepts.append(len(path))
        nexts.append(nxt)
    return paths, kepts, nexts


def keep(cache, lens, path, kept):
    """The cache ``[B, H, S, D]`` after the accepted rows have moved together."""
    out = cache.clone()
    for b in range(cache.shape[0]):
        L = int(lens[b])
        for j in range(int(kept[b])):
            out[b, :, L + j] = cache[b, :, L + int(path[b][j])]
    return out
