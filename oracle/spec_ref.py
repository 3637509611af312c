"""Speculative decoding in 64 bits, the plain restatement the tests check against.

The reference has no counterpart (its ``generate`` decodes one token per step,
``kempnerforge/model/generate.py:60-131``); the attention it restates is the decode
of ``kempnerforge/model/attention.py:165-175,229-231`` with a mask among the new
tokens, RoPE rounded as the reference's eager ``apply_rope`` rounds it.
"""

from __future__ import annotations

import torch

from oracle import attention_ref as ref


def ancestors(parents: list[int]) -> list[list[int]]:
    """For each node, itself and its ancestors (parents come before children)."""
    out: list[list[int]] = []
    for i, p in enumerate(parents):
        assert -1 <= p < i
        out.append(([] if p < 0 else out[p]) + [i])
    return out


def rms_norm(x, w, eps):
    """RMSNorm over the last dimension in float32, rounded to x's dtype
    (``kempnerforge/model/norm.py:22-27``)."""
    f = x.float()
    f = f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + eps)
    return (f * w.float()).to(x.dtype)


def tree_step(q, k, v, kc, vc, lens, cos, sin, parents, counts=None, row_offset=0,
              q_norm=None, k_norm=None, eps=1e-5):
    """out (float64), the caches after the step, and per output element the sum
    of p |v| (what errors of the probabilities multiply).  ``parents``: one list
    per sequence.  Unused nodes: zeros, cache rows as they were."""
    B, N, Hq, D = q.shape
    Hkv = k.shape[2]
    rep = Hq // Hkv
    kc, vc = kc.clone(), vc.clone()
    out = torch.zeros(B, N, Hq, D, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        n = N if counts is None else int(counts[b])
        L = int(lens[b])
        anc = ancestors(parents[b][:n])
        qb, kb = q[b, :n], k[b, :n]
        if q_norm is not None:
            qb, kb = rms_norm(qb, q_norm, eps), rms_norm(kb, k_norm, eps)
        for i in range(n):
            at = L + len(anc[i]) - 1 - row_offset
            c, s = cos[at:at + 1], sin[at:at + 1]
            kc[b, :, L + i] = ref.apply_rope(kb[i][None, :, None], c, s)[0, :, 0]
            vc[b, :, L + i] = v[b, i]
        for i in range(n):
            at = L + len(anc[i]) - 1 - row_offset
            qi = ref.apply_rope(qb[i][None, :, None], cos[at:at + 1], sin[at:at + 1])[0, :, 0]
            rows = list(range(L)) + [L + j for j in anc[i]]
            kk, vv = kc[b][:, rows].double(), vc[b][:, rows].double()
            p = torch.softmax(
                (qi.double().view(Hkv, rep, D) @ kk.transpose(1, 2)) * D ** -0.5, dim=-1)
            out[b, i] = (p @ vv).view(Hq, D)
            mag[b, i] = (p @ vv.abs()).view(Hq, D)
    return out, kc, vc, mag


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
                    if torch.isnan(row).any():
                        w = None
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
                nxt = -1 if torch.isnan(logits[b, cur]).any() else best
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
