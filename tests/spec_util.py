"""Inputs, tolerances and checks shared by the tests of speculative decoding."""

from __future__ import annotations

import torch

from gpu_util import half_ulp, seeded
from oracle import attention_ref as ref
from oracle import spec_ref

# relative step of a 32-bit float, and half the relative step of the type that the
# kernels' probabilities are rounded to before they multiply V (none in float32)
U32 = 2.0 ** -24
P_STEP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def trees(kind: str, B: int, N: int, seed: int = 0) -> list[list[int]]:
    """Parents per sequence."""
    if kind == "chain":
        return [list(range(-1, N - 1))] * B
    if kind == "star":  # every drafted token follows the last one
        return [[-1] + [0] * (N - 1)] * B
    if kind == "forest":  # nodes that follow the prefix directly
        return [[-1] * N] * B
    if kind == "binary":
        return [[-1] + [(i - 1) // 2 for i in range(1, N)]] * B
    g = torch.Generator().manual_seed(seed + N)
    return [[-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, N)]
            for _ in range(B)]


def tree_inputs(dtype, B, N, Hq, Hkv, D, Smax, seed=0):
    q, k, v = (seeded((B, N, h, D), seed + j, dtype) for j, h in enumerate((Hq, Hkv, Hkv)))
    kc, vc = (seeded((B, Hkv, Smax, D), seed + 10 + j, dtype) for j in range(2))
    cos, sin = ref.rope_tables(D, Smax, 5e5)
    return q, k, v, kc, vc, cos, sin


# what is left of q when it is the sum of two numbers of the type (float32: q itself)
Q_LEFT = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}


def check_rows(kcd, kc, k64, lens, counts, dtype, more=0.0):
    """The nodes' keys in the cache: the rotation in 32 bits (two products and a
    sum, 3 steps of 2^-24 of their magnitude, below 8 for N(0, 1) rows), rounded
    once; all other rows as they were.  ``more``: relative error before the
    rotation."""
    got, want = kcd.cpu(), kc.clone()
    for b, L in enumerate(lens):
        n = k64.shape[1] if counts is None else counts[b]
        rows = k64[b, :n].transpose(0, 1)
        new = got[b, :, L:L + n].double()
        bound = (half_ulp(rows, dtype) + 8 * (3 * U32 + more)) * (1 + 2.0 ** -7)
        assert ((new - rows).abs() <= bound).all(), b
        want[b, :, L:L + n] = got[b, :, L:L + n]
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def tree_bound(want, mag, dtype, D, keys, dot=12.0, moved=0.0):
    """Per element, how far an output may be from the 64-bit one over the same
    cache rows.

    Scores are sums of D products in 32 bits, each rounded at most once more than
    exactly (D + 8 steps of 2^-24 of the products' magnitudes, the rotation's
    among them, whose sum times D^-1/2 is at most ``dot``: the rows are N(0, 1), so
    it is below |q| |k| D^-1/2, about D^1/2 = 11.3 with the spread of the norms), and q
    enters them to Q_LEFT; a hardware exponential adds 2^-22.  Numerator and
    denominator both carry that, so the probabilities are off by twice it,
    relatively; sums over the keys add one step each, and P is rounded to the
    storage type before it multiplies V (half a step).  All of it multiplies sum
    p |v| = ``mag``.  The result is rounded once more.  ``moved``: what the scores
    are off by beyond that."""
    rel = (2 * (((D + 8) * U32 + Q_LEFT[dtype]) * dot + moved) + 2 ** -21
           + 2 * (keys + 8) * U32 + P_STEP[dtype])
    return rel * mag + half_ulp(want, dtype)


def check_tree(out, want, mag, dtype, D, keys, name, **more) -> float:
    got = out.detach().cpu().double()
    ratio = ((got - want).abs() / tree_bound(want, mag, dtype, D, keys, **more)).max().item()
    print(f"[{name}] worst error / bound {ratio:.3f}", flush=True)
    assert torch.isfinite(got).all() and ratio <= 1.0, (name, ratio)
    return ratio


def verify_inputs(dtype, B, N, V, seed=0, parents=None, temperature=1.0, drafts=False, peak=0.6):
    """Logits with one favourite a row, and drafts that hit it often."""
    g = torch.Generator().manual_seed(seed)
    t = temperature if temperature > 0 else 1.0
    logits = 2.0 * t * torch.randn(B, N, V, generator=g)
    fav = torch.randint(V, (B, N), generator=g)
    lift = t * (2.0 + torch.log(torch.tensor(V * peak / (1 - peak))))
    logits.scatter_(2, fav[..., None], lift.item())
    logits = logits.to(dtype)
    tokens = torch.randint(V, (B, N), generator=g)
    draft = None
    if drafts:
        draft = (logits[:, :-1].float() + t * torch.randn(B, N - 1, V, generator=g)).to(dtype)
        p = torch.softmax(draft.float() / t, -1).view(-1, V)
        if N > 1:
            tokens[:, 1:] = torch.multinomial(p, 1, generator=g).view(B, N - 1)
    else:
        for b in range(B):
            for i in range(1, N):
                if torch.rand((), generator=g) < 0.4:
                    tokens[b, i] = fav[b, max(parents[b][i], 0)]
    return logits, tokens, torch.rand(B, N, generator=g), draft


__all__ = ["trees", "tree_inputs", "check_rows", "tree_bound", "check_tree", "verify_inputs",
           "spec_ref"]
