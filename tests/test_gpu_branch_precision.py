"""How exact the attention behind shared prefixes (kf_attn_branch) is: its error against 64
bits is that of rounding the outputs, with nothing of q and P lost before."""

from __future__ import annotations

import pytest
import torch

from gpu_util import announce, seeded
from oracle import branch_ref
from spec_util import P_STEP, tree_bound
from test_gpu_branch import BF, F32, FH, inputs, reference, spread, step

CASES = [
    # dtype, (G, W, N, Hq, Hkv, D), prefix lengths, own lengths: a wavefront a share; tiles of 64
    # and of 128 rows over the prefix, beside wavefronts and beside tiles over the own rows; one
    # list of tiles over both; the way of other head sizes
    (BF, (1, 4, 1, 32, 8, 128), [900], [64] * 4),
    (FH, (2, 2, 2, 8, 2, 64), [900, 400], [64, 0, 9, 200]),
    (BF, (1, 12, 1, 8, 2, 128), [700], spread(12, 5, 90)),
    (FH, (1, 40, 1, 8, 2, 64), [500], spread(40, 5, 90)),
    (BF, (2, 2, 6, 8, 2, 128), [333, 800], [40, 0, 9, 130]),
    (FH, (1, 3, 40, 8, 2, 128), [1500], [30, 0, 9]),
    (BF, (1, 3, 40, 8, 2, 64), [60], [30, 200, 9]),
    (FH, (1, 2, 130, 8, 4, 64), [90], [30, 0]),
    (BF, (1, 3, 4, 6, 2, 96), [120], [9, 0, 30]),
]


def rms(x):
    return x.square().mean().sqrt().item()


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", CASES, ids=lambda c: "-".join(map(str, (str(c[0])[6:], *c[1]))))
def test_the_error_is_that_of_rounding_the_outputs(cfg):
    """The root mean square of the error is at most 1.05 times that of rounding the
    64-bit outputs.  What is left besides: rounding to bfloat16 costs 2^-9 / 3^1/2 =
    1.1e-3 of a value (float16 1.4e-4); q is kept to 2^-17 (2^-23) of itself, which over
    scores of N(0, 1) rows, a dot of D independent errors times D^-1/2, moves a
    probability by some 2^-17; P to 2^-17 (2^-22 and an absolute 2^-25); float32 sums and
    exponentials by some 2^-21 with the spread of their arguments.  Together below 3e-5
    (5e-6) of a value, a thirtieth of the rounding's, which adds its square: 0.1%."""
    dtype, (G, W, N, Hq, Hkv, D), plens, lens = cfg
    announce(f"branch precision {cfg}")
    x = inputs(dtype, G, W, N, Hq, Hkv, D, max(plens), max(lens) + N, seed=3)
    out, kcd, vcd = step(*x, plens, lens, max(plens), max(lens) + N)
    want, _ = reference(*x, kcd, vcd, plens, lens, None)
    ratio = rms(out.cpu().double() - want) / rms(want.to(dtype).double() - want)
    print(f"[{dtype} {cfg[1]}] error / rounding {ratio:.3f}", flush=True)
    assert ratio <= 1.05


@pytest.mark.parametrize("lost", ["p", "q"])
def test_a_lost_half_would_be_seen(monkeypatch, lost):
    """The 64-bit restatement with P, or q, rounded to one number of the type: more than
    1.05 times the rounding's error."""
    dtype, (G, W, N, Hq, Hkv, D), plens, lens = CASES[2]
    kp, vp, kc, vc = inputs(dtype, G, W, N, Hq, Hkv, D, max(plens), max(lens) + N, seed=3)[3:7]
    q = seeded((G * W, N, Hq, D), 9, torch.float32)  # (rotated: not of the type)
    rest = kp, vp, plens, kc, vc, lens, [N] * (G * W)
    want, _ = branch_ref.branch_attention(q, *rest)
    if lost == "q":
        got, _ = branch_ref.branch_attention(q.to(dtype), *rest)
    else:
        softmax = torch.softmax
        monkeypatch.setattr(torch, "softmax", lambda *a, **k: softmax(*a, **k).to(dtype).double())
        got, _ = branch_ref.branch_attention(q, *rest)
    assert rms(got.to(dtype).double() - want) > 1.05 * rms(want.to(dtype).double() - want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(FH, 128), (FH, 64), (BF, 128), (F32, 64), (FH, 96)])
@pytest.mark.parametrize("X", [13.0, 17.2])
@pytest.mark.parametrize("sink", ["prefix", "own"])
@pytest.mark.parametrize("W,N", [(2, 2), (9, 1), (3, 12), (1, 40)])
def test_a_key_that_takes_the_mass_and_gives_nothing(dtype, D, X, sink, W, N):
    """One key's score stands X above thousands of equal others and its value is zero (as
    the first token's of many models does), so the outputs are made of probabilities e^-X
    of the largest: all rounded alike, by the same error, if they are rounded."""
    announce(f"branch sink {dtype} {D} {X} {sink} {W} {N}")
    Hq, Hkv, P, L = 4, 2, 5000, 1300
    q, k, v, kp, vp, kc, vc, cos, sin = inputs(dtype, 1, W, N, Hq, Hkv, D, P, L + N, seed=5)
    cos, sin = torch.ones_like(cos), torch.zeros_like(sin)
    q[:] = 1.0
    k[:], kc[:], kp[:] = 0.0, 0.0, 0.0
    v[:], vc[:], vp[:] = v.abs() + 0.5, vc.abs() + 0.5, vp.abs() + 0.5
    kx, vx, at = (kp, vp, 3) if sink == "prefix" else (kc, vc, L - 5)
    kx[:, :, at, 0] = X * D ** 0.5
    vx[:, :, at] = 0.0
    x = q, k, v, kp, vp, kc, vc, cos, sin
    out, kcd, vcd = step(*x, [P], [L] * W, P, L + N)
    want, mag = reference(*x, kcd, vcd, [P], [L] * W, None)
    # (scores of X or 0; P is not what is rounded, so nothing is allowed for it)
    bound = tree_bound(want, mag, dtype, D, P + L + N, dot=X) - P_STEP[dtype] * mag
    ratio = ((out.cpu().double() - want).abs() / bound).max().item()
    print(f"[sink {dtype} {D} {X} {sink} {W} {N}] worst error / bound {ratio:.3f}", flush=True)
    assert ratio <= 1.0
