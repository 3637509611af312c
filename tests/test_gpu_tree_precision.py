"""How exact the attention of drafted trees (kf_attn_tree) is: its error against 64
bits is that of rounding the outputs, with nothing of q and P lost before."""

from __future__ import annotations

import pytest
import torch

from gpu_util import announce
from spec_util import P_STEP, tree_bound, tree_inputs, trees
from test_gpu_tree import BF, F32, FH, _reference, _step

pytestmark = pytest.mark.gpu

CASES = [
    # dtype, (B, N, Hq, Hkv, D), prefix lengths, tree: one, two and four row waves of
    # either head size, rows whose partials are merged and rows that are not, the way
    # of other head sizes
    (BF, (2, 8, 8, 2, 128), [900, 64], "binary"),
    (FH, (2, 8, 8, 2, 64), [900, 64], "random"),
    (BF, (2, 16, 8, 2, 64), [400, 1300], "random"),
    (FH, (2, 16, 8, 2, 128), [400, 1300], "binary"),
    (BF, (2, 40, 8, 2, 128), [333, 2000], "random"),
    (FH, (2, 40, 8, 2, 128), [333, 2000], "chain"),
    (BF, (1, 70, 12, 12, 64), [40], "binary"),
    (FH, (1, 200, 8, 4, 64), [10], "chain"),
    (BF, (2, 12, 6, 2, 96), [120, 9], "random"),
]


@pytest.mark.parametrize("cfg", CASES, ids=lambda c: "-".join(map(str, (str(c[0])[6:], *c[1], c[3]))))
def test_the_error_is_that_of_rounding_the_outputs(cfg):
    """The root mean square of the error is at most 1.05 times that of rounding the
    64-bit outputs.  What is left besides: rounding to bfloat16 costs 2^-9 / 3^1/2 =
    1.1e-3 of a value (float16 1.4e-4); q is kept to 2^-17 (2^-23) of itself, which over
    scores of N(0, 1) rows, a dot of D independent errors times D^-1/2, moves a
    probability by some 2^-17; P to 2^-17 (2^-22 and an absolute 2^-25); float32 sums and
    exponentials by some 2^-21 with the spread of their arguments.  Together below 3e-5
    (5e-6) of a value, a thirtieth of the rounding's, which adds its square: 0.1%.
    P in a single number of the type makes it 1.2 to 1.4 times, q 1.3 to 1.5."""
    dtype, (B, N, Hq, Hkv, D), lens, tree = cfg
    announce(f"tree precision {cfg}")
    q, k, v, kc, vc, cos, sin = tree_inputs(dtype, B, N, Hq, Hkv, D, max(lens) + N, seed=3)
    par = trees(tree, B, N)
    out, kcd, vcd = _step(q, k, v, kc, vc, lens, cos, sin, max(lens) + N,
                          None if tree == "chain" else par)
    want, _ = _reference(q, k, v, kc, vc, kcd, vcd, lens, cos, sin, par)
    rms = lambda x: x.square().mean().sqrt().item()  # noqa: E731
    ratio = rms(out.cpu().double() - want) / rms(want.to(dtype).double() - want)
    print(f"[{dtype} {cfg[1]}] error / rounding {ratio:.3f}", flush=True)
    assert ratio <= 1.05


@pytest.mark.parametrize("dtype,D", [(FH, 128), (FH, 64), (BF, 128), (F32, 64), (FH, 96)])
@pytest.mark.parametrize("X", [12.0, 14.0, 16.0, 17.2])
@pytest.mark.parametrize("first", [True, False])
def test_a_key_that_takes_the_mass_and_gives_nothing(dtype, D, X, first):
    """One key's score stands X above thousands of equal others and its value is zero (as
    the first token's of many models does), so the outputs are made of probabilities e^-X
    of the largest: all rounded alike, by the same error, if they are rounded."""
    announce(f"tree sink {dtype} {D} {X} {first}")
    B, N, Hq, Hkv, L = 1, 9, 4, 2, 7000
    q, k, v, kc, vc, cos, sin = tree_inputs(dtype, B, N, Hq, Hkv, D, L + N, seed=5)
    cos, sin = torch.ones_like(cos), torch.zeros_like(sin)
    q[:] = 1.0
    k[:], kc[:] = 0.0, 0.0
    sink = 3 if first else L - 5
    kc[:, :, sink, 0] = X * D ** 0.5
    vc[:], v[:] = vc.abs() + 0.5, v.abs() + 0.5
    vc[:, :, sink] = 0.0
    out, kcd, vcd = _step(q, k, v, kc, vc, [L], cos, sin, L + N)
    want, mag = _reference(q, k, v, kc, vc, kcd, vcd, [L], cos, sin, trees("chain", B, N))
    # (scores of X or 0; P is not what is rounded, so nothing is allowed for it)
    got = out.cpu().double()
    bound = tree_bound(want, mag, dtype, D, L + N, dot=X) - P_STEP[dtype] * mag
    ratio = ((got - want).abs() / bound).max().item()
    print(f"[sink {dtype} {D} {X} {first}] worst error / bound {ratio:.3f}", flush=True)
    assert ratio <= 1.0
