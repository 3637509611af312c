"""The native calls for several continuations of one prompt: what they answer and what
they leave to the checks in Python."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce
from kempnerforge_amd import _lib, ops
from test_gpu_speculative_calls import _bad

pytestmark = pytest.mark.gpu

BF, I32, F32 = torch.bfloat16, torch.int32, torch.float32


def new(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype, device=DEV)


def test_native_calls_refuse_every_other_form():
    """With all other arguments in their plain form, each argument in another one is
    answered with None (and nothing is launched: the caches stay)."""
    announce("native branch forms")
    G, W, N, Hq, Hkv, D, P, S, V = 2, 2, 3, 4, 2, 64, 8, 16, 9
    B, stream = G * W, torch.cuda.current_stream().cuda_stream
    kc, vc = new(B, Hkv, S, D), new(B, Hkv, S, D)
    branch = [new(B, N, Hq, D), new(B, N, Hkv, D), new(B, N, Hkv, D), new(G, Hkv, P, D),
              new(G, Hkv, P, D), new(G, dtype=I32), kc, vc, new(B, dtype=I32),
              new(P + S, D // 2, dtype=F32), new(P + S, D // 2, dtype=F32),
              torch.full((B,), N, dtype=I32, device=DEV), new(D, dtype=F32), new(D, dtype=F32),
              1e-5, 0, P, S, 0, stream]
    select = [new(G, W, V), new(G, W, dtype=F32), 3, 0, stream]
    reorder = [[kc], [vc], new(B, dtype=I32), new(G, W, dtype=I32), 0, stream]
    native = _lib.native()
    for f, args in ((native.branch, branch), (native.select, select), (native.reorder, reorder)):
        last = len(args) - 1  # (the stream: any number is one)
        for i, a in enumerate(args[:last]):
            if isinstance(a, torch.Tensor):
                bad = list(_bad(a))
                if f is native.select and i == 0:  # (fewer values of wider rows are a form of it)
                    bad[2] = new(G, W, 2 * V)[..., ::2]
            elif isinstance(a, list):
                bad = [[x] for x in _bad(a[0])] + [tuple(a), a * 2, [], [None], None]
            else:
                bad = [None, "x", 1 << 70, torch.tensor(1)] + ([7] if i >= last - 1 else [])
            for x in bad:
                got = f(*args[:i], x, *args[i + 1:])
                assert got is None, (f.__name__, i, x if not torch.is_tensor(x) else x.shape)
        assert f(*args) is not None
    torch.cuda.synchronize()


@pytest.mark.parametrize("D", [64, 96])
def test_other_forms_give_the_same(D):
    """Counts of 64 bits, strided queries, half-precision norm weights, a table of 64-bit
    numbers, strided scores, parents of another layout: the same results, to the last
    bit, as the plain forms."""
    announce(f"branch other forms {D}")
    g = torch.Generator().manual_seed(3)
    G, W, N, Hq, Hkv, P, S = 2, 3, 2, 4, 2, 40, 16
    B = G * W
    r = lambda *s: torch.randn(*s, generator=g).to(DEV, BF)  # noqa: E731
    q, k, v, kp, vp = r(B, N, Hq, D), r(B, N, Hkv, D), r(B, N, Hkv, D), r(G, Hkv, P, D), r(
        G, Hkv, P, D)
    kc, vc = r(B, Hkv, S, D), r(B, Hkv, S, D)
    cos, sin = torch.rand(P + S, D // 2, device=DEV), torch.rand(P + S, D // 2, device=DEV)
    plens, lens = new(G, dtype=I32) + 33, new(B, dtype=I32) + 5
    counts = torch.tensor([2, 1, 0, 2, 2, 1], dtype=I32, device=DEV)
    qn, kn = r(D), r(D)

    def call(q, counts, qn, cos, lens):
        kc1, vc1 = kc.clone(), vc.clone()
        out = ops.branch_decode_raw(q, k, v, kp, vp, plens, kc1, vc1, lens, cos, sin,
                                    rope_row_offset=0, max_prefix=P, max_len=S, counts=counts,
                                    q_norm_weight=qn, k_norm_weight=kn.float())
        return out, kc1, vc1

    plain = call(q, counts, qn.float(), cos, lens)
    wide = new(B, N, Hq, 2 * D)[..., :D]
    wide.copy_(q)
    for other in ((wide, counts, qn.float(), cos, lens), (q, counts.long(), qn.float(), cos, lens),
                  (q, counts, qn, cos, lens), (q, counts, qn.float(), cos.double(), lens)):
        assert all(torch.equal(a, b) for a, b in zip(call(*other), plain))

    x, s = r(G, W, 77), torch.randn(G, W, generator=g).to(DEV)
    best = ops.beam_select_raw(x, s, select=5)
    strided = new(G, 2 * W, dtype=F32)[:, ::2]
    strided.copy_(s)
    assert all(torch.equal(a, b) for a, b in zip(ops.beam_select_raw(x, strided, select=5), best))

    parents = torch.tensor([[1, 1, 0], [2, 0, 0]], dtype=I32, device=DEV)
    moved, same = [kc.clone()], [kc.clone()]
    other = [vc.clone()], [vc.clone()]
    ops.cache_reorder_raw(moved, other[0], lens, parents)
    ops.cache_reorder_raw(same, other[1], lens, parents.t().contiguous().t())
    assert torch.equal(moved[0], same[0]) and torch.equal(other[0][0], other[1][0])


def test_a_leaf_that_wants_gradients():
    """Serving operators: no graph is kept of them."""
    announce("branch no graph")
    q, k, v = (new(2, 1, h, 64).requires_grad_() for h in (4, 2, 2))
    out = ops.branch_decode_raw(q, k, v, new(1, 2, 8, 64), new(1, 2, 8, 64), new(1, dtype=I32),
                                new(2, 2, 8, 64), new(2, 2, 8, 64), new(2, dtype=I32),
                                new(16, 32, dtype=F32), new(16, 32, dtype=F32), rope_row_offset=0,
                                max_prefix=8, max_len=8)
    assert not out.requires_grad
    best, _, _ = ops.beam_select_raw(new(1, 2, 9).requires_grad_(), new(1, 2, dtype=F32), select=2)
    assert not best.requires_grad
    torch.cuda.synchronize()


@pytest.mark.parametrize("other", [False, True])
def test_what_is_out_of_range_raises_the_same_whatever_the_form(other):
    """Arguments out of their range raise ValueError where the native call meets them too
    (``other``: tensors that only the checks in Python take)."""
    announce(f"branch refusals of either form {other}")
    form = (lambda t: t.t().contiguous().t()) if other else (lambda t: t)
    scores = form(torch.zeros(2, 3, dtype=F32, device=DEV))
    x = new(2, 3, 40)
    for k in (0, -1, ops.BEAM_MAX_SELECT + 1, 1 << 40):
        with pytest.raises(ValueError, match="select must lie in"):
            ops.beam_select_raw(x, scores, select=k)
    with pytest.raises(ValueError, match="64 beams"):
        ops.beam_select_raw(new(2, 65, 9), form(new(2, 65, dtype=F32)), select=4)
    with pytest.raises(ValueError, match="beams of a group"):
        ops.beam_select_raw(new(2, 0, 9), form(new(2, 0, dtype=F32)), select=4)
    k = new(130, 1, 4, 8)
    k[:] = 3.0
    with pytest.raises(ValueError, match="at most 64 beams"):
        ops.cache_reorder_raw([k], [k.clone()], new(130, dtype=I32),
                              form(new(2, 65, dtype=I32)))
    torch.cuda.synchronize()
    assert (k == 3.0).all()
