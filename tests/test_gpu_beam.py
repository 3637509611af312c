"""GPU parity of the beams' selection (kf_beam_select) and the caches' reordering
(kf_kv_cache_reorder) with the 64-bit restatement."""

from __future__ import annotations

import math

import pytest
import torch

from gpu_util import DEV, announce, half_ulp
from kempnerforge_amd import ops
from oracle import branch_ref

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
INF = float("inf")

# How far a row's log of its sum may be off.  A term 2^t is off by |t| 2^-24 (its
# argument's rounding) and |t| 2^-25 (log2 e in 32 bits) times ln 2, and by 2^-22 (the
# instruction); the mean of |t| over a distribution of V <= 2^17 values is at most 17 +
# log2 e; a thread's values are 128 at most, in sums of 8 and 16: 24 steps of 2^-24.
LSE = 18.5 * 1.5 * 2.0 ** -24 * 0.7 + 2.0 ** -22 + 24 * 2.0 ** -24


def inputs(dtype, G, W, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = 2.5 * torch.randn(G, W, V, generator=g)
    if V > 16:
        top = torch.randint(V, (G, W, 6), generator=g)
        x.scatter_(2, top, 6.0 + 2.0 * torch.randn(G, W, 6, generator=g))
    return x.to(dtype), -9.0 * torch.rand(G, W, generator=g)


def call(x, s, K):
    out = ops.beam_select_raw(x.to(DEV) if not x.is_cuda else x, s.to(DEV), select=K)
    torch.cuda.synchronize()
    return out


def check(x, s, K, got):
    """The scores at every place, to their error; the candidates the same where the
    64-bit values tell them apart by more than that, and in the order of places where
    they are equal."""
    G, W, V = x.shape
    best, parents, tokens = (t.cpu() for t in got)
    want, wp, wt = branch_ref.select(x, s, K)
    assert best.dtype == F32 and parents.dtype == torch.int32 and tokens.dtype == torch.int64
    none = torch.isinf(want)
    assert torch.equal(torch.isinf(best), none) and (best[none] == -INF).all()
    assert (parents[none] == -1).all() and (tokens[none] == -1).all()
    ok = ~none
    err = (best.double() - want)[ok].abs()
    assert (err <= LSE + half_ulp(want[ok], F32)).all(), err.max()
    total = branch_ref.totals(x, s).view(G, W * V)
    at = parents.long() * V + tokens
    for g in range(G):
        n = int(ok[g].sum())
        assert len(set(at[g, :n].tolist())) == n
        mine = total[g, at[g, :n]]
        assert ((mine - want[g, :n]).abs() <= 2 * LSE).all(), g
        # equal values of one beam: lowest token first
        for i in range(1, n):
            if mine[i] == mine[i - 1] and parents[g, i] == parents[g, i - 1]:
                assert tokens[g, i] > tokens[g, i - 1]
        apart = torch.ones(n, dtype=torch.bool)
        nxt = total[g].topk(min(n + 1, W * V)).values
        gap = (nxt[:-1] - nxt[1:])
        gap[gap == 0] = INF  # (equals have an order of their own)
        for i in range(n):
            near = [gap[j] for j in (i - 1, i) if 0 <= j < len(gap)]
            apart[i] = not near or min(near) > 2 * LSE
        assert torch.equal(parents[g, :n][apart], wp[g, :n][apart])
        assert torch.equal(tokens[g, :n][apart], wt[g, :n][apart])


@pytest.mark.parametrize("dtype,G,W,V,K", [
    (F32, 1, 1, 1, 1), (F32, 1, 4, 1, 8), (BF, 1, 1, 7, 7), (BF, 2, 3, 5, 9), (FH, 3, 1, 300, 2),
    (F32, 1, 4, 32000, 8), (BF, 3, 5, 50001, 10), (FH, 2, 4, 50001, 5), (BF, 5, 8, 8192, 16),
    (F32, 2, 3, 4097, 6), (BF, 1, 64, 1000, 128), (F32, 2, 16, 3001, 32), (FH, 1, 33, 2048, 47),
    (BF, 2, 2, 33000, 48), (BF, 2, 7, 1234, 49), (BF, 16, 8, 131072, 16), (F32, 64, 8, 40003, 16),
    (BF, 9, 64, 9000, 128),
])
def test_against_64_bits(dtype, G, W, V, K):
    announce(f"select {dtype} {G} {W} {V} {K}")
    x, s = inputs(dtype, G, W, V, seed=V + K)
    check(x, s, K, call(x, s, K))


@pytest.mark.parametrize("dtype,G,W,V,K", [
    (F32, 1, 64, 40003, 64), (F32, 2, 33, 40003, 128), (BF, 1, 64, 40003, 3), (FH, 1, 3, 131072, 128),
    (F32, 1, 5, 131072, 40),
])
def test_more_slices_than_threads_and_fewer(dtype, G, W, V, K):
    """A group's slices against the 256 threads that look through their candidates: several
    a thread, several threads a slice, a number that does not divide them."""
    announce(f"select slices {dtype} {G} {W} {V} {K}")
    x, s = inputs(dtype, G, W, V, seed=V + K)
    check(x, s, K, call(x, s, K))


@pytest.mark.parametrize("dtype,W,V,K,ruling", [
    (BF, 16, 131072, 128, 1), (BF, 16, 131072, 128, 3), (F32, 9, 60001, 128, 2), (FH, 64, 20000, 100, 4),
    (BF, 16, 131072, 128, 11), (BF, 12, 131072, 41, 2), (F32, 33, 40003, 33, 1),
])
def test_few_beams_rule(dtype, W, V, K, ruling):
    """The scores of some beams are so far above the others' that all are picked of them:
    many candidates a slice."""
    announce(f"select ruling {dtype} {W} {V} {K} {ruling}")
    x, s = inputs(dtype, 2, W, V, seed=V + ruling)
    s[0, -ruling:] += 60.0
    s[1, :ruling] += 60.0
    out = call(x, s, K)
    assert (out[1][0] >= W - ruling).all() and (out[1][1] < ruling).all()
    check(x, s, K, out)


@pytest.mark.parametrize("dtype,fill", [(BF, 0.0), (F32, -3.5), (FH, 2.0)])
@pytest.mark.parametrize("K", [4, 64])
def test_equal_values(dtype, fill, K):
    """Rows of one value, and of two: the lowest beams and tokens."""
    announce(f"select equals {dtype} {K}")
    x = torch.full((2, 3, 5003), fill, dtype=dtype)
    x[1, :, ::2] += 1
    s = torch.zeros(2, 3)
    best, parents, tokens = (t.cpu() for t in call(x, s, K))
    assert (parents == 0).all()
    assert torch.equal(tokens[0], torch.arange(K)) and torch.equal(tokens[1], 2 * torch.arange(K))
    check(x, s, K, (best, parents, tokens))


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("K,allowed", [(8, 3), (16, 0), (128, 60), (48, 47), (5, 5)])
@pytest.mark.parametrize("lead", [0, 5])
def test_masked_by_the_lowest_value(dtype, K, allowed, lead):
    """All tokens but a few hold the type's lowest value (another mask than -inf): they
    follow those that are left, lowest first; slices of nothing else."""
    announce(f"select lowest {dtype} {K} {allowed} {lead}")
    V, G, W = 40003, 2, 2
    g = torch.Generator().manual_seed(5 + K)
    x = torch.full((G, W, V), torch.finfo(dtype).min, dtype=dtype)
    for i in range(G):
        for w in range(W):
            at = torch.randperm(V, generator=g)[:allowed]
            x[i, w, at] = torch.randn(allowed, generator=g).to(dtype)
    x[1, 0, ::3] = -INF
    s = torch.tensor([[-0.5, 0.0], [0.0, -0.25]])
    buf = torch.zeros(G * W * V + lead, dtype=dtype, device=DEV)
    view = buf[lead:].view(G, W, V)
    view.copy_(x)
    best, parents, tokens = (t.cpu() for t in call(view, s, K))
    want = branch_ref.select(x, s, K)[0]
    # (the largest are some 3.4e38: the error is relative there)
    assert torch.isfinite(best).all()
    assert ((best.double() - want).abs() <= LSE + half_ulp(want, F32)).all()
    # each beam's tokens: those allowed by value, then masked ones, lowest first
    for i in range(G):
        for w in range(W):
            mine = tokens[i][parents[i] == w]
            vals = x[i, w].float()[mine]
            assert (vals[:-1] >= vals[1:]).all() and not torch.isinf(vals).any()
            low = mine[vals == torch.finfo(dtype).min]
            order = (x[i, w] == torch.finfo(dtype).min).nonzero()[:, 0]
            assert torch.equal(low, order[:len(low)])
            left = int((x[i, w].float() > torch.finfo(dtype).min).sum())
            assert len(low) == 0 or len(mine) - len(low) == left


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logits_of_any_size(dtype):
    """Largest logits from 2^100 to the type's largest value, of either sign: all of the
    probability lies with them."""
    announce(f"select far out {dtype}")
    V, top = 20011, torch.finfo(dtype).max
    for at, far in enumerate((2.0 ** 100, 2.0 ** 126, -(2.0 ** 126), 2.0 ** 127, top, -(2.0 ** 127))):
        x = torch.full((1, 2, V), -top, dtype=dtype)
        x[0, 0, 7 + at::911] = far
        x[0, 1] = torch.randn(V, generator=torch.Generator().manual_seed(at)).to(dtype)
        n = len(range(7 + at, V, 911))
        s = torch.tensor([[0.0, -3.0]])
        best, parents, tokens = (t.cpu() for t in call(x, s, 9))
        want, wp, wt = branch_ref.select(x, s, 9)
        assert torch.equal(parents, wp) and torch.equal(tokens, wt), far
        assert ((best.double() - want).abs() <= LSE + half_ulp(want, F32)).all()
        assert n > 9 and (parents == 0).all()


# Magnitudes of masks and of favourites that are no powers of two, which a rounded multiple of
# log2 e is not exact for.
FAR = [1e4, 1e7, 3e8, 1e9, 1.3e9, 3e9, 1e10, 1e12, 1e15, 1e20, 1e30, 1e37, 3e38]


def _far_rows(dtype, V, far, kind, seed):
    """One row a kind: few tokens allowed (most threads hold nothing else than the mask);
    a thread's first granules masked, the others not; its last ones; the first by the type's
    lowest value, the others by the mask but for a few."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(V, generator=g)
    e = 16 // torch.empty((), dtype=dtype).element_size()
    late = torch.arange(V) // (256 * 4 * e) % 2 == 1  # granules 4 .. 7 of the threads
    few = torch.zeros(V, dtype=torch.bool)
    few[torch.randperm(V, generator=g)[:23]] = True
    if kind == "few":
        x[~few] = far
    elif kind == "first":
        x[~late] = far
    elif kind == "last":
        x[late] = far
    else:
        x[~few] = far
        x[~late & ~few] = torch.finfo(dtype).min
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["few", "first", "last", "two masks"])
@pytest.mark.parametrize("far", FAR)
def test_masks_of_any_size(dtype, kind, far):
    """Tokens masked by -far: those that are left are picked in order, whatever the mask,
    and the masked ones behind them by the lowest token."""
    announce(f"select mask {dtype} {kind} {far}")
    V, K = 40003, 40
    x = torch.stack([_far_rows(dtype, V, -far, kind, 10 * w) for w in range(3)])
    s = torch.tensor([[-0.3, 0.0, -1.7]])
    # three beams of one prompt, as many candidates as are left of one
    check(x[None], s, 20, call(x[None], s, 20))
    # each by itself, the masked ones among the candidates
    best, parents, tokens = (t.cpu() for t in call(x[:, None], s.view(3, 1), K))
    want, wp, wt = branch_ref.select(x[:, None], s.view(3, 1), K)
    assert torch.equal(parents, wp) and torch.equal(tokens, wt)
    assert ((best.double() - want).abs() <= LSE + half_ulp(want, F32)).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("rest", [0.0, -1.0])
def test_favourites_of_any_size(dtype, far, rest):
    """Largest logits of +far beside ordinary ones, or among -far: all of the probability
    lies with them, and a row of nothing else is the even distribution."""
    announce(f"select favourites {dtype} {far} {rest}")
    V, n = 40003, 11
    g = torch.Generator().manual_seed(int(far) % 1000)
    x = torch.randn(1, 3, V, generator=g) + rest * far
    hot = torch.stack([torch.randperm(V, generator=g)[:n] for _ in range(3)])
    x[0].scatter_(1, hot, far)
    x[0, 2] = far
    x = x.to(dtype)
    for third in (7.0, 9.0):  # (behind the other two's favourites, and in front of them)
        s = torch.tensor([[-0.25, -0.5, third]])
        best, parents, tokens = (t.cpu() for t in call(x, s, 2 * n))
        want, wp, wt = branch_ref.select(x, s, 2 * n)
        assert torch.equal(parents, wp) and torch.equal(tokens, wt)
        assert ((best.double() - want).abs() <= LSE + half_ulp(want, F32)).all()


@pytest.mark.parametrize("at", [2.0 ** 24, -3e7, 1e8, -1.5e9, 2.0 ** 30 - 64])
def test_sums_of_far_logits(at):
    """Logits a few units (of their last place) about one of 2^24 to 2^30: the sums keep the
    terms that are left, as exactly as of other logits (the differences are whole numbers)."""
    announce(f"select far sums {at}")
    ulp = 2.0 ** (math.frexp(at)[1] - 24)
    g = torch.Generator().manual_seed(2)
    x = (at + ulp * torch.randint(-5, 6, (2, 3, 9001), generator=g).double()).float()
    s = -torch.rand(2, 3, generator=g)
    best, parents, tokens = (t.cpu() for t in call(x, s, 6))
    want, wp, wt = branch_ref.select(x, s, 6)
    assert torch.equal(parents, wp) and torch.equal(tokens, wt)
    assert ((best.double() - want).abs() <= LSE + half_ulp(want, F32)).all()


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("V", [300, 32000, 131072, 1 << 20])
def test_how_exact_a_rows_sum_is(dtype, V):
    """Scores that bring the best candidate's total to zero, so that its rounding hides
    nothing: it is off by what the log of the row's sum is, 4e-6 at most as the header says
    (LSE with 21.5 for 18.5, |log2 p| of 2^20 values, and 2.25 steps of it: 3.7e-6)."""
    announce(f"select sums {dtype} {V}")
    for spread in (0.01, 1.0, 8.0):
        g = torch.Generator().manual_seed(V)
        x = (spread * torch.randn(8, 1, V, generator=g)).to(dtype)
        top = x.double().amax(-1)
        lse = torch.logsumexp(x.double(), -1)
        s = (lse - top).float()
        err = (call(x, s, 1)[0].cpu().double() - (s.double() + top - lse)).abs().max().item()
        print(f"[sums {dtype} {V} {spread}] off by {err:.2e}", flush=True)
        assert err <= 4e-6


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("V", [1, 3, 9, 40003])
@pytest.mark.parametrize("score", [0.0, -7.25])
def test_beams_sure_of_their_next_token_are_equals(dtype, V, score):
    """One token has all of a row's probability (or is all there is), whatever its logit: its
    total is the beam's score, to the last bit, and equal scores go to the lowest beams."""
    announce(f"select sure {dtype} {V} {score}")
    G, W = 3, 16
    g = torch.Generator().manual_seed(V)
    top = (20 * torch.randn(G, W, 1, generator=g)).to(dtype).double()
    x = top - 60.0 - torch.rand(G, W, V, generator=g).double()
    at = torch.randint(V, (G, W, 1), generator=g)
    x = x.scatter(2, at, top).to(dtype)
    s = torch.full((G, W), score)
    best, parents, tokens = (t.cpu() for t in call(x, s, W))
    assert (best == score).all() and torch.equal(tokens, at[..., 0])
    assert torch.equal(parents, torch.arange(W).int().expand(G, W))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("K,hot", [(16, 10), (48, 40), (100, 40), (3, 2)])
@pytest.mark.parametrize("lead", [0, 3])
def test_values_ordered_against_the_threads(dtype, K, hot, lead):
    """All of the large values lie with few threads: more of them pass the bound on the
    K-th largest than are gathered at once."""
    announce(f"select hot lanes {dtype} {K} {hot} {lead}")
    V, e = 40000, 16 // torch.empty((), dtype=dtype).element_size()
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 2, V, generator=g)
    lane = (torch.arange(V) + lead) // e % 64
    x = torch.where(lane < hot, x.abs() + 8, x).to(dtype)
    s = torch.tensor([[-0.3, 0.0]])
    buf = torch.zeros(2 * V + lead + e, dtype=dtype, device=DEV)
    view = buf[lead:lead + 2 * V].view(1, 2, V)
    view.copy_(x)
    check(x, s, K, call(view, s, K))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("K,hot", [(16, 10), (48, 40), (100, 40), (3, 2)])
@pytest.mark.parametrize("lead", [0, 3])
def test_values_of_few_threads(dtype, K, hot, lead):
    """The same by the places that the threads take: granules counted from a row's first
    value, whatever its alignment."""
    announce(f"select hot threads {dtype} {K} {hot} {lead}")
    V, e = 40000, 16 // torch.empty((), dtype=dtype).element_size()
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, 2, V, generator=g)
    x = torch.where(torch.arange(V) // e % 64 < hot, x.abs() + 8, x).to(dtype)
    s = torch.tensor([[-0.3, 0.0]])
    buf = torch.zeros(2 * V + lead + e, dtype=dtype, device=DEV)
    view = buf[lead:lead + 2 * V].view(1, 2, V)
    view.copy_(x)
    check(x, s, K, call(view, s, K))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_beams_without_candidates(dtype):
    """Beams that are not in use, rows that are no distribution, tokens of no
    probability."""
    announce(f"select none {dtype}")
    G, W, V, K = 4, 5, 3000, 10
    x, s = inputs(dtype, G, W, V)
    s[0, 1], s[0, 3], s[1, 2] = -INF, float("nan"), INF
    x[1, 0, 2999], x[1, 1, 5], x[1, 3] = float("nan"), INF, -INF
    x[2, :, 4:] = -INF              # twenty candidates
    x[3, :, 1:] = -INF              # five
    out = call(x, s, K)
    check(x, s, K, out)
    best, parents, tokens = (t.cpu() for t in out)
    assert set(parents[0].tolist()) <= {0, 2, 4} and (parents[1] == 4).all()
    assert (tokens[3, :5] == 0).all() and (tokens[3, 5:] == -1).all() and (best[3, 5:] == -INF).all()
    # nothing at all
    best, parents, tokens = call(x, torch.full((G, W), -INF), K)
    assert (best == -INF).all() and (parents == -1).all() and (tokens == -1).all()


@pytest.mark.parametrize("shift", [0.0, 1000.0, -3e4])
def test_a_constant_moves_nothing(shift):
    """Rows of whole numbers, so that the constant is exact."""
    announce(f"select shift {shift}")
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-20, 20, (2, 4, 9001), generator=g).float()
    s = -torch.rand(2, 4, generator=g)
    a, b = call(x, s, 8), call(x + shift, s, 8)
    assert torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
    assert (a[0] - b[0]).abs().max().item() <= 2 * LSE + 2.0 ** -20


def test_scores_far_apart():
    """A beam that lies far behind is not picked, and one far down picks among its own."""
    announce("select far scores")
    x, s = inputs(F32, 2, 3, 5000)
    s[0], s[1] = torch.tensor([0.0, -1e4, -2e30]), torch.tensor([-1e4, -1e4 - 50, -3e4])
    check(x[:1], s[:1], 6, call(x[:1], s[:1], 6))
    _, parents, tokens = (t.cpu() for t in call(x[1:], s[1:], 6))
    assert (parents == 0).all()
    assert torch.equal(tokens[0], x[1, 0].sort(descending=True, stable=True).indices[:6])


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("score", [-1e12, -1e17, -1e30, 2e38])
@pytest.mark.parametrize("V,K", [(300, 9), (40003, 9), (131072, 40), (40003, 128)])
def test_scores_that_leave_no_bits_for_logits(dtype, score, V, K):
    """Beams whose score is so far out (one that took a masked token) that 64 bits do not tell
    their totals apart: of equal totals the lowest beam's, and of a beam the largest
    logits, equals by the lowest token, as of any other beam."""
    announce(f"select absorbed {dtype} {score} {V} {K}")
    x, _ = inputs(dtype, 3, 3, V, seed=K)
    s = torch.full((3, 3), -INF)
    s[0, 1] = score               # one beam
    s[1, 1:] = score              # two equal ones
    s[2] = torch.tensor([score * 1.5, 0.0, score])  # behind (in front of) an ordinary one
    x[2, 1, K // 2:] = -INF
    best, parents, tokens = (t.cpu() for t in call(x, s, K))
    order = x.double().sort(dim=-1, descending=True, stable=True).indices
    if abs(score) >= 1e17:        # (ulp / 2 above any difference of theirs)
        assert (parents[:2] == 1).all() and torch.equal(tokens[:2], order[:2, 1, :K])
    n = K // 2
    if score < 0:
        assert (parents[2, :n] == 1).all() and torch.equal(tokens[2, :n], order[2, 1, :n])
        assert (parents[2, n:] == 2).all() and torch.equal(tokens[2, n:], order[2, 2, :K - n])
    else:
        assert (parents[2] == 0).all() and torch.equal(tokens[2], order[2, 0, :K])
    for g, w in ((0, 1), (1, 1), (1, 2)):  # each beam's own, whatever the other's
        mine = tokens[g][parents[g] == w]
        assert torch.equal(mine, order[g, w, :len(mine)])
    assert torch.isfinite(best).all()


def test_strided_logits():
    """The last token's logits of every sequence: rows apart, off 16-byte boundaries."""
    announce("select strides")
    B, T, V, W = 6, 3, 4001, 3
    x, _ = inputs(BF, B, T, V)
    s = -torch.rand(2, W, generator=torch.Generator().manual_seed(0))
    last = x.to(DEV)[:, -1].view(2, W, V)
    assert not last.is_contiguous()
    check(x[:, -1].reshape(2, W, V), s, 6, call(last, s, 6))


def test_graph_replays():
    announce("select graph")
    x, s = inputs(BF, 3, 4, 20000)
    x, s = x.to(DEV), s.to(DEV)
    ops.beam_select_raw(x, s, select=8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.beam_select_raw(x, s, select=8)
    for rep in range(4):
        a, b = inputs(BF, 3, 4, 20000, seed=10 + rep)
        if rep == 2:
            b[1, 1:] = -INF
        x.copy_(a)
        s.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = ops.beam_select_raw(x, s, select=8)
        assert all(torch.equal(p, q) for p, q in zip(got, want)), rep


# ------------------------------------------------------------------ reorder
def _caches(dtype, n, B, H, S, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, H, S, D, generator=g).to(dtype) for _ in range(2 * n)]


def _reorder(caches, lens, parents, to=lambda t: t.to(DEV)):
    n = len(caches) // 2
    dev = [to(t) for t in caches]
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    ops.cache_reorder_raw(dev[:n], dev[n:], lens_d,
                          torch.tensor(parents, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert lens_d.tolist() == list(lens)
    return dev


@pytest.mark.parametrize("dtype,n,parents,H,S,D,lens", [
    (BF, 2, [[0]], 2, 9, 64, [5]),
    (BF, 3, [[1, 0]], 2, 9, 64, [5, 5]),                      # a swap
    (BF, 2, [[0, 0, 1, 3], [3, 2, 1, 0]], 8, 70, 128, [64, 64, 64, 64, 1, 33, 70, 0]),
    (FH, 1, [[2, 2, 2, 2, 2]], 1, 40, 128, [40, 3, 17, 9, 0]),
    (F32, 2, [[1, 2, 0], [2, 0, 2]], 2, 33, 64, [33, 12, 7, 1, 2, 3]),  # a cycle
    (BF, 2, [[(5 * w + 3) % 9 for w in range(9)]], 2, 300, 64, list(range(9, 18))),
    (BF, 1, [[(7 * w) % 16 for w in range(16)]] * 2, 2, 129, 128, [128 - w for w in range(32)]),
    (BF, 1, [[(3 * w + 1) % 17 // 2 for w in range(17)]], 1, 50, 128, [50] * 17),
    (F32, 1, [[(11 * w + 5) % 64 for w in range(64)]], 1, 20, 128, [20 - w % 5 for w in range(64)]),
    (BF, 2, [[1, 0, 0]], 3, 21, 6, [21, 20, 0]),              # rows of 12 bytes
    (FH, 1, [[2, 0, 1]], 2, 11, 81 * 2, [11, 4, 9]),
    (BF, 70, [[1, 1]], 1, 5, 64, [5, 4]),                     # more caches than one launch takes
    (BF, 2, [[-1, 0, 9, 1]], 2, 12, 64, [12, 3, 5, 6]),       # parents out of range
    (BF, 2, [[1, 0, 3, 2]], 2, 12, 64, [12, 13, -1, 6]),      # lengths out of range
])
def test_reorder(dtype, n, parents, H, S, D, lens):
    announce(f"reorder {dtype} {parents} {S} {D}")
    caches = _caches(dtype, n, len(lens), H, S, D)
    got = _reorder(caches, lens, parents)
    for c, (x, y) in enumerate(zip(caches, got)):
        assert torch.equal(y.cpu(), branch_ref.reorder(x, lens, parents)), c


def test_reorder_misaligned():
    announce("reorder misaligned")

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        o = buf[1:].view(t.shape)
        o.copy_(t)
        return o

    lens, parents = [30, 7, 30], [[2, 2, 0]]
    caches = _caches(BF, 2, 3, 2, 31, 128)
    for x, y in zip(caches, _reorder(caches, lens, parents, off)):
        assert torch.equal(y.cpu(), branch_ref.reorder(x, lens, parents))


def test_reorder_leaves_nan_rows_alone():
    announce("reorder NaN")
    caches = _caches(BF, 1, 4, 2, 20, 64)
    for t in caches:
        t[:, :, 9:] = float("nan")
        t[2, :, 3] = INF
    parents = [[2, 0, 1, 2]]
    for x, y in zip(caches, _reorder(caches, [9] * 4, parents)):
        want = branch_ref.reorder(x, [9] * 4, parents)
        assert torch.equal(y.cpu().view(torch.int16), want.view(torch.int16))


def test_reorder_captured():
    """Replayed with other parents and lengths."""
    announce("reorder graph")
    caches = [t.to(DEV) for t in _caches(BF, 2, 4, 2, 50, 64)]
    lens = torch.tensor([3, 4, 5, 6], dtype=torch.int32, device=DEV)
    par = torch.tensor([[1, 0, 3, 2]], dtype=torch.int32, device=DEV)
    ops.cache_reorder_raw(caches[:2], caches[2:], lens, par)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.cache_reorder_raw(caches[:2], caches[2:], lens, par)
    for rep in range(4):
        par.copy_(torch.tensor([[rep, 3, 0, (rep + 1) % 4]], dtype=torch.int32))
        lens.copy_(torch.tensor([50 - rep, 7, 20 * rep % 51, 33], dtype=torch.int32))
        before = [t.cpu() for t in caches]
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(before, caches):
            assert torch.equal(y.cpu(), branch_ref.reorder(x, lens.tolist(), par.tolist())), rep


def test_reorder_past_32_bit_offsets():
    announce("reorder long caches")
    k = torch.zeros(4, 2, 1 << 22, 128, dtype=BF, device=DEV)  # 8.6 GB
    v = torch.zeros(4, 2, 1 << 22, 128, dtype=BF, device=DEV)
    rows = torch.randn(2, 4, 2, 40, 128, generator=torch.Generator().manual_seed(0)).bfloat16()
    at = (1 << 22) - 40
    for t, r in zip((k, v), rows):
        t[:, :, at:] = r.to(DEV)
    parents = [[3, 0, 0, 1]]
    lens = torch.tensor([(1 << 22)] * 4, dtype=torch.int32, device=DEV)
    ops.cache_reorder_raw([k], [v], lens, torch.tensor(parents, dtype=torch.int32, device=DEV))
    for t, r in zip((k, v), rows):
        assert torch.equal(t[:, :, at:].cpu(), branch_ref.reorder(r, [40] * 4, parents))
