"""How exact the verification's probabilities are (kf_verify_drafts): wherever the row's
maximum lies and however low the temperature, a drafted token is accepted at a random
number just below its probability and refused just above it."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce
from kempnerforge_amd import ops
from oracle import spec_ref

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32

# A row's sum: arguments off by 2^-23 of themselves (a difference, a product, the
# constant in float32), which times ln 2 and the mean |x| (below 12 here, the logarithm of
# 4000 values) is 12 ln 2 2^-23 = 2^-19.9; a hardware exponential 2^-22; 32 float32
# additions a batch, at most 31 2^-24 = 2^-19.05, half of it at the mean of a
# running sum.  Together below 2^-18.  The random number is rounded to float32 (2^-24).
EPS = 2.0 ** -18


def _rows(dtype, B, N, V, T, offset, seed):
    """Rows round ``offset`` whose favourite token holds a fair part of the mass, in
    steps of the temperature (or ties, where the type has no such steps)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, N, V, generator=g)
    fav = torch.randint(V, (B, N, 1), generator=g)
    x.scatter_(2, fav, 8.0 + torch.rand(B, N, 1, generator=g))
    x.scatter_(2, (fav + 1) % V, 8.5)
    return (offset + T * x.double()).to(dtype), fav


@pytest.mark.parametrize("T,offset", [(1.0, 0.0), (1.0, 30.0), (1.0, 1000.0), (1.0, -1000.0),
                                      (0.05, 25.0), (1e-3, 25.0), (1e-6, 23.5), (1e-6, 0.0),
                                      (50.0, 3.0), (0.7, 3e4)])
@pytest.mark.parametrize("dtype,way", [(F32, "all"), (F32, "walk"), (BF, "all"), (FH, "walk"),
                                       (F32, "drafts"), (FH, "drafts")])
def test_acceptance_at_the_probability(dtype, way, T, offset):
    announce(f"verify sums {dtype} {way} T={T} offset={offset}")
    # (trees of more than 2200 bytes a value go row by row down the path)
    B, N, V = (160 if dtype == F32 else 300, 4, 3999) if way == "walk" else (64, 2, 4000)
    logits, fav = _rows(dtype, B, N, V, T, offset, 1)
    p = torch.softmax(logits[:, 0].double() / T, -1)
    tokens = torch.zeros(B, N, dtype=torch.long)
    tokens[:, 1] = fav[:, 0, 0]
    border = p.gather(1, tokens[:, 1:2])[:, 0]
    draft, tol = None, EPS
    if way == "drafts":
        draft, _ = _rows(dtype, B, N - 1, V, T, offset, 2)
        draft[torch.arange(B), 0, tokens[:, 1]] = draft.amax(-1)[:, 0]  # (q about p)
        q = torch.softmax(draft[:, 0].double() / T, -1).gather(1, tokens[:, 1:2])[:, 0]
        border, tol = border / q, 2 * EPS
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    parents = torch.tensor([-1] + [0] * (N - 1), dtype=torch.int32) if way == "walk" else None
    asked = 0
    for side in (-1, 1):
        u = torch.full((B, N), 0.5)
        u[:, 1] = (border * (1 + side * tol)).float()
        ok = u[:, 1] < 1  # (a border past 1 is never asked for)
        u[:, 1].clamp_(max=1 - 2.0 ** -24)
        path, kept, _ = (t.cpu() for t in ops.verify_drafts_raw(
            dev(logits), dev(tokens), dev(u), temperature=T, parents=dev(parents),
            draft_logits=dev(draft)))
        # (behind a refused first child the walk tries the others, of token 0)
        taken = path[:, 1] == 1
        assert (taken | (kept == 1) | (path[:, 1] > 1)).all()
        assert (taken == (side < 0))[ok].all(), (side, border[ok & (taken != (side < 0))][:4])
        asked += int(ok.sum())
    # (a draft that gives its token no more than the target does has no border)
    assert way == "drafts" or asked >= B


def test_equal_top_logits_share_the_mass():
    """Two equal tops far above the rest at a temperature of 1e-6: each token is drawn in
    half of the draws."""
    announce("verify equal tops")
    B, V = 4096, 1000
    logits = torch.full((B, 1, V), 23.0, device=DEV)
    logits[:, :, [17, 900]] = 23.5
    u = (torch.arange(B, device=DEV, dtype=F32) / B)[:, None]
    tokens = torch.zeros(B, 1, dtype=torch.long, device=DEV)
    got = ops.verify_drafts_raw(logits, tokens, u, temperature=1e-6)[2].tolist()
    assert got == [17] * (B // 2) + [900] * (B // 2)


@pytest.mark.parametrize("way", ["all", "walk", "drafts"])
@pytest.mark.parametrize("T", [5e-324, 1e-300, 1e-40, 1e-38, 1e39, 1e46, 1e308])
def test_temperatures_at_the_ends_of_their_range(T, way):
    """The most likely tokens share the mass, or all tokens that are possible do."""
    announce(f"verify temperature {T} {way}")
    B, N, V = (160, 4, 600) if way == "walk" else (8, 2, 600)
    logits = torch.randn(B, N, V, generator=torch.Generator().manual_seed(0)).to(DEV)
    logits[:, :, 200:] = float("-inf")
    logits[:, :, [7, 150]] = 9.0
    share = 0.5 if T < 1 else 1 / 200
    tokens = torch.full((B, N), 7, device=DEV)
    u = torch.full((B, N), share * 0.999, device=DEV)
    u[B // 2:, 1] = share * 1.001
    draft = parents = None
    if way == "walk":
        tokens[:, 2:] = 300  # impossible
        parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=DEV)
    if way == "drafts":  # certain of the token
        draft = torch.full((B, 1, V), float("-inf"), device=DEV)
        draft[:, :, 7] = 0.0
    u[:, 0] = 0.9999
    _, kept, token = ops.verify_drafts_raw(logits, tokens, u, temperature=T, parents=parents,
                                           draft_logits=draft)
    assert kept.tolist() == [2] * (B // 2) + [1] * (B - B // 2)
    assert token.tolist() == [150 if T < 1 else 199] * B


@pytest.mark.parametrize("way", ["all", "walk"])
@pytest.mark.parametrize("dtype", [F32, FH])
def test_greedy_rows_without_a_distribution(dtype, way):
    """At temperature 0 too a row with +inf, or of -inf throughout, ends the path with no
    token: of node 0, and of a node further down."""
    announce(f"verify greedy bad rows {dtype} {way}")
    B, N, V = (400, 4, 700) if way == "walk" else (40, 4, 700)
    inf = float("inf")
    logits = torch.randn(B, N, V, generator=torch.Generator().manual_seed(0)).to(dtype)
    logits[:, :, 5] = 20.0
    for at in range(8):
        bad = logits[at::10, at % 2]
        if at < 2:
            bad[:, 333] = inf
        elif at < 4:
            bad[:] = -inf
        elif at < 6:
            bad[:, 699] = float("nan")
        else:
            bad[:, 6:] = -inf  # (a distribution)
    tokens = torch.full((B, N), 5)
    tokens[:, 3] = 0  # (what a row of -inf must not take)
    parents = None
    par = [[-1, 0, 1, 0]] * B if way == "walk" else [[-1, 0, 1, 2]] * B
    if way == "walk":
        parents = torch.tensor(par, dtype=torch.int32, device=DEV)
    got = ops.verify_drafts_raw(logits.to(DEV), tokens.to(DEV), torch.zeros(B, N, device=DEV),
                                temperature=0.0, parents=parents)
    path, kept, token = (t.tolist() for t in got)
    want = spec_ref.verify(logits, tokens, torch.zeros(B, N), 0.0, par)
    wrong = [b for b in range(B) if (path[b], kept[b], token[b]) != tuple(x[b] for x in want)]
    assert not wrong, wrong[:10]
    assert kept[:10] == [1, 2, 1, 2, 1, 2, 3, 3, 3, 3] and token[:10] == [-1] * 6 + [5] * 4
