"""GPU checks of the verification of drafted tokens (kf_verify_drafts) and of the
accepted path's move in the caches (kf_kv_cache_keep)."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce, seeded
from kempnerforge_amd import ops
from spec_util import spec_ref, trees, verify_inputs

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731


def _verify(logits, tokens, u, T, parents=None, counts=None, drafts=None):
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    path, kept, token = ops.verify_drafts_raw(dev(logits), dev(tokens), dev(u), temperature=T,
                                              parents=i32(parents), counts=i32(counts),
                                              draft_logits=dev(drafts))
    torch.cuda.synchronize()
    return path.tolist(), kept.tolist(), token.tolist()


CASES = [
    # dtype, B, N, V, tree, temperature, drafts, counts
    (F32, 1, 1, 50, "chain", 1.0, False, None),          # no drafts: a plain draw
    (F32, 6, 5, 97, "chain", 1.0, True, None),
    (F32, 8, 5, 32000, "chain", 0.7, True, None),
    (BF, 8, 6, 1000, "chain", 1.3, True, [6, 1, 0, 3, 2, 6, 5, 4]),
    (FH, 5, 9, 50001, "chain", 1.0, True, None),         # rows off 16-byte boundaries
    (BF, 6, 16, 4096, "binary", 1.0, False, None),
    (BF, 6, 31, 8191, "random", 0.6, False, [31, 3, 9, 0, 1, 20]),
    (FH, 6, 12, 1, "star", 1.0, False, None),            # a vocabulary of one
    (FH, 6, 12, 7, "star", 2.0, False, None),            # repeated tokens among siblings
    (F32, 4, 64, 131072, "random", 1.0, False, None),
    (F32, 3, 256, 300, "random", 1.0, False, None),
    (BF, 24, 48, 1001, "random", 1.0, False, [48, 0, 30] * 8),  # many nodes: row by row
    (FH, 24, 60, 515, "binary", 0.0, False, None),
    (F32, 70, 33, 333, "chain", 1.0, False, None),       # a long chain: all rows
    (BF, 8, 20, 1001, "random", 0.0, False, None),       # greedy
    (FH, 8, 6, 50001, "chain", 0.0, False, [6, 6, 0, 2, 1, 6, 6, 6]),
    (F32, 4, 3, 200000, "chain", 0.0, False, None),
]


@pytest.mark.parametrize("cfg", CASES, ids=lambda c: "-".join(map(str, (str(c[0])[6:], *c[1:7]))))
def test_against_64_bits(cfg):
    """Whole numbers, equal to the walk in 64 bits: a test or a draw is decided
    otherwise only within the kernel's error of a border (about 1e-7 of its
    interval), which these inputs do not meet."""
    dtype, B, N, V, tree, T, drafts, counts = cfg
    announce(f"verify {cfg}")
    par = trees(tree, B, N)
    for seed in range(3):
        logits, tokens, u, draft = verify_inputs(dtype, B, N, V, seed, par, T, drafts)
        got = _verify(logits, tokens, u, T, None if tree == "chain" else par, counts, draft)
        want = spec_ref.verify(logits, tokens, u, T, par, counts, draft)
        assert got == tuple(want), seed


def test_greedy_takes_the_lowest_of_equals():
    announce("verify ties")
    logits = torch.zeros(2, 3, 5000, dtype=BF)
    logits[0, 0, [700, 4999, 31]] = 3.0
    logits[1, :, 4000:] = 1.0
    tokens = torch.tensor([[0, 31, 0], [0, 4000, 4000]])
    got = _verify(logits, tokens, torch.zeros(2, 3), 0.0)
    assert got == ([[0, 1, 2], [0, 1, 2]], [3, 3], [0, 4000])


def test_uniforms_at_their_ends():
    """u = 0 accepts any drafted token of positive probability and draws the first
    possible one; the largest u accepts only what is certain and draws the last."""
    announce("verify uniform ends")
    V, last = 1000, 1.0 - 2.0 ** -24
    logits = torch.full((2, 2, V), float("-inf"))
    logits[:, 0, [10, 500, 900]] = 0.0
    logits[:, 1, 77] = -4.0
    tokens = torch.tensor([[0, 500], [0, 500]])
    u = torch.tensor([[0.0, 0.0], [last, last]])
    assert _verify(logits, tokens, u, 1.0) == ([[0, 1], [0, -1]], [2, 1], [77, 900])
    # the only token: certain at every u
    tokens[:, 1] = 77
    only = logits.roll(-1, 1)  # node 0 has only 77 left
    assert _verify(only, tokens, u, 1.0) == ([[0, 1], [0, 1]], [2, 2], [10, 900])


def test_draft_equal_to_the_target_is_always_accepted():
    announce("verify q = p")
    B, N, V = 64, 6, 777
    logits, _, u, _ = verify_inputs(F32, B, N, V, 3, trees("chain", B, N))
    p = torch.softmax(logits[:, :-1], -1).view(-1, V)
    tokens = torch.zeros(B, N, dtype=torch.long)
    tokens[:, 1:] = torch.multinomial(p, 1, generator=torch.Generator().manual_seed(1)).view(B, -1)
    _, kept, _ = _verify(logits, tokens, u, 1.0, drafts=logits[:, :-1].clone())
    assert kept == [N] * B


@pytest.mark.parametrize("drafts", [True, False])
def test_emitted_tokens_follow_the_target(drafts):
    """The first emitted token (the accepted node's, or the draw) over 200000
    sequences: every token's share is within 5 standard deviations of the
    target's probability (16 tokens: a fair sampler fails once in 10^5 runs; the
    seeds are fixed)."""
    announce(f"verify distribution drafts={drafts}")
    B, V, N = 50000, 16, 2 if drafts else 4
    g = torch.Generator(device=DEV).manual_seed(5)
    row = torch.randn(V, generator=g, device=DEV) * 1.5
    q = torch.randn(V, generator=g, device=DEV)
    count = torch.zeros(V, dtype=torch.long, device=DEV)
    parents = None if drafts else i32([-1, 0, 0, 0])
    for rep in range(4):
        tokens = torch.zeros(B, N, dtype=torch.long, device=DEV)
        if drafts:
            tokens[:, 1] = torch.multinomial(torch.softmax(q / 0.8, 0), B, True, generator=g)
        else:
            tokens[:, 1:] = torch.tensor([3, 9, 3], device=DEV)  # one repeated
        u = torch.rand(B, N, generator=g, device=DEV)
        logits = row.expand(B, N, V)  # strides of zero
        path, kept, token = ops.verify_drafts_raw(
            logits, tokens, u, temperature=0.8, parents=parents,
            draft_logits=q.expand(B, N - 1, V) if drafts else None)
        first = torch.where(kept > 1, tokens.gather(1, path[:, 1:2].long().clamp_min(0))[:, 0],
                            token)
        count += torch.bincount(first, minlength=V)
    p = torch.softmax(row.double() / 0.8, 0)
    n = 4 * B
    z = (count - n * p) / (n * p * (1 - p)).sqrt()
    print(f"[verify distribution] worst z {z.abs().max().item():.2f}", flush=True)
    assert z.abs().max().item() < 5


def test_rows_without_a_distribution():
    announce("verify bad rows")
    V = 600
    logits = torch.zeros(6, 2, V)
    logits[1, 0, 3] = float("nan")
    logits[2, 0, 3] = float("inf")
    logits[3, 0] = float("-inf")
    logits[4, 1, 599] = float("nan")
    logits[5, 0, 1:] = float("-inf")  # certain: token 0
    tokens = torch.tensor([[0, 5]] * 5 + [[0, 0]])
    u = torch.zeros(6, 2)
    path, kept, token = _verify(logits, tokens, u, 1.0)
    assert kept == [2, 1, 1, 1, 2, 2]
    assert token == [0, -1, -1, -1, -1, 0]
    path, kept, token = _verify(logits[[0, 1, 4]], torch.zeros(3, 2, dtype=torch.long), u[:3], 0.0)
    assert kept == [2, 1, 2] and token == [0, -1, -1]


def test_refusals_on_the_device():
    """Counts and parents out of range, and sequences without nodes."""
    announce("verify device refusals")
    B, N, V = 7, 4, 40
    par = [list(p) for p in trees("binary", B, N)]
    logits, tokens, u, _ = verify_inputs(F32, B, N, V, 1, par)
    counts = [4, 5, -1, 0, 4, 4, 2]
    par[4][2] = -1       # a second root
    par[5][0] = 0
    par[6][3] = 99       # unused
    got = _verify(logits, tokens, u, 1.0, par, counts)
    good = [0, 6]
    want = spec_ref.verify(logits[good], tokens[good], u[good], 1.0, [par[0], par[6]], [4, 2])
    for k, b in enumerate(good):
        assert [x[b] for x in got] == [x[k] for x in want]
    for b in (1, 2, 3, 4, 5):
        assert got[0][b] == [-1] * N and got[1][b] == 0 and got[2][b] == -1
    # tokens outside the vocabulary are refused, not read
    tokens[:, 1:] = torch.tensor([V, -1, 1 << 40])
    path, kept, token = _verify(logits, tokens, u, 1.0, par[0:1] * B)
    assert kept == [1] * B and all(0 <= t < V for t in token)


def test_row_strides():
    """Logits of a padded vocabulary, and a batch in another order of strides."""
    announce("verify strides")
    B, N, V = 3, 5, 1003
    par = trees("chain", B, N)
    logits, tokens, u, draft = verify_inputs(BF, B, N, V, 2, par, drafts=True)
    want = _verify(logits, tokens, u, 1.0, drafts=draft)
    wide = torch.full((N, B, V + 21), float("nan"), dtype=BF, device=DEV)
    view = wide.transpose(0, 1)[:, :, 5:5 + V]
    view.copy_(logits)
    wided = torch.full((B, N, V + 2), float("nan"), dtype=BF, device=DEV)
    dview = wided[:, 1:, 1:1 + V]
    dview.copy_(draft)
    path, kept, token = ops.verify_drafts_raw(view, tokens.to(DEV).int(), u.to(DEV),
                                              draft_logits=dview)
    assert (path.tolist(), kept.tolist(), token.tolist()) == want


def test_verify_graph_replays():
    announce("verify graph")
    B, N, V = 4, 7, 5003
    par = trees("random", B, N)
    bufs = [t.to(DEV) for t in verify_inputs(BF, B, N, V, 0, par)[:3]]
    pd = i32(par)

    def step():
        return ops.verify_drafts_raw(*bufs, temperature=0.9, parents=pd)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for rep in range(4):
        for t, x in zip(bufs, verify_inputs(BF, B, N, V, 10 + rep, par)[:3]):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), rep


@pytest.mark.parametrize("dtype,shape,n_caches", [
    (BF, (3, 2, 60, 64), 3), (F32, (2, 4, 40, 128), 70), (FH, (1, 3, 50, 96), 2),
    (BF, (2, 2, 60, 6), 2)], ids=str)
def test_keep_moves_the_path(dtype, shape, n_caches):
    announce(f"keep {dtype} {shape} {n_caches}")
    B, H, S, D = shape
    N = 20
    paths = [[0, 2, 3, 7, 9, 12, 13, 14, 15, 19], [0, 1, 2], [0, 19]][:B]
    kept = [len(p) for p in paths]
    lens = [S - N, 3, 0][:B]
    path = i32([p + [-1] * (N - len(p)) for p in paths])
    kc = [seeded(shape, c, dtype) for c in range(n_caches)]
    vc = [seeded(shape, 100 + c, dtype) for c in range(n_caches)]
    kd, vd = [t.to(DEV) for t in kc], [t.to(DEV) for t in vc]
    ld = [i32(lens) for _ in range(n_caches)]
    ops.cache_keep_raw(kd, vd, ld, path, i32(kept))
    for c in range(n_caches):
        assert torch.equal(kd[c].cpu(), spec_ref.keep(kc[c], lens, paths, kept))
        assert torch.equal(vd[c].cpu(), spec_ref.keep(vc[c], lens, paths, kept))
        assert ld[c].tolist() == [a + b for a, b in zip(lens, kept)]
    # with lens_out the lengths stay
    out = [torch.zeros(B, dtype=torch.int32, device=DEV) for _ in range(n_caches)]
    one = [i32(lens)] * n_caches
    ops.cache_keep_raw(kd, vd, one, path, i32([0] * B), lens_out=out)
    assert one[0].tolist() == lens and out[-1].tolist() == lens


def test_keep_whole_trees_and_bad_paths():
    """Nothing to move on a whole chain; paths that fall, repeat, leave the nodes
    or the cache, and counts out of range, leave the sequence alone."""
    announce("keep bad paths")
    B, H, S, D, N = 9, 2, 30, 64, 6
    kc, vc = seeded((B, H, S, D), 0, BF).to(DEV), seeded((B, H, S, D), 1, BF).to(DEV)
    k0, v0 = kc.clone(), vc.clone()
    path = [[0, 1, 2, 3, 4, 5], [0, 2, 1, -1, -1, -1], [0, 2, 2, -1, -1, -1], [-1, 0, 3, 0, 0, 0],
            [0, 6, 7, 0, 0, 0], [0, 2, 4, 5, 0, 0], [0, 2, 4, 5, 0, 0], [0, 2, 4, 5, 0, 0],
            [0, 2, 4, 5, 0, 0]]
    kept = [6, 3, 3, 3, 3, 7, -1, 4, 4]
    lens = [24, 3, 3, 3, 3, 3, 3, 25, -1]  # row 7: node 5 would be row 30 of 30
    ld = i32(lens)
    ops.cache_keep_raw([kc], [vc], [ld], i32(path), i32(kept))
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    assert ld.tolist() == [30] + lens[1:]


def test_keep_graph_replays():
    announce("keep graph")
    shape, N = (2, 2, 80, 64), 8
    kc = [torch.zeros(shape, dtype=BF, device=DEV) for _ in range(3)]
    vc = [torch.zeros(shape, dtype=BF, device=DEV) for _ in range(3)]
    lens = [torch.zeros(2, dtype=torch.int32, device=DEV) for _ in range(3)]
    path, kept = i32([[0, 2, 5, -1, -1, -1, -1, -1]] * 2), i32([3, 2])

    def step():
        ops.cache_keep_raw(kc, vc, lens, path, kept)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for rep in range(4):
        for c in range(3):
            kc[c].copy_(seeded(shape, 20 + 7 * rep + c, BF))
            vc[c].copy_(seeded(shape, 50 + 7 * rep + c, BF))
            lens[c].fill_(10 * rep)
        want = [spec_ref.keep(t.cpu(), [10 * rep] * 2, path.tolist(), kept.tolist())
                for t in kc + vc]
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip(kc + vc, want):
            assert torch.equal(t.cpu(), w), rep
        assert all(x.tolist() == [10 * rep + 3, 10 * rep + 2] for x in lens)
