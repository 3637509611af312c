"""GPU parity of the attention of drafted trees (kf_attn_tree) with the 64-bit
restatement: sizes, trees, unused nodes, masked places, refusals on the device."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce, seeded
from kempnerforge_amd import ops
from oracle import attention_ref as ref
from spec_util import check_rows, check_tree, spec_ref, tree_inputs, trees

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _step(q, k, v, kc, vc, lens, cos, sin, max_len, parents=None, counts=None, row_offset=0, **kw):
    kcd, vcd = kc.to(DEV), vc.to(DEV)
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = ops.tree_decode_raw(q.to(DEV), k.to(DEV), v.to(DEV), kcd, vcd, i32(lens), cos.to(DEV),
                              sin.to(DEV), rope_row_offset=row_offset, max_len=max_len,
                              parents=i32(parents), counts=i32(counts), **kw)
    torch.cuda.synchronize()
    return out, kcd, vcd


def _reference(q, k, v, kc, vc, kcd, vcd, lens, cos, sin, par, counts=None, more=0.0, **norms):
    """Checks the cache rows of the step and returns what the outputs are over them."""
    vw = vc.clone()
    for b, L in enumerate(lens):
        n = q.shape[1] if counts is None else counts[b]
        vw[b, :, L:L + n] = v[b, :n].transpose(0, 1)
    assert torch.equal(vcd.cpu(), vw)
    k64 = spec_ref.rotated(k, lens, cos, sin, par, counts, norm=norms.get("k_norm"))
    check_rows(kcd, kc, k64, lens, counts, q.dtype, more)
    q64 = spec_ref.rotated(q, lens, cos, sin, par, counts, norm=norms.get("q_norm"))
    return spec_ref.tree_attention(q64, kcd.cpu(), vcd.cpu(), lens, par, counts)


def _check(cfg, name):
    dtype, (B, N, Hq, Hkv, D), lens, tree, counts = cfg
    announce(name)
    Smax = max(lens) + N + 3
    q, k, v, kc, vc, cos, sin = tree_inputs(dtype, B, N, Hq, Hkv, D, Smax)
    par = trees(tree, B, N)
    out, kcd, vcd = _step(q, k, v, kc, vc, lens, cos, sin, max(lens) + N,
                          None if tree == "chain" else par, counts)
    want, mag = _reference(q, k, v, kc, vc, kcd, vcd, lens, cos, sin, par, counts)
    check_tree(out, want, mag, dtype, D, max(lens) + N, name)
    if counts is not None:
        for b, n in enumerate(counts):
            assert (out[b, n:] == 0).all()


CASES = [
    # dtype, (B, N, Hq, Hkv, D), prefix lengths, tree, counts
    (BF, (1, 1, 8, 2, 128), [37], "chain", None),            # one token
    (BF, (1, 1, 8, 2, 128), [0], "chain", None),             # an empty cache
    (BF, (2, 5, 8, 2, 128), [0, 1], "chain", None),
    (BF, (3, 5, 32, 8, 128), [31, 32, 33], "binary", None),  # around a block of 32 keys
    (BF, (3, 7, 8, 2, 64), [63, 64, 65], "random", None),
    (BF, (3, 9, 8, 2, 128), [127, 128, 129], "star", [9, 0, 4]),
    (BF, (2, 16, 12, 12, 64), [100, 250], "random", None),   # no groups
    (BF, (2, 16, 10, 2, 128), [255, 700], "random", [16, 1]),  # five heads a group
    (BF, (2, 33, 16, 2, 128), [500, 90], "binary", [33, 20]),
    (BF, (1, 64, 64, 8, 128), [300], "random", None),        # 512 rows a KV head
    (BF, (2, 64, 8, 1, 128), [77, 1000], "forest", None),
    (BF, (1, 100, 8, 2, 128), [45], "random", None),         # masks of four words
    (BF, (2, 200, 8, 2, 128), [0, 333], "chain", [200, 131]),
    (BF, (1, 256, 4, 2, 64), [129], "random", None),         # the most nodes
    (BF, (40, 4, 8, 2, 64), [9 * i for i in range(40)], "random", None),
    (BF, (70, 3, 4, 2, 64), [5 * i for i in range(70)], "chain", None),
    (FH, (2, 27, 10, 2, 128), [401, 13], "random", None),
    (FH, (2, 12, 8, 8, 64), [64, 5], "binary", [7, 12]),
    (F32, (2, 9, 4, 2, 64), [250, 31], "binary", None),
    (F32, (2, 20, 8, 2, 128), [128, 300], "random", [20, 3]),
    (F32, (1, 70, 8, 1, 128), [65], "random", None),
    (F32, (2, 29, 10, 2, 128), [210, 64], "binary", [29, 5]),  # 145 rows: three tiles of 64
    (F32, (2, 33, 8, 2, 64), [99, 1], "random", None),         # 132 rows
    (F32, (1, 100, 8, 2, 128), [33], "random", None),          # 400 rows: tiles of 128
    (BF, (2, 6, 32, 1, 128), [70, 9], "binary", None),       # 32 heads a group
    (BF, (2, 6, 6, 2, 96), [70, 9], "binary", None),         # other head sizes
    (FH, (1, 11, 4, 4, 80), [90], "random", None),
    (F32, (1, 11, 4, 2, 32), [90], "random", None),
    (BF, (1, 5, 4, 2, 256), [40], "star", None),
    (F32, (1, 5, 4, 2, 6), [40], "star", None),
]


@pytest.mark.parametrize("cfg", CASES, ids=lambda c: "-".join(
    map(str, (str(c[0])[6:], *c[1], c[3], "counts" if c[4] else "all"))))
def test_against_64_bits(cfg):
    _check(cfg, f"tree {cfg}")


@pytest.mark.parametrize("dtype,shape", [(BF, (2, 24, 32, 8, 128)), (F32, (1, 24, 8, 2, 64))])
def test_long_prefixes(dtype, shape):
    """Prefixes that many workgroups share."""
    _check((dtype, shape, [4097, 3000][:shape[0]], "random", None), f"tree long {dtype} {shape}")


def test_one_node_is_a_decode_step():
    """A single node is kf_attn_decode's token: the same values, keys that differ
    by the roundings of the reference's eager rotation (each product and the sum
    in bfloat16, half a step of 2^-8 each on magnitudes below 8), and outputs that
    keys and queries so far apart explain."""
    announce("tree of one node against decode")
    B, Hq, Hkv, D, lens = 3, 8, 2, 128, [5, 300, 1024]
    q, k, v, kc, vc, cos, sin = tree_inputs(BF, B, 1, Hq, Hkv, D, 1100)
    out, kcd, vcd = _step(q, k, v, kc, vc, lens, cos, sin, 1025)
    kd, vd = kc.to(DEV), vc.to(DEV)
    dec = ops.decode_raw(q.to(DEV), k.to(DEV), v.to(DEV), kd, vd,
                         torch.tensor(lens, dtype=torch.int32, device=DEV), cos.to(DEV),
                         sin.to(DEV), rope_row_offset=0, max_len=1025)
    assert torch.equal(vcd, vd)
    assert (kcd.float() - kd.float()).abs().max().item() <= 4 * 2.0 ** -8 * 8
    want, mag = _reference(q, k, v, kc, vc, kcd, vcd, lens, cos, sin, [[-1]] * B)
    check_tree(out, want, mag, BF, D, 1025, "one node")
    check_tree(dec, want, mag, BF, D, 1025, "decode", moved=4 * 2.0 ** -8 * 12)


def test_chain_equals_successive_steps_of_one_node():
    """The same rows and, over them, the same outputs to rounding as one node a
    call; in float32 the eager rotation differs by steps of 2^-24 only."""
    announce("chain against single steps")
    B, N, Hq, Hkv, D, lens = 2, 6, 8, 2, 64, [40, 3]
    for dtype in (BF, F32):
        q, k, v, kc, vc, cos, sin = tree_inputs(dtype, B, N, Hq, Hkv, D, 64)
        out, kcd, vcd = _step(q, k, v, kc, vc, lens, cos, sin, 60)
        want, mag = _reference(q, k, v, kc, vc, kcd, vcd, lens, cos, sin, trees("chain", B, N))
        k1, v1 = kc, vc
        for i in range(N):
            one = [t[:, i:i + 1] for t in (q, k, v)]
            o, k1, v1 = _step(*one, k1, v1, [n + i for n in lens], cos, sin, 60)
            check_tree(o, want[:, i:i + 1], mag[:, i:i + 1], dtype, D, 60, f"step {i}")
        assert torch.equal(kcd, k1) and torch.equal(vcd, v1)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_qk_norm(dtype):
    """The norm adds at most D steps of 2^-24 to the sum of squares, a hardware
    reciprocal root (2^-22) and two products: below 2^-16 relatively for q and for
    k; the normalised rows have |q| |k| D^-1/2 = D^1/2 times the weights' 1.4 each at
    most."""
    announce(f"tree qk-norm {dtype}")
    B, N, Hq, Hkv, D, lens = 2, 9, 8, 2, 128, [70, 300]
    q, k, v, kc, vc, cos, sin = tree_inputs(dtype, B, N, Hq, Hkv, D, 320)
    qn, kn = (1 + 0.1 * seeded((D,), 50 + j, torch.float32) for j in range(2))
    par = trees("random", B, N)
    out, kcd, vcd = _step(q, k, v, kc, vc, lens, cos, sin, 310, par, q_norm_weight=qn.to(DEV),
                          k_norm_weight=kn.to(DEV), norm_eps=1e-5)
    want, mag = _reference(q, k, v, kc, vc, kcd, vcd, lens, cos, sin, par, more=2.0 ** -16,
                           q_norm=qn, k_norm=kn)
    dot = 1.4 * 1.4 * D ** 0.5
    check_tree(out, want, mag, dtype, D, 310, "qk-norm", dot=dot, moved=2.0 ** -16 * dot)


def test_tables_that_start_at_the_prefix():
    """A model hands over its tables from position seq_len on (row offset)."""
    announce("tree row offset")
    B, N, L = 2, 6, 50
    q, k, v, kc, vc, cos, sin = tree_inputs(BF, B, N, 8, 2, 64, 80)
    par = trees("binary", B, N)
    a = _step(q, k, v, kc, vc, [L, L], cos, sin, 60, par)
    b = _step(q, k, v, kc, vc, [L, L], cos[L:L + N], sin[L:L + N], 60, par, row_offset=L)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64), (BF, 96)])
def test_what_a_node_does_not_see_does_not_reach_it(dtype, D):
    """Stale cache rows and a sibling branch hold NaN and Inf."""
    announce(f"tree masked NaN {dtype} {D}")
    B, N, Hq, Hkv, lens, counts = 2, 12, 4, 2, [45, 0], [12, 7]
    q, k, v, kc, vc, cos, sin = tree_inputs(dtype, B, N, Hq, Hkv, D, 70)
    par = [[-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 7]] * B
    for b, L in enumerate(lens):
        kc[b, :, L:], vc[b, :, L:] = float("nan"), float("inf")
    # node 2 and its descendants (5, 6, 9, 10), and the unused nodes of row 1
    k[:, 2], v[:, 2] = float("inf"), float("nan")
    v[:, 5, :, 3] = float("inf")
    v[0, 11, 1, :] = float("-inf")  # the last row of the cache in use, seen by itself alone
    k[1, 7:], v[1, 7:], q[1, 7:] = (float("nan"),) * 3
    out, kcd, vcd = _step(q, k, v, kc, vc, lens, cos, sin, 60, par, counts)
    clean = [t.clone() for t in (q, k, v, kc, vc)]
    for t in clean:
        t[~torch.isfinite(t)] = 1.0
    # the clean run's rows: what the others' outputs are made of
    o2, k2, v2 = _step(*clean, lens, cos, sin, 60, par, counts)
    want, mag = _reference(*clean, k2, v2, lens, cos, sin, par, counts)
    got = out.cpu().double()
    for b in range(B):
        for i in range(counts[b]):
            seen = spec_ref.ancestors(par[b])[i]
            hit = 2 in seen or 5 in seen
            rows = slice(None) if not (b == 0 and i == 11) else slice(0, 2)
            if hit:
                assert not torch.isfinite(got[b, i]).all(), (b, i)
            else:
                check_tree(out[b, i, rows], want[b, i, rows], mag[b, i, rows], dtype, D, 60,
                           f"node {b} {i}")
    assert not torch.isfinite(got[0, 11, 2:]).any()
    assert (got[1, 7:] == 0).all()
    # rows behind the last node are as they were
    for b, L in enumerate(lens):
        assert torch.isnan(kcd[b, :, L + counts[b]:]).all()
        assert torch.isinf(vcd[b, :, L + counts[b]:]).all()


@pytest.mark.parametrize("D", [128, 96])
def test_refusals_on_the_device(D):
    """A sequence whose length, count, parents or tables are out of range gets NaN
    and no cache write; the others are served."""
    announce(f"tree device refusals D={D}")
    B, N, L = 8, 6, 20
    q, k, v, kc, vc, cos, sin = tree_inputs(BF, B, N, 4, 2, D, 40)
    par = [list(p) for p in trees("binary", B, N)]
    lens, counts = [L] * B, [N] * B
    lens[1] = 36          # 36 + 6 beyond max_len
    lens[2] = -1
    counts[3] = N + 1
    counts[4] = -1
    par[5][3] = 3         # its own parent
    par[6][2] = -2
    par[7] = [-1, 0, 1, 9, 3, 3]
    counts[7] = 3         # an unused node's parent does not matter
    out, kcd, vcd = _step(q, k, v, kc, vc, lens, cos, sin, 40, par, counts)
    for b in range(B):
        if b in (0, 7):
            assert torch.isfinite(out[b].float()).all()
        else:
            assert torch.isnan(out[b].float()).all(), b
            assert torch.equal(kcd[b].cpu(), kc[b]) and torch.equal(vcd[b].cpu(), vc[b])
    # tables that end before the deepest node
    out, kcd, _ = _step(q, k, v, kc, vc, [L] * B, cos[:L + 2], sin[:L + 2], 40, par, [3] * 6 + [1, 3])
    deep = [max(len(x) for x in spec_ref.ancestors(par[b][:3])) if b < 6 else 1 for b in range(B)]
    for b in (0, 1, 2, 3, 4, 5, 6):
        assert torch.isnan(out[b].float()).any() == (deep[b] > 2), b
    assert torch.isnan(out[7].float()).all() and torch.equal(kcd[7].cpu(), kc[7])


def test_strided_and_misaligned_inputs():
    """Projections' views with other strides, and tensors off 16-byte boundaries,
    give what contiguous aligned ones give."""
    announce("tree strides")
    B, N, Hq, Hkv, D, lens = 2, 7, 8, 2, 64, [33, 90]
    q, k, v, kc, vc, cos, sin = tree_inputs(BF, B, N, Hq, Hkv, D, 110)
    par = trees("binary", B, N)
    a = _step(q, k, v, kc, vc, lens, cos, sin, 100, par)
    # one fused projection's slices
    fused = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1).to(DEV)
    qs, ks, vs = (x.view(B, N, -1, D) for x in
                  fused.split([Hq * D, Hkv * D, Hkv * D], dim=-1))
    b = _step(qs, ks, vs, kc, vc, lens, cos, sin, 100, par)
    assert all(torch.equal(x, y) for x, y in zip(a, b))

    def off(t):  # one element behind an aligned address
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        o = buf[1:].view(t.shape)
        o.copy_(t)
        return o

    kcd, vcd = off(kc), off(vc)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = ops.tree_decode_raw(off(q), off(k), off(v), kcd, vcd, i32(lens), cos.to(DEV),
                              sin.to(DEV), rope_row_offset=0, max_len=100, parents=i32(par))
    assert torch.equal(kcd.cpu(), a[1].cpu()) and torch.equal(vcd.cpu(), a[2].cpu())
    want, mag = _reference(q, k, v, kc, vc, kcd, vcd, lens, cos, sin, par)
    check_tree(out, want, mag, BF, D, 100, "misaligned")


def test_graph_replays_and_streams():
    """Captured on one stream and replayed, eager calls of other sizes between:
    every replay equals the eager call on the same inputs."""
    announce("tree graph")
    B, N, Hq, Hkv, D, Smax = 3, 12, 8, 2, 128, 900
    q, k, v, kc, vc, cos, sin = (t.to(DEV) for t in tree_inputs(BF, B, N, Hq, Hkv, D, Smax))
    lens = torch.tensor([5, 700, 333], dtype=torch.int32, device=DEV)
    counts = torch.tensor([12, 3, 9], dtype=torch.int32, device=DEV)
    par = torch.tensor(trees("random", B, N), dtype=torch.int32, device=DEV)

    def step():
        return ops.tree_decode_raw(q, k, v, kc, vc, lens, cos, sin, rope_row_offset=0,
                                   max_len=Smax, parents=par, counts=counts)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(4):
        for t, s in ((q, 0), (k, 1), (v, 2)):
            t.copy_(seeded(t.shape, 100 + 10 * rep + s, BF))
        lens.copy_(torch.tensor([rep, 700 - 90 * rep, 800], dtype=torch.int32))
        counts.copy_(torch.tensor([12 - rep, rep, 12], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got, kg = out.clone(), kc.clone()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(kg, kc), rep


def test_a_cache_past_32_bit_offsets():
    """Rows that begin more than 2^32 bytes into the cache (batch row 1 of 2)."""
    announce("tree long cache")
    B, N, Hq, Hkv, D, Smax = 2, 4, 8, 8, 128, 1 << 21
    kc = torch.zeros(B, Hkv, Smax, D, dtype=BF, device=DEV)  # 8.6 GB
    vc = torch.zeros_like(kc)
    q, k, v = (seeded((B, N, h, D), j, BF) for j, h in enumerate((Hq, Hkv, Hkv)))
    lens, W = [100, 60], 200
    kp, vp = (seeded((B, Hkv, W, D), 10 + j, BF) for j in range(2))
    kc[:, :, :W], vc[:, :, :W] = kp.to(DEV), vp.to(DEV)
    cos, sin = ref.rope_tables(D, W, 5e5)
    out = ops.tree_decode_raw(q.to(DEV), k.to(DEV), v.to(DEV), kc, vc,
                              torch.tensor(lens, dtype=torch.int32, device=DEV), cos.to(DEV),
                              sin.to(DEV), rope_row_offset=0, max_len=W)
    want, mag = _reference(q, k, v, kp, vp, kc[:, :, :W], vc[:, :, :W], lens, cos, sin,
                           trees("chain", B, N))
    check_tree(out, want, mag, BF, D, W, "long cache")
