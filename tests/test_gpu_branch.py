"""GPU parity of the attention behind shared prefixes (kf_attn_branch) with the 64-bit
restatement: sizes, lengths, unused tokens, masked places, refusals on the device."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce, seeded
from kempnerforge_amd import ops
from oracle import attention_ref as ref
from oracle import branch_ref
from spec_util import check_rows, check_tree

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
I32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731


def inputs(dtype, G, W, N, Hq, Hkv, D, Pmax, Smax, seed=0):
    B = G * W
    q, k, v = (seeded((B, N, h, D), seed + j, dtype) for j, h in enumerate((Hq, Hkv, Hkv)))
    kp, vp = (seeded((G, Hkv, Pmax, D), seed + 20 + j, dtype) for j in range(2))
    kc, vc = (seeded((B, Hkv, Smax, D), seed + 10 + j, dtype) for j in range(2))
    cos, sin = ref.rope_tables(D, Pmax + Smax, 5e5)
    return q, k, v, kp, vp, kc, vc, cos, sin


def step(q, k, v, kp, vp, kc, vc, cos, sin, plens, lens, max_prefix, max_len, counts=None,
         row_offset=0, **kw):
    kcd, vcd = kc.to(DEV), vc.to(DEV)
    out = ops.branch_decode_raw(q.to(DEV), k.to(DEV), v.to(DEV), kp.to(DEV), vp.to(DEV), I32(plens),
                                kcd, vcd, I32(lens), cos.to(DEV), sin.to(DEV),
                                rope_row_offset=row_offset, max_prefix=max_prefix,
                                max_len=max_len, counts=I32(counts), **kw)
    torch.cuda.synchronize()
    return out, kcd, vcd


def reference(q, k, v, kp, vp, kc, vc, cos, sin, kcd, vcd, plens, lens, counts, more=0.0,
              q_norm=None, k_norm=None):
    """Checks the cache rows of the step and returns what the outputs are over them."""
    W, vw = q.shape[0] // kp.shape[0], vc.clone()
    counts = [q.shape[1]] * q.shape[0] if counts is None else counts
    starts = [plens[b // W] + L for b, L in enumerate(lens)]
    for b, L in enumerate(lens):
        vw[b, :, L:L + counts[b]] = v[b, :counts[b]].transpose(0, 1)
    assert torch.equal(vcd.cpu(), vw)
    k64 = branch_ref.rotated(k, starts, cos, sin, counts, norm=k_norm)
    check_rows(kcd, kc, k64, lens, counts, q.dtype, more)
    q64 = branch_ref.rotated(q, starts, cos, sin, counts, norm=q_norm)
    return branch_ref.branch_attention(q64, kp, vp, plens, kcd.cpu(), vcd.cpu(), lens, counts)


def check(dtype, shape, plens, lens, counts, name):
    announce(name)
    G, W, N, Hq, Hkv, D = shape
    Pmax, Smax = max(plens) + 2, max(lens) + N + 3
    x = inputs(dtype, G, W, N, Hq, Hkv, D, Pmax, Smax)
    out, kcd, vcd = step(*x, plens, lens, max(plens), max(lens) + N, counts)
    want, mag = reference(*x, kcd, vcd, plens, lens, counts)
    check_tree(out, want, mag, dtype, D, max(plens) + max(lens) + N, name)
    if counts is not None:
        for b, n in enumerate(counts):
            assert (out[b, n:] == 0).all()


def spread(n, lo, hi):
    """n lengths from lo to hi, out of order."""
    return [lo + (7 * i + 3) % n * (hi - lo) // max(n - 1, 1) for i in range(n)]


CASES = [
    # dtype, (G, W, N, Hq, Hkv, D), prefix lengths, own lengths, counts
    (BF, (1, 1, 1, 8, 2, 128), [37], [0], None),                # the first token behind a prompt
    (BF, (1, 1, 1, 8, 2, 128), [0], [0], None),                 # one key: its own
    (BF, (1, 4, 1, 32, 8, 128), [100], [11] * 4, None),         # four beams, 16 rows
    (BF, (2, 3, 1, 8, 2, 128), [0, 65], spread(6, 0, 40), None),  # an empty prefix beside another
    (BF, (3, 4, 1, 8, 2, 64), [31, 32, 33], spread(12, 30, 34), None),  # around a chunk of keys
    (BF, (2, 5, 1, 10, 2, 128), [127, 129], spread(10, 62, 66), [1] * 5 + [0, 1, 1, 0, 1]),
    (BF, (1, 8, 1, 12, 12, 64), [250], [5] * 8, None),          # no groups of heads
    (BF, (1, 16, 1, 64, 8, 128), [300], spread(16, 1, 90), None),  # 128 rows of one prefix
    (BF, (1, 70, 1, 16, 2, 128), [200], spread(70, 0, 69), None),  # 560 rows
    (BF, (70, 1, 1, 4, 2, 64), [3 * i for i in range(70)], spread(70, 0, 69), None),
    (BF, (1, 3, 1, 32, 1, 128), [90], [17, 0, 40], None),       # 32 heads a group
    (BF, (1, 2, 4, 8, 2, 128), [100], [30, 0], None),           # 16 own rows
    (BF, (2, 2, 5, 8, 2, 128), [64, 40], [30, 0, 27, 63], [5, 0, 2, 4]),
    (BF, (2, 2, 3, 12, 12, 64), [40, 7], [1, 0, 2, 31], [3, 1, 2, 3]),
    (BF, (1, 3, 40, 8, 2, 128), [77], [0, 50, 9], [40, 13, 1]),  # questions behind a prompt
    (BF, (1, 2, 130, 8, 1, 128), [300], [0, 3], None),
    (BF, (2, 1, 300, 4, 2, 64), [10, 0], [0, 5], [300, 211]),
    (FH, (2, 3, 1, 10, 2, 128), [401, 13], spread(6, 5, 77), None),
    (FH, (1, 12, 1, 8, 2, 128), [210], spread(12, 0, 20), None),
    (FH, (1, 2, 12, 8, 8, 64), [64], [5, 0], [7, 12]),
    (F32, (2, 3, 1, 4, 2, 64), [250, 31], [31] * 6, None),
    (F32, (1, 20, 1, 8, 2, 128), [128], spread(20, 0, 70), None),
    (F32, (1, 2, 29, 10, 2, 128), [210], [64, 0], [29, 5]),
    (F32, (1, 40, 1, 8, 1, 64), [99], [1] * 40, None),          # 320 rows
    (BF, (2, 3, 2, 6, 2, 96), [70, 9], spread(6, 0, 40), [2, 2, 1, 0, 2, 2]),  # other head sizes
    (FH, (1, 3, 1, 4, 4, 80), [90], [1, 2, 3], None),
    (F32, (1, 2, 3, 4, 2, 32), [90], [0, 12], None),
    (BF, (1, 2, 2, 4, 2, 256), [40], [3, 4], None),
    (F32, (1, 2, 2, 4, 2, 6), [40], [3, 4], None),
]


@pytest.mark.parametrize("cfg", CASES, ids=lambda c: "-".join(
    map(str, (str(c[0])[6:], *c[1], "counts" if c[4] else "all"))))
def test_against_64_bits(cfg):
    check(*cfg, f"branch {cfg}")


@pytest.mark.parametrize("dtype,shape,plens,hi", [
    (BF, (1, 3, 1, 32, 8, 128), [4097], 700), (BF, (2, 9, 1, 16, 2, 128), [4097, 300], 40),
    (BF, (1, 2, 33, 32, 8, 128), [3000], 900), (F32, (1, 5, 1, 8, 2, 64), [2049], 500)])
def test_long_prefixes(dtype, shape, plens, hi):
    """Prefixes that many workgroups share."""
    n = shape[0] * shape[1]
    check(dtype, shape, plens, spread(n, hi // 8, hi), None, f"branch long {dtype} {shape}")


@pytest.mark.parametrize("dtype,shape,plens,lens,counts", [
    (BF, (1, 4, 17, 8, 2, 128), [40], [64, 3, 0, 90], None),       # 68 rows of 128, short prefix
    (BF, (1, 4, 17, 8, 2, 128), [1500], [0, 3, 0, 9], [17, 4, 0, 1]),  # and a long one
    (BF, (1, 1, 20, 8, 2, 128), [1200], [130], None),              # one sequence, 80 rows
    (FH, (3, 1, 9, 16, 2, 64), [65, 0, 700], [0, 200, 1], [9, 5, 9]),
    (BF, (2, 6, 12, 8, 2, 128), [130, 64], spread(12, 0, 70), None),   # 48 rows of 128
    (F32, (2, 2, 12, 16, 2, 128), [33, 130], [31, 0, 64, 5], [12, 12, 0, 7]),
    (F32, (1, 3, 24, 8, 2, 64), [900], [0, 4, 31], None),
])
def test_tiles_of_prefix_and_own_rows(dtype, shape, plens, lens, counts):
    """Sequences of 17 rows and more a pair: their own tiles over prefix and cache, or the
    group's over the prefix and theirs over the cache, as the lengths have it."""
    check(dtype, shape, plens, lens, counts, f"branch tiles {dtype} {shape} {plens}")


def test_many_unused_tokens():
    """More rows of a pair than a launch's second dimension has places."""
    announce("branch many tokens")
    N, plens, lens, counts = 140000, [40], [5], [3]
    check(BF, (1, 1, N, 8, 1, 64), plens, lens, counts, "branch many tokens")


def test_a_branch_is_a_decode_step():
    """One sequence behind its own prompt is kf_attn_decode over a cache that holds both:
    the same value rows, keys that differ by the roundings of the eager rotation (each
    product and the sum in bfloat16), and outputs that those explain."""
    announce("branch against decode")
    G, Hq, Hkv, D, plens, lens = 3, 8, 2, 128, [5, 300, 1000], [0, 17, 24]
    x = inputs(BF, G, 1, 1, Hq, Hkv, D, 1000, 32)
    q, k, v, kp, vp, kc, vc, cos, sin = x
    out, kcd, vcd = step(*x, plens, lens, 1000, 30)
    whole = [torch.zeros(G, Hkv, 1100, D, dtype=BF, device=DEV) for _ in range(2)]
    for w, p, c in zip(whole, (kp, vp), (kc, vc)):
        for b in range(G):
            w[b, :, :plens[b]] = p[b, :, :plens[b]].to(DEV)
            w[b, :, plens[b]:plens[b] + lens[b]] = c[b, :, :lens[b]].to(DEV)
    total = [p + n for p, n in zip(plens, lens)]
    dec = ops.decode_raw(q.to(DEV), k.to(DEV), v.to(DEV), *whole, I32(total), cos.to(DEV),
                         sin.to(DEV), rope_row_offset=0, max_len=1025)
    want, mag = reference(*x, kcd, vcd, plens, lens, None)
    check_tree(out, want, mag, BF, D, 1025, "branch")
    check_tree(dec, want, mag, BF, D, 1025, "decode", moved=4 * 2.0 ** -8 * 12)
    for b in range(G):
        new = kcd[b, :, lens[b]].float() - whole[0][b, :, total[b]].float()
        assert new.abs().max().item() <= 4 * 2.0 ** -8 * 8
        assert torch.equal(vcd[b, :, lens[b]], whole[1][b, :, total[b]])


@pytest.mark.parametrize("dtype", [BF, FH, F32])
def test_tokens_at_once_equal_one_at_a_time(dtype):
    announce(f"branch tokens at once {dtype}")
    G, W, N, Hq, Hkv, D, plens, lens = 1, 3, 6, 8, 2, 64, [75], [40, 3, 0]
    x = inputs(dtype, G, W, N, Hq, Hkv, D, 75, 64)
    q, k, v, kp, vp, kc, vc, cos, sin = x
    out, kcd, vcd = step(*x, plens, lens, 75, 60)
    want, mag = reference(*x, kcd, vcd, plens, lens, None)
    check_tree(out, want, mag, dtype, D, 135, "at once")
    k1, v1 = kc, vc
    for i in range(N):
        one = [t[:, i:i + 1] for t in (q, k, v)]
        o, k1, v1 = step(*one, kp, vp, k1, v1, cos, sin, plens, [n + i for n in lens], 75, 60)
        check_tree(o, want[:, i:i + 1], mag[:, i:i + 1], dtype, D, 135, f"step {i}")
    assert torch.equal(kcd, k1) and torch.equal(vcd, v1)


@pytest.mark.parametrize("dtype,N", [(BF, 1), (BF, 40), (FH, 3), (F32, 2)])
def test_qk_norm(dtype, N):
    """Errors of the norm as in the tree's test: below 2^-16 relatively for q and for k."""
    announce(f"branch qk-norm {dtype} {N}")
    G, W, Hq, Hkv, D, plens, lens = 2, 2, 8, 2, 128, [70, 300], [9, 0, 33, 5]
    x = inputs(dtype, G, W, N, Hq, Hkv, D, 300, 80)
    qn, kn = (1 + 0.1 * seeded((D,), 50 + j, torch.float32) for j in range(2))
    out, kcd, vcd = step(*x, plens, lens, 300, 80, q_norm_weight=qn.to(DEV),
                         k_norm_weight=kn.to(DEV), norm_eps=1e-5)
    want, mag = reference(*x, kcd, vcd, plens, lens, None, more=2.0 ** -16, q_norm=qn, k_norm=kn)
    dot = 1.4 * 1.4 * D ** 0.5
    check_tree(out, want, mag, dtype, D, 380, "qk-norm", dot=dot, moved=2.0 ** -16 * dot)


def test_tables_that_start_at_the_new_tokens():
    """A model hands over its tables from position seq_len on (row offset)."""
    announce("branch row offset")
    x = inputs(BF, 2, 2, 4, 8, 2, 64, 50, 40)
    q, k, v, kp, vp, kc, vc, cos, sin = x
    a = step(*x, [50, 50], [20] * 4, 50, 30)
    b = step(*x[:7], cos[70:74], sin[70:74], [50, 50], [20] * 4, 50, 30, row_offset=70)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("dtype,N,W,D", [(BF, 1, 3, 128), (BF, 4, 2, 128), (FH, 6, 3, 64),
                                         (BF, 40, 2, 128), (F32, 5, 3, 64), (BF, 4, 2, 96)])
def test_what_a_token_does_not_see_does_not_reach_it(dtype, N, W, D):
    """Stale rows of the prefix and the caches, unused tokens, later tokens and the other
    sequences hold NaN and Inf."""
    masked(dtype, N, W, D, 70)


@pytest.mark.parametrize("dtype,N,W,D", [(BF, 12, 8, 128), (FH, 12, 8, 64), (F32, 20, 5, 64)])
@pytest.mark.parametrize("bound", [70, 2000])
def test_masked_rows_of_both_kinds_of_tiles(dtype, N, W, D, bound):
    """The same where sequences have tiles of their own: with a short bound on the prefix
    they walk it themselves, with a long one the group does."""
    masked(dtype, N, W, D, bound)


def masked(dtype, N, W, D, bound):
    announce(f"branch masked NaN {dtype} {N} {W} {D} {bound}")
    G, Hq, Hkv = 2, 4, 2
    B, plens, Pmax, Smax = G * W, [45, 64], bound + 30, 40 + N + 30
    lens = [(11 * b) % 37 for b in range(B)]
    counts = [N] * B
    counts[-1] = N // 2
    x = inputs(dtype, G, W, N, Hq, Hkv, D, Pmax, Smax)
    q, k, v, kp, vp, kc, vc, cos, sin = x
    for g, P in enumerate(plens):
        kp[g, :, P:], vp[g, :, P:] = float("nan"), float("inf")
    for b, L in enumerate(lens):
        kc[b, :, L:], vc[b, :, L:] = float("nan"), float("inf")
    # sequence 0's last token, sequence 1's own row 0 (if it has one), unused tokens
    v[0, N - 1, 1, :] = float("-inf")
    v[0, N - 1, 0, 3] = float("nan")
    k[-1, counts[-1]:], v[-1, counts[-1]:], q[-1, counts[-1]:] = (float("nan"),) * 3
    vc[1, :, 0] = float("inf")
    out, kcd, vcd = step(*x, plens, lens, bound, 37 + N, counts)
    clean = [t.clone() for t in x]
    for t in clean:
        t[~torch.isfinite(t)] = 1.0
    o2, k2, v2 = step(*clean, plens, lens, bound, 37 + N, counts)
    want, mag = reference(*clean, k2, v2, plens, lens, counts)
    got = out.cpu().double()
    for b in range(B):
        for i in range(counts[b]):
            if b == 1:
                assert not torch.isfinite(got[b, i]).any(), i
            elif b == 0 and i == N - 1:
                assert not torch.isfinite(got[b, i, Hq // 2:]).any()
                assert torch.isnan(got[b, i, :Hq // 2, 3]).all()
            else:
                check_tree(out[b, i], want[b, i], mag[b, i], dtype, D, 37 + N + 70,
                           f"token {b} {i}")
    assert (got[-1, counts[-1]:] == 0).all()
    for b, L in enumerate(lens):
        assert torch.isnan(kcd[b, :, L + counts[b]:]).all()
        assert torch.isinf(vcd[b, :, L + counts[b]:]).all()


@pytest.mark.parametrize("N,W,D", [(1, 2, 128), (6, 2, 128), (1, 40, 128), (6, 2, 96)])
def test_refusals_on_the_device(N, W, D):
    """A sequence whose prefix, length, count or tables are out of range gets NaN and no
    cache write; the others are served, those of its group too."""
    refused(N, W, D, 60)


@pytest.mark.parametrize("bound", [60, 2000])
def test_refusals_in_both_kinds_of_tiles(bound):
    refused(12, 8, 128, bound)


def refused(N, W, D, bound):
    announce(f"branch device refusals {N} {W} {D} {bound}")
    G, P, L = 4, 50, 20
    B = G * W
    x = inputs(BF, G, W, N, 4, 2, D, bound, 40)
    q, k, v, kp, vp, kc, vc, cos, sin = x
    plens, lens, counts = [P] * G, [L] * B, [N] * B
    plens[3] = bound + 1                # beyond max_prefix: the whole group
    lens[0], lens[W] = 41 - N, -1       # beyond max_len; negative
    counts[W + 1], counts[2 * W] = N + 1, -1
    bad = {0, W, W + 1, 2 * W, *range(3 * W, 4 * W)}
    out, kcd, vcd = step(*x, plens, lens, bound, 40, counts)
    good = [b for b in range(B) if b not in bad]
    for b in bad:
        assert torch.isnan(out[b].float()).all(), b
        assert torch.equal(kcd[b].cpu(), kc[b]) and torch.equal(vcd[b].cpu(), vc[b])
    ref_counts = [0 if b in bad else n for b, n in enumerate(counts)]
    ref_lens = [0 if b in bad else n for b, n in enumerate(lens)]
    want, mag = reference(*x, kcd, vcd, [P] * G, ref_lens, ref_counts)
    check_tree(out[good], want[good], mag[good], BF, D, 110, "served")
    # tables that end before the last token of the longer sequences
    lens = [L + b % 2 for b in range(B)]
    rows = P + L + N
    out, kcd, _ = step(*x[:7], cos[:rows], sin[:rows], [P] * G, lens, bound, 40)
    for b in range(B):
        assert torch.isnan(out[b].float()).all() == (b % 2 == 1), b
        assert b % 2 == 0 or torch.equal(kcd[b].cpu(), kc[b])


@pytest.mark.parametrize("N,W", [(1, 3), (7, 2), (1, 24)])
def test_strided_and_misaligned_inputs(N, W):
    announce(f"branch strides {N} {W}")
    G, Hq, Hkv, D = 2, 8, 2, 64
    B, plens, lens = G * W, [33, 90], spread(G * W, 0, 30)
    x = inputs(BF, G, W, N, Hq, Hkv, D, 90, 40)
    q, k, v, kp, vp, kc, vc, cos, sin = x
    a = step(*x, plens, lens, 90, 38)
    # one fused projection's slices
    fused = torch.cat([q.flatten(2), k.flatten(2), v.flatten(2)], -1).to(DEV)
    qs, ks, vs = (t.view(B, N, -1, D) for t in fused.split([Hq * D, Hkv * D, Hkv * D], dim=-1))
    b = step(qs, ks, vs, *x[3:], plens, lens, 90, 38)
    assert all(torch.equal(s, t) for s, t in zip(a, b))

    def off(t):  # one element behind an aligned address
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        o = buf[1:].view(t.shape)
        o.copy_(t)
        return o

    kcd, vcd = off(kc), off(vc)
    out = ops.branch_decode_raw(off(q), off(k), off(v), off(kp), off(vp), I32(plens), kcd, vcd,
                                I32(lens), cos.to(DEV), sin.to(DEV), rope_row_offset=0,
                                max_prefix=90, max_len=38)
    assert torch.equal(kcd.cpu(), a[1].cpu()) and torch.equal(vcd.cpu(), a[2].cpu())
    want, mag = reference(*x, kcd, vcd, plens, lens, None)
    check_tree(out, want, mag, BF, D, 130, "misaligned")


@pytest.mark.parametrize("N,W", [(1, 4), (1, 30), (12, 3)])
def test_graph_replays_and_streams(N, W):
    """Captured on one stream and replayed, eager calls between: every replay equals the
    eager call on the same inputs."""
    announce(f"branch graph {N} {W}")
    G, Hq, Hkv, D = 2, 8, 2, 128
    B = G * W
    q, k, v, kp, vp, kc, vc, cos, sin = (t.to(DEV) for t in inputs(BF, G, W, N, Hq, Hkv, D, 900, 64))
    plens, lens, counts = I32([5, 700]), I32(spread(B, 0, 50)), I32([N] * B)

    def call():
        return ops.branch_decode_raw(q, k, v, kp, vp, plens, kc, vc, lens, cos, sin,
                                     rope_row_offset=0, max_prefix=900, max_len=64, counts=counts)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(), call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for rep in range(4):
        for t, s in ((q, 0), (k, 1), (v, 2)):
            t.copy_(seeded(t.shape, 100 + 10 * rep + s, BF))
        plens.copy_(torch.tensor([900 - 300 * rep, 17 * rep], dtype=torch.int32))
        lens.copy_(torch.tensor(spread(B, rep, 50 - rep), dtype=torch.int32))
        counts.copy_(torch.tensor([max(N - (b + rep) % 3, 0) for b in range(B)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got, kg = out.clone(), kc.clone()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(kg, kc), rep


@pytest.mark.parametrize("N,W", [(1, 2), (1, 20), (24, 2)])
def test_caches_past_32_bit_offsets(N, W):
    """Rows that begin more than 2^32 bytes into the prefixes and the caches."""
    announce(f"branch long caches {N} {W}")
    G, Hq, Hkv, D = 2, 8, 8, 128
    big, Pw, Sw = 1 << 20, 150, 80
    kp, vp = (torch.zeros(G, Hkv, 1 << 21, D, dtype=BF, device=DEV) for _ in range(2))  # 8.6 GB
    kc, vc = (torch.zeros(G * W, Hkv, big // W, D, dtype=BF, device=DEV) for _ in range(2))
    x = inputs(BF, G, W, N, Hq, Hkv, D, Pw, Sw)
    for t, s in zip((kp, vp, kc, vc), x[3:7]):
        t[:, :, :s.shape[2]] = s.to(DEV)
    plens, lens = [100, 150], spread(G * W, 0, 50)
    q, k, v = (t.to(DEV) for t in x[:3])
    out = ops.branch_decode_raw(q, k, v, kp, vp, I32(plens), kc, vc, I32(lens), x[7].to(DEV),
                                x[8].to(DEV), rope_row_offset=0, max_prefix=Pw, max_len=Sw)
    want, mag = reference(*x, kc[:, :, :Sw], vc[:, :, :Sw], plens, lens, None)
    check_tree(out, want, mag, BF, D, Pw + Sw, "long caches")


SIXTEEN = [
    # (G, W, N, Hq, Hkv, D), prefix lengths, own lengths, counts: without groups of heads, 16 new
    # tokens are all the rows that a wavefront takes, and (float32) all the keys of a chunk
    ((1, 1, 16, 12, 12, 64), [40], [0], None),
    ((1, 1, 16, 4, 4, 128), [0], [21], None),
    ((2, 1, 16, 2, 2, 64), [7, 33], [16, 5], [16, 16]),
    ((1, 3, 16, 4, 4, 64), [50], [17, 0, 3], None),             # beside tiles over the prefix
    ((2, 2, 16, 4, 4, 128), [31, 64], [0, 9, 16, 40], [16, 3, 16, 0]),
    ((1, 6, 16, 16, 16, 64), [100], spread(6, 0, 40), [16] * 6),  # 96 rows of one prefix
    ((1, 5, 16, 2, 2, 128), [90], spread(5, 0, 70), [16, 15, 16, 1, 16]),
    ((70, 1, 16, 1, 1, 64), [i % 9 for i in range(70)], spread(70, 0, 40), None),
]


@pytest.mark.parametrize("dtype", [F32, BF, FH])
@pytest.mark.parametrize("cfg", SIXTEEN, ids=lambda c: "-".join(
    map(str, (*c[0], "counts" if c[3] else "all"))))
def test_as_many_new_tokens_as_a_chunk_has_keys(dtype, cfg):
    shape, plens, lens, counts = cfg
    check(dtype, shape, plens, lens, counts, f"branch sixteen {dtype} {cfg}")


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("W,D", [(1, 64), (1, 128), (3, 64), (5, 128)])
def test_a_later_one_of_sixteen_tokens_holds_nan(dtype, W, D):
    """Token 11's key and value and token 15's value are not finite: tokens before 11 do not
    see them, those from 11 on give NaN."""
    announce(f"branch sixteen NaN {dtype} {W} {D}")
    G, N, H, plens = 2, 16, 2, [45, 0]
    lens = [(11 * b) % 37 for b in range(G * W)]
    x = inputs(dtype, G, W, N, H, H, D, 45, 60)
    clean = [t.clone() for t in x]
    k, v = x[1], x[2]
    k[:, 11], v[:, 11], v[:, 15] = float("nan"), float("inf"), float("-inf")
    out, _, _ = step(*x, plens, lens, 45, 60)
    _, kcd, vcd = step(*clean, plens, lens, 45, 60)
    want, mag = reference(*clean, kcd, vcd, plens, lens, None)
    check_tree(out[:, :11], want[:, :11], mag[:, :11], dtype, D, 105, "before the eleventh")
    assert torch.isnan(out[:, 11:]).all()
