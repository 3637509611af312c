"""CPU checks of speculative decoding's entry points: what they refuse before any
launch (the pointers here are never read), and the 64-bit restatement itself."""

from __future__ import annotations

import ctypes
import os

import pytest
import torch

from kempnerforge_amd import _lib, ops
from spec_util import spec_ref, trees, verify_inputs

P = ctypes.c_void_p(1 << 20)  # non-null, never dereferenced


def _library():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return _lib.load()


def _tree(lib, **change):
    a = dict(B=2, N=8, Smax=64, Hq=8, Hkv=2, D=64, max_len=40, stride=0, offset=0, rows=64,
             qn=None, kn=None, dtype=1, ws=P, ws_bytes=1 << 30, q=P, parents=P, counts=P) | change
    return lib.kf_attn_tree(a["q"], P, P, P, P, P, a["parents"], a["stride"], a["counts"], P, P,
                            a["offset"], a["rows"], P, a["ws"], a["ws_bytes"], a["B"], a["N"],
                            a["Smax"], a["Hq"], a["Hkv"], a["D"], a["max_len"], a["qn"], a["kn"],
                            ctypes.c_float(1e-5), a["dtype"], None)


@pytest.mark.parametrize("change,code,word", [
    (dict(B=0), 1, b"positive"), (dict(N=0), 1, b"positive"), (dict(N=257), 1, b"256 nodes"),
    (dict(Hq=7), 1, b"multiple"), (dict(D=63), 1, b"even"), (dict(dtype=3), 1, b"dtype"),
    (dict(max_len=65), 1, b"exceeds"), (dict(rows=0), 1, b"row"), (dict(q=None), 1, b"null"),
    (dict(stride=7), 1, b"parents_stride"), (dict(qn=P), 1, b"both"), (dict(ws=None), 4, b"workspace"),
    (dict(ws_bytes=100), 4, b"workspace"), (dict(B=70000), 1, b"65535"),
    (dict(B=60000, N=256, Hq=256, Hkv=2), 1, b"2^31"),
])
def test_tree_refusals(change, code, word):
    lib = _library()
    assert _tree(lib, **change) == code and word in lib.kf_last_error()


def test_tree_workspace_size():
    lib, n = _library(), _lib.size_out()
    assert lib.kf_attn_tree_workspace_size(4, 16, 32, 8, 128, 4096, 1, ctypes.byref(n)) == 0
    assert n.value >= 4 * 16 * 32 * 128 * 2  # the rotated queries
    assert lib.kf_attn_tree_workspace_size(4, 257, 32, 8, 128, 4096, 1, ctypes.byref(n)) == 1
    assert lib.kf_attn_tree_workspace_size(4, 16, 32, 8, 128, 4096, 1, None) == 1


@pytest.mark.parametrize("change,word", [
    (dict(B=0), b"positive"), (dict(N=257), b"256 nodes"), (dict(V=0), b"positive"),
    (dict(V=(1 << 20) + 1), b"vocabulary"), (dict(dtype=7), b"dtype"), (dict(logits=None), b"null"),
    (dict(T=-1.0), b"temperature"), (dict(T=float("nan")), b"temperature"),
    (dict(T=float("inf")), b"temperature"), (dict(drafts=P), b"chain"),
    (dict(drafts=P, parents=None, T=0.0), b"chain"), (dict(stride=3), b"parents_stride"),
    (dict(ws=None), b"workspace"), (dict(ws_bytes=8), b"workspace"), (dict(B=70000), b"65535"),
])
def test_verify_refusals(change, word):
    lib = _library()
    a = dict(B=2, N=8, V=100, dtype=1, logits=P, T=1.0, drafts=None, parents=P, stride=8,
             ws=P, ws_bytes=1 << 30) | change
    rc = lib.kf_verify_drafts(a["logits"], 800, 100, P, a["parents"], a["stride"], P, a["drafts"],
                              800, 100, P, a["T"], P, P, P, a["ws"], a["ws_bytes"], a["B"],
                              a["N"], a["V"], a["dtype"], None)
    assert rc == (4 if word == b"workspace" else 1) and word in lib.kf_last_error()


@pytest.mark.parametrize("change,word", [
    (dict(n=0), b"n_caches"), (dict(N=300), b"256 nodes"), (dict(k=[4096, None]), b"null"),
    (dict(k=[4096, 4096]), b"share"), (dict(v=[8192, 8192]), b"share"),
    (dict(v=[4096, 16384]), b"one tensor for K and V"), (dict(v=[8192, 4096]), b"share"),
    (dict(out=[256, 512], lens=[256, 256]), b"share"), (dict(path=None), b"null"),
])
def test_keep_refusals(change, word):
    lib = _library()
    a = dict(k=[4096, 12288], v=[8192, 16384], lens=[256, 512], out=[256, 512], n=2, N=8,
             path=P) | change
    arr = ctypes.c_void_p * 2
    rc = lib.kf_kv_cache_keep(arr(*a["k"]), arr(*a["v"]), arr(*a["lens"]), arr(*a["out"]), a["n"],
                              a["path"], P, a["N"], 1, 2, 64, 64, 1, None)
    assert rc == 1 and word in lib.kf_last_error()


def test_cpu_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="GPU"):
        ops.tree_decode_raw(z(1, 2, 4, 64), z(1, 2, 2, 64), z(1, 2, 2, 64), z(1, 2, 8, 64),
                            z(1, 2, 8, 64), z(1, dtype=torch.int32), z(8, 32), z(8, 32),
                            rope_row_offset=0, max_len=8)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.verify_drafts_raw(z(1, 2, 5), z(1, 2, dtype=torch.long), z(1, 2))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.cache_keep_raw([z(1, 2, 8, 64)], [z(1, 2, 8, 64)], [z(1, dtype=torch.int32)],
                           z(1, 2, dtype=torch.int32), z(1, dtype=torch.int32))


def test_ancestors():
    assert spec_ref.ancestors([-1, 0, 0, 2, 1]) == [[0], [0, 1], [0, 2], [0, 2, 3], [0, 1, 4]]


@pytest.mark.parametrize("drafts", [True, False])
def test_the_walk_keeps_the_targets_distribution(drafts):
    """Exactly, not by sampling: over a fine grid of uniforms the first emitted
    token's frequencies are the target's probabilities, to the grid's steps."""
    V, G = 5, 64
    p = torch.tensor([0.4, 0.3, 0.15, 0.1, 0.05]).log()
    q = torch.tensor([0.1, 0.5, 0.1, 0.2, 0.1]).log()
    got = torch.zeros(V, dtype=torch.float64)
    grid = (torch.arange(G) + 0.5) / G
    if drafts:
        par, steps = [[-1, 0]], [(t, w) for t, w in enumerate(q.exp().double().tolist())]
    else:
        par, steps = [[-1, 0]], [(1, 1.0)]
    for tok, weight in steps:
        for a in grid.tolist():
            for b in grid.tolist():
                path, kept, nxt = spec_ref.verify(
                    p.expand(1, 2, V), torch.tensor([[0, tok]]), torch.tensor([[b, a]]), 1.0, par,
                    None, q.expand(1, 1, V) if drafts else None)
                got[tok if kept[0] > 1 else nxt[0]] += weight / G / G
    assert (got - p.exp().double()).abs().max() < 2.0 / G


def test_inputs_exercise_both_answers():
    """The shared inputs accept some drafts and refuse others."""
    par = trees("binary", 16, 15)
    logits, tokens, u, _ = verify_inputs(torch.float32, 16, 15, 500, 0, par)
    kept = spec_ref.verify(logits, tokens, u, 1.0, par)[1]
    assert min(kept) == 1 and max(kept) >= 3


def test_native_checks_of_lists():
    """The pointers of a list of like tensors, and what it refuses."""
    import array

    same = _lib.native().same
    buf = array.array("Q", bytes(8 * 4))
    ts = [torch.zeros(2, 3) for _ in range(3)]
    assert same(ts, buf, 1) == -1
    assert buf.tolist() == [0] + [t.data_ptr() for t in ts]
    for bad in ([ts[0], torch.zeros(3, 2)], [ts[0], torch.zeros(2, 3, dtype=torch.int32)],
                [torch.zeros(3, 2).t()], [ts[0], 5], [], ts + ts):
        with pytest.raises(ValueError):
            same(bad, buf, 0)
    with pytest.raises(TypeError):
        same(tuple(ts), buf, 0)
    with pytest.raises(ValueError):
        same(ts, buf, -2)
