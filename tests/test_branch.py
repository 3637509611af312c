"""Several continuations of one prompt without a GPU: the branch caches' bookkeeping, beam
search with the oracle in place of the kernels against all continuations, and the
refusals of the entry points."""

from __future__ import annotations

import ctypes
import itertools
import os

import pytest
import torch

from kempnerforge_amd import Attention, BranchKVCache, KVCache, _lib, ops, reorder_branches
from kempnerforge_amd.generate import beam_generate, generate
from oracle import branch_ref
from test_spec_refusals import BIG, _meta
from test_speculative import Bigram, no_device  # noqa: F401

z = torch.zeros
INF = float("inf")


def _prefix(B=2, T=16, fill=5):
    c = KVCache(B, T, 2, 8, torch.float32, torch.device("cpu"))
    c.seq_len = fill
    return c


# ------------------------------------------------------------------ caches
def test_levels_count_the_prompt():
    p = _prefix()
    c = p.branch(3, 7)
    assert isinstance(c, BranchKVCache) and c.k.shape == (6, 2, 7, 8) and c.prefix is p
    assert c.seq_len == 5 and c.max_seq_len == 12 and c.lens.tolist() == [0] * 6
    c._advance(4)
    assert c.seq_len == 9 and c.lens.tolist() == [4] * 6
    c._check_room(3)
    with pytest.raises(ValueError, match="overflow"):
        c._check_room(4)
    c.seq_len = 6
    assert c.lens.tolist() == [1] * 6 and c._seq_len == 1
    for bad in (4, 13):
        with pytest.raises(ValueError):
            c.seq_len = bad
    c.set_lengths([0, 7, 1, 1, 1, 1])
    assert c.ragged and c.seq_len == 12
    with pytest.raises(ValueError):
        c.set_lengths([8] * 6)
    with pytest.raises(ValueError):
        c.update(z(6, 2, 1, 8), z(6, 2, 1, 8))


def test_a_prompt_that_goes_on_is_not_seen():
    p = _prefix()
    c = p.branch(2, 4)
    p._advance(1)
    assert c.seq_len == 5 and c.prefix_lens.tolist() == [5, 5] and p.lens.tolist() == [6, 6]


def test_tables():
    p = _prefix()
    cos, sin = z(1, 4), torch.ones(1, 4)
    c = p.branch(2, 4)
    c._advance(2)
    assert c._decode_tables(cos, sin) == (cos, sin, 7)  # the caller's begin at seq_len
    p.set_lengths([3, 5])
    c = p.branch(2, 4)
    with pytest.raises(ValueError, match="RoPE tables"):
        c._decode_tables(cos, sin)
    full = z(16, 4), z(16, 4)
    p.use_rope_tables(*full)
    assert p.branch(2, 4)._decode_tables(cos, sin) == (*full, 0)
    c.use_rope_tables(*full)
    assert c._decode_tables(cos, sin) == (*full, 0)


def test_cache_refusals():
    p = _prefix()
    for bad in ((0, 3), (2, 0)):
        with pytest.raises(ValueError):
            p.branch(*bad)
    with pytest.raises(ValueError, match="branches of branches"):
        p.branch(2, 3).branch(2, 3)


def test_attention_refuses_what_branches_do_not_take():
    attn = Attention(32, 4, 2)
    c = _prefix().branch(2, 4)
    x, t = z(4, 1, 32), z(1, 4)
    with pytest.raises(ValueError, match="branches take no"):
        attn(x, t, t, kv_cache=c, doc_ids=z(4, 1).int())
    c.tree = (None, None)
    with pytest.raises(ValueError, match="branches take no"):
        attn(x, t, t, kv_cache=c)
    c.tree = None
    attn.capture_attention_weights = True
    with pytest.raises(ValueError, match="branches take no"):
        attn(x, t, t, kv_cache=c)


def test_reorder_moves_the_levels_of_a_ragged_cache(monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "cache_reorder_raw", lambda *a: calls.append(a))
    p = _prefix()
    caches = [p.branch(2, 9) for _ in range(3)]
    par = torch.tensor([[1, 1], [0, -1]], dtype=torch.int32)
    reorder_branches(caches, par)
    assert len(calls) == 1 and calls[0][3] is par and caches[1].lens.tolist() == [0] * 4
    for c in caches:
        c.set_lengths([1, 2, 3, 4])
    reorder_branches(caches, par)
    assert all(c.lens.tolist() == [2, 2, 3, 4] for c in caches)


@pytest.mark.parametrize("shape", [(1, 4), (4, 1), (2, 1), (4,), (2, 3)])
def test_reorder_keeps_to_a_prompts_own_branches(monkeypatch, shape):
    calls = []
    monkeypatch.setattr(ops, "cache_reorder_raw", lambda *a: calls.append(a))
    caches = [_prefix().branch(2, 9)]
    with pytest.raises(ValueError, match="parents must be"):
        reorder_branches(caches, torch.zeros(shape, dtype=torch.int32))
    assert not calls


# ------------------------------------------------------------------ generation
@pytest.fixture
def oracle(monkeypatch):
    def select(logits, scores, *, select):
        s, p, t = branch_ref.select(logits, scores, select)
        return s.float(), p, t

    monkeypatch.setattr(ops, "beam_select_raw", select)
    monkeypatch.setattr(ops, "cache_reorder_raw", lambda *a: None)


def _all(model, prompt, n, eos, penalty):
    """Every continuation with its score, best first."""
    table = torch.log_softmax(model.table.detach().double(), -1)
    V, out = table.shape[0], []
    for k in range(1, n + 1):
        for seq in itertools.product(range(V), repeat=k):
            ended = eos is not None and seq[-1] == eos
            if (k < n and not ended) or (eos is not None and eos in seq[:-1]):
                continue
            s, at = 0.0, int(prompt[-1])
            for t in seq:
                s, at = s + float(table[at, t]), t
            out.append((s / k ** penalty, seq))
    return sorted(out, key=lambda x: -x[0])


@pytest.mark.parametrize("eos", [None, 0])
@pytest.mark.parametrize("penalty", [0.0, 1.0, 2.0, -0.5])
def test_beams_for_every_continuation_find_the_best(oracle, eos, penalty):
    """27 beams of 3 tokens lose no continuation of 3."""
    model = Bigram(3, 7)
    prompt = torch.tensor([[1, 2], [0, 1]])
    out, scores = beam_generate(model, prompt, 3, beams=27, num_return=4, length_penalty=penalty,
                                eos_token_id=eos)
    for b in range(2):
        best = _all(model, prompt[b], 3, eos, penalty)[:4]
        for r, (s, seq) in enumerate(best):
            assert abs(scores[b, r].item() - s) < 1e-5
            row = out[b, r].tolist()
            assert row[:2] == prompt[b].tolist() and tuple(row[2:2 + len(seq)]) == seq
            assert all(t == (eos or 0) for t in row[2 + len(seq):])


def test_one_beam_is_greedy(oracle):
    model = Bigram(11, 3)
    prompt = torch.tensor([[1, 4, 2], [5, 0, 9]])
    out, _ = beam_generate(model, prompt, 9, beams=1)
    assert torch.equal(out[:, 0], generate(model, prompt, 9, temperature=0))


@pytest.mark.parametrize("penalty", [0.0, 1.0, -1.0])
@pytest.mark.parametrize("every", [1, 2, 50])
def test_an_early_end_changes_nothing(oracle, penalty, every):
    """The search that reads back rarely gives what the one that reads back each step does."""
    model = Bigram(9, 4)
    with torch.no_grad():
        model.table[:, 0] += 1.5  # ends often
    prompt = torch.tensor([[1], [5], [8]])
    ref = beam_generate(model, prompt, 12, beams=4, num_return=4, eos_token_id=0,
                        length_penalty=penalty, eos_check_every=1000)
    got = beam_generate(model, prompt, 12, beams=4, num_return=4, eos_token_id=0,
                        length_penalty=penalty, eos_check_every=every)
    assert torch.equal(ref[1], got[1])
    assert torch.equal(ref[0], got[0])


def test_ragged_prompts_and_modes(oracle):
    model = Bigram(7, 5)
    model.train()
    prompt = torch.tensor([[1, 4, 2], [5, 6, 0]])
    out, scores = beam_generate(model, prompt, 4, beams=3, num_return=2, prompt_lens=[3, 1])
    assert model.training
    for b, n in enumerate((3, 1)):
        alone, s = beam_generate(model, prompt[b:b + 1, :n], 4, beams=3, num_return=2)
        assert torch.equal(out[b, :, :n + 4], alone[0]) and torch.allclose(scores[b], s[0])


def test_fewer_continuations_than_asked_for(oracle):
    model = Bigram(2, 5)
    with torch.no_grad():
        model.table[:, 1] = -INF
    out, scores = beam_generate(model, torch.tensor([[0]]), 3, beams=4, num_return=3)
    assert out[0, 0].tolist() == [0] * 4 and torch.isfinite(scores[0, 0])
    assert torch.isinf(scores[0, 1:]).all()


@pytest.mark.parametrize("change", [dict(beams=0), dict(beams=65), dict(num_return=5),
                                    dict(num_return=0), dict(max_new_tokens=0),
                                    dict(max_new_tokens=70), dict(prompt_lens=[3]),
                                    dict(prompt_lens=[0, 1]), dict(eos_check_every=0)])
def test_beam_generate_refusals(oracle, change):
    model = Bigram(7, 5)
    args = dict(max_new_tokens=3, beams=4) | change
    with pytest.raises(ValueError):
        beam_generate(model, torch.tensor([[1, 4], [5, 6]]), args.pop("max_new_tokens"), **args)
    assert model.training


@pytest.mark.parametrize("lens", [None, [2, 1]])
def test_samples_follow_their_prompt(lens):
    """A model whose next token is certain: every sample is the greedy continuation."""
    model = Bigram(5, 1)
    with torch.no_grad():
        model.table.copy_(1e4 * torch.eye(5).roll(1, 1))
    prompt = torch.tensor([[1, 2], [3, 4]])
    out = generate(model, prompt, 3, num_samples=3, prompt_lens=lens)
    one = generate(model, prompt, 3, temperature=0, prompt_lens=lens)
    assert torch.equal(out, one.repeat_interleave(3, 0))
    assert torch.equal(generate(model, prompt, 0, num_samples=2),
                       prompt.repeat_interleave(2, 0))
    with pytest.raises(ValueError):
        generate(model, prompt, 3, num_samples=0)


# ------------------------------------------------------------------ refusals
Q, KV, PRE, C = z(2, 1, 4, 64), z(2, 1, 2, 64), z(1, 2, 6, 64), z(2, 2, 8, 64)
TAB, PLENS, LENS = torch.ones(16, 32), z(1).int(), z(2).int()


@pytest.mark.parametrize("change,kind", [
    (dict(counts=z(3).int()), ValueError), (dict(counts=z(2)), TypeError),
    (dict(q_norm_weight=torch.ones(64)), ValueError), (dict(q=Q.bfloat16()), TypeError),
    (dict(kp=PRE.half(), vp=PRE.half()), TypeError), (dict(k=KV[:1]), ValueError),
    (dict(kp=z(3, 2, 6, 64), vp=z(3, 2, 6, 64)), ValueError), (dict(vp=z(1, 2, 7, 64)), ValueError),
    (dict(kp=z(1, 3, 6, 64), vp=z(1, 3, 6, 64)), ValueError),
    (dict(kp=z(0, 2, 6, 64), vp=z(0, 2, 6, 64)), ValueError),
    (dict(kc=z(2, 8, 2, 64).transpose(1, 2)), ValueError),
    (dict(vp=z(1, 6, 2, 64).transpose(1, 2)), ValueError), (dict(lens=LENS.long()), TypeError),
    (dict(plens=z(2).int()), TypeError), (dict(vc=z(2, 2, 9, 64)), ValueError),
    (dict(q=Q[0]), ValueError), (dict(cos=torch.ones(16, 16)), ValueError),
    (dict(cos=torch.ones(9, 32)), ValueError), (dict(kp=PRE[0]), ValueError),
], ids=lambda x: "-".join(x) if isinstance(x, dict) else x.__name__)
def test_branch_argument_refusals(no_device, change, kind):  # noqa: F811
    a = dict(q=Q, k=KV, v=KV, kp=PRE, vp=PRE.clone(), plens=PLENS, kc=C, vc=C.clone(), lens=LENS,
             cos=TAB, sin=TAB) | change
    tensors = [a.pop(n) for n in ("q", "k", "v", "kp", "vp", "plens", "kc", "vc", "lens", "cos",
                                  "sin")]
    with pytest.raises(kind):
        ops.branch_decode_raw(*tensors, rope_row_offset=0, max_prefix=6, max_len=8, **a)


@pytest.mark.parametrize("max_prefix,max_len,what", [
    (7, 8, "max_prefix"), (6, 9, "max_len"), (-1, 8, "max_prefix"), (6, 0, "positive"),
    (1 << 32, 8, "max_prefix"), (6, (1 << 32) + 8, "max_len"), (-(1 << 40), 8, "max_prefix")])
def test_bounds_past_the_caches(no_device, max_prefix, max_len, what):  # noqa: F811
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    ops_stream, ops._stream = ops._stream, lambda t: 0
    try:
        with pytest.raises(_lib.KernelError, match=what):
            ops.branch_decode_raw(Q, KV, KV, PRE, PRE.clone(), PLENS, C, C.clone(), LENS, TAB, TAB,
                                  rope_row_offset=0, max_prefix=max_prefix, max_len=max_len)
    finally:
        ops._stream = ops_stream


@pytest.mark.parametrize("what", ["batch", "new_tokens", "n_heads", "n_kv_heads", "max_seq_len",
                                  "head_dim", "prefix_length"])
def test_sizes_past_a_c_int(no_device, what):  # noqa: F811
    B, N, Hq, Hkv, S, D, P = 1, 2, 8, 8, 16, 8, 9
    if what == "batch":
        B = BIG
    elif what == "new_tokens":
        N = BIG
    elif what == "n_heads":
        Hq = BIG
    elif what == "n_kv_heads":
        Hkv = BIG
    elif what == "max_seq_len":
        S = BIG
    elif what == "head_dim":
        D = BIG
    else:
        P = BIG
    i32, f32 = torch.int32, torch.float32
    pre = [_meta(1, Hkv, P, D) for _ in range(2)]
    caches = [_meta(B, Hkv, S, D) for _ in range(2)]
    with pytest.raises(ValueError, match=f"{what} is at most"):
        ops.branch_decode_raw(_meta(B, N, Hq, D), _meta(B, N, Hkv, D), _meta(B, N, Hkv, D), *pre,
                              _meta(1, dtype=i32), *caches, _meta(B, dtype=i32),
                              _meta(16, D // 2, dtype=f32), _meta(16, D // 2, dtype=f32),
                              rope_row_offset=0, max_prefix=9, max_len=10)


@pytest.mark.parametrize("logits,scores,select,kind", [
    (z(1, 2, 18)[..., ::2], z(1, 2), 3, ValueError), (z(2, 18), z(2), 3, ValueError),
    (z(1, 65, 4), z(1, 65), 3, ValueError), (z(1, 0, 4), z(1, 0), 3, ValueError),
    (z(1, 2, 4), z(1, 2), 0, ValueError), (z(1, 2, 4), z(1, 2), 129, ValueError),
    (z(1, 2, 4), z(1, 3), 3, ValueError), (z(1, 2, 4), z(1, 2).double(), 3, ValueError),
    (z(1, 2, 4).double(), z(1, 2), 3, TypeError), (_meta(BIG, 1, 4), _meta(BIG, 1), 1, ValueError),
    (_meta(1, 1, BIG), z(1, 1), 1, ValueError)])
def test_select_argument_refusals(no_device, logits, scores, select, kind):  # noqa: F811
    with pytest.raises(kind):
        ops.beam_select_raw(logits, scores, select=select)


@pytest.mark.parametrize("change,kind", [
    (dict(v=[]), ValueError), (dict(k=[], v=[]), ValueError), (dict(v=[C.half()]), ValueError),
    (dict(v=[z(2, 2, 9, 64)]), ValueError), (dict(k=[C.transpose(1, 2)]), ValueError),
    (dict(k=[C[0]], v=[C[0].clone()]), ValueError), (dict(parents=z(2).int()), ValueError),
    (dict(parents=z(3, 1).int()), ValueError), (dict(parents=z(1, 2).long()), TypeError),
    (dict(lens=z(1).int()), TypeError), (dict(lens=LENS.long()), TypeError),
    (dict(k=[z(65, 1, 1, 2)], v=[z(65, 1, 1, 2)], parents=z(1, 65).int(), lens=z(65).int()),
     ValueError),
], ids=lambda x: "-".join(x) if isinstance(x, dict) else x.__name__)
def test_reorder_argument_refusals(change, kind):
    a = dict(k=[C], v=[C.clone()], lens=LENS, parents=z(1, 2).int()) | change
    with pytest.raises(kind):
        ops.cache_reorder_raw(a["k"], a["v"], a["lens"], a["parents"])


def test_entry_points_need_a_gpu():
    for call in (lambda: ops.branch_decode_raw(Q, KV, KV, PRE, PRE, PLENS, C, C, LENS, TAB, TAB,
                                               rope_row_offset=0, max_prefix=6, max_len=8),
                 lambda: ops.beam_select_raw(z(1, 2, 4), z(1, 2), select=2),
                 lambda: ops.cache_reorder_raw([C], [C.clone()], LENS, z(1, 2).int())):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


# ------------------------------------------------------------------ the C ABI
P16 = ctypes.c_void_p(1 << 40)


def _branch(G=1, B=2, N=1, Pmax=9, Smax=8, Hq=4, Hkv=2, D=64, max_prefix=9, max_len=8, dtype=1,
            kp=1 << 44, kc=1 << 45, rows=64, ws=1 << 30, norm=(None, None), q=P16):
    v = ctypes.c_void_p
    return _lib.load().kf_attn_branch(
        q, P16, P16, v(kp), v(kp + (1 << 40)), P16, v(kc), v(kc + (1 << 40)), P16, None, P16, P16, 0,
        rows, P16, P16, ws, G, B, N, Pmax, Smax, Hq, Hkv, D, max_prefix, max_len, *norm, 1e-5, dtype,
        None)


@pytest.mark.parametrize("change,message", [
    (dict(G=0), "multiple"), (dict(B=3, G=2), "multiple"), (dict(max_prefix=-1), "negative"),
    (dict(max_prefix=10), "prefix caches"), (dict(max_len=9), "cache length"), (dict(N=0), "positive"),
    (dict(Hq=5), "multiple"), (dict(D=63), "head_dim"), (dict(D=258), "head_dim"),
    (dict(dtype=3), "dtype"), (dict(B=65536), "65535"), (dict(N=1 << 24), "2\\^26"),
    (dict(rows=0), "rope"), (dict(norm=(P16, None)), "QK-norm"), (dict(q=None), "null"),
    (dict(kp=0), "null"), (dict(kp=(1 << 45) + 64), "overlaps"),
    (dict(Pmax=1 << 31 - 1, max_prefix=(1 << 31) - 4), "."), (dict(ws=0), "workspace")])
def test_branch_abi_refusals(change, message):
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    import re

    assert _branch(**change) != 0
    assert re.search(message, _lib.load().kf_last_error().decode())


@pytest.mark.parametrize("B,N,H,fits", [(2731, 8191, 3, False), (2, (1 << 25) - 1, 1, False),
                                        (4, (1 << 24) - 1, 1, True)])
def test_the_most_rows_a_launch_takes(B, N, H, fits):
    """A workgroup of 256 threads per four rows, and fewer than 2^32 threads: 2^26 - 1 and
    2^26 - 2 rows are refused before anything is written, 2^26 - 4 are not."""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib, n = _lib.load(), _lib.size_out()
    rc = lib.kf_attn_branch_workspace_size(1, B, N, H, H, 96, 9, N, 1, ctypes.byref(n))
    assert (rc == 0) == fits
    assert fits or "2^26" in lib.kf_last_error().decode()


@pytest.mark.parametrize("G,W,V,K,dtype,message", [
    (0, 1, 9, 1, 1, "positive"), (65536, 1, 9, 1, 1, "65535"), (1, 65, 9, 1, 1, "beams"),
    (1, 1, 9, 129, 1, "picked"), (1, 1, (1 << 20) + 1, 1, 1, "vocabulary"), (1, 1, 9, 1, 4, "dtype"),
    (1, 1, 9, 0, 1, "positive")])
def test_select_abi_refusals(G, W, V, K, dtype, message):
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib, n = _lib.load(), _lib.size_out()
    assert lib.kf_beam_select_workspace_size(G, W, V, K, dtype, ctypes.byref(n)) != 0
    assert message in lib.kf_last_error().decode()
    assert lib.kf_beam_select(P16, 9, 9, P16, P16, P16, P16, P16, 1 << 30, G, W, V, K, dtype,
                              None) != 0
    assert lib.kf_beam_select_workspace_size(1, 4, 32000, 8, 0, ctypes.byref(n)) == 0
    assert lib.kf_beam_select(P16, 9, 9, P16, P16, P16, P16, P16, n.value - 1, 1, 4, 32000, 8, 0,
                              None) != 0
    assert "workspace" in lib.kf_last_error().decode()


@pytest.mark.parametrize("n", [2, 300])
@pytest.mark.parametrize("what", ["k", "v", "k and v", "null", "W", "beams"])
def test_reorder_abi_refusals(what, n):
    """Views that overlap, among others.  (The addresses are never read.)"""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    lib = _lib.load()
    B, H, S, D, W = 4, 2, 64, 64, 2
    size, row = B * H * S * D * 2, D * 2
    base = 1 << 40
    k = [base + 2 * c * size for c in range(n)]
    v = [base + (2 * c + 1) * size for c in range(n)]
    if what == "k":
        k[-1] = k[0] + row
    elif what == "v":
        v[0] = v[-1] + size - row
    elif what == "k and v":
        k[-1] = v[0] - row
    elif what == "null":
        v[-1] = 0
    elif what == "W":
        W = 3
    else:
        W = B = 65
    arr = lambda x: (ctypes.c_void_p * n)(*x)  # noqa: E731
    assert lib.kf_kv_cache_reorder(arr(k), arr(v), n, P16, P16, W, B, H, S, D, 1, None) != 0
    message = lib.kf_last_error().decode()
    assert {"null": "null", "W": "multiple", "beams": "at most"}.get(what, "overlap") in message


def test_native_calls_answer_only_their_plain_form():
    native = _lib.native()
    branch = [Q, KV, KV, PRE, PRE, PLENS, C, C, LENS, TAB, TAB, None, None, None, 1e-5, 0, 6, 8, 0, 0]
    select = [z(1, 2, 4), z(1, 2), 2, 0, 0]
    reorder = [[C], [C], LENS, z(1, 2).int(), 0, 0]
    for f, args in ((native.branch, branch), (native.select, select), (native.reorder, reorder)):
        assert f(*args) is None and f() is None and f(*args, 0) is None
        for i in range(len(args)):
            for bad in (None, 3, 1 << 70, "x", [], [None], float("nan")):
                assert f(*args[:i], bad, *args[i + 1:]) is None
    with pytest.raises(TypeError):
        native.bind_branches(1)
