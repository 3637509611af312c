"""Generation with drafts without a GPU: its bookkeeping with the oracle in place of
the kernels, and the refusals of the entry points."""

from __future__ import annotations

import contextlib
from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn

from kempnerforge_amd import Attention, KVCache, _lib, begin_tree, keep_path, ops
from kempnerforge_amd.generate import generate, speculative_generate
from oracle import spec_ref

z = torch.zeros


class Bigram(nn.Module):
    """Logits from a table of the last token; the caches only count.  Refuses tokens
    outside its table and positions past its length."""

    def __init__(self, vocab, seed, max_seq_len=64):
        super().__init__()
        self.config = SimpleNamespace(max_seq_len=max_seq_len, n_layers=2, n_kv_heads=1,
                                      head_dim=8, rope_theta=1e4)
        g = torch.Generator().manual_seed(seed)
        self.table = nn.Parameter(2 * torch.randn(vocab, vocab, generator=g))

    def forward(self, tokens, kv_caches=None):
        assert 0 <= tokens.min() and tokens.max() < self.table.shape[0]
        for c in kv_caches or ():
            c._check_room(tokens.shape[1])
            if c.tree is None:
                c._advance(tokens.shape[1])
            else:
                assert c.lens.max() < self.config.max_seq_len
        return self.table[tokens]


@pytest.fixture
def oracle(monkeypatch):
    def verify(logits, tokens, uniforms, *, temperature, parents=None, counts=None,
               draft_logits=None):
        B, N = tokens.shape
        chain = list(range(-1, N - 1))
        par = [chain if parents is None else parents.tolist()] * B
        path, kept, nxt = spec_ref.verify(logits, tokens, uniforms, temperature, par, counts,
                                          draft_logits)
        path = [list(p) + [-1] * (N - len(p)) for p in path]
        return torch.tensor(path, dtype=torch.int32), torch.tensor(kept), torch.tensor(nxt)

    def keep(ks, vs, lens, path, kept):
        for t in lens:
            t += kept.to(torch.int32)

    monkeypatch.setattr(ops, "verify_drafts_raw", verify)
    monkeypatch.setattr(ops, "cache_keep_raw", keep)


@pytest.mark.parametrize("tree", [None, [-1, 0], [-1, 0, 0, 1, 1, 2, 3], [-1] + [0] * 6])
@pytest.mark.parametrize("new", [1, 2, 13])
def test_greedy_bookkeeping(oracle, tree, new):
    model, draft = Bigram(5, 0), Bigram(5, 1)
    prompt = torch.randint(0, 5, (6, 7), generator=torch.Generator().manual_seed(2))
    want = generate(model, prompt, new, temperature=0)
    for d in (draft, model):
        assert torch.equal(speculative_generate(model, d, prompt, new, temperature=0, tree=tree,
                                                draft_len=3), want)
    lens = [1, 7, 3, 4, 5, 2]
    got = speculative_generate(model, draft, prompt, new, temperature=0, tree=tree,
                               prompt_lens=lens, eos_token_id=3)
    for b, n in enumerate(lens):
        alone = generate(model, prompt[b:b + 1, :n], new, temperature=0, eos_token_id=3)[0]
        assert torch.equal(got[b, :alone.numel()], alone) and (got[b, alone.numel():] == 3).all()


def test_up_to_the_models_length(oracle):
    """No position past max_seq_len is asked for, however deep the drafts."""
    model, draft = Bigram(5, 0, max_seq_len=12), Bigram(5, 1, max_seq_len=12)
    prompt = torch.tensor([[1, 2, 3]])
    out = speculative_generate(model, model, prompt, 9, temperature=0, draft_len=20)
    assert torch.equal(out, generate(model, prompt, 9, temperature=0))
    out = speculative_generate(model, draft, prompt, 9, temperature=0.5, draft_len=20)
    assert out.shape == (1, 12)


def test_a_model_without_distribution(oracle):
    bad = Bigram(5, 0)
    with torch.no_grad():
        bad.table[:] = float("nan")
    with pytest.raises(RuntimeError, match="distribution"):
        speculative_generate(bad, Bigram(5, 1), torch.tensor([[1, 2]]), 4)


@pytest.mark.parametrize("kw,word", [
    (dict(tree=[-1, 0, 1, 0]), "level by level"), (dict(tree=[-1, 0, -1]), "parent"),
    (dict(tree=[-1, 2, 0]), "parent"), (dict(tree=[-1]), "nodes"),
    (dict(tree=[-1] + [0] * 256), "nodes"), (dict(draft_len=256), "draft_len"),
    (dict(draft_len=0), "draft_len"), (dict(max_new_tokens=70), "max_seq_len"),
    (dict(prompt_lens=[0]), "prompt_lens"), (dict(prompt_lens=[1, 1]), "prompt_lens"),
    (dict(draft=Bigram(9, 1)), "vocabularies"), (dict(draft=Bigram(3, 1)), "vocabularies"),
])
def test_generation_refusals(oracle, kw, word):
    """Before any token of one model reaches the other: the last token of the prompt
    is not in the smaller vocabulary."""
    kw = dict(kw)
    draft, new = kw.pop("draft", None) or Bigram(5, 1), kw.pop("max_new_tokens", 4)
    with pytest.raises(ValueError, match=word):
        speculative_generate(Bigram(5, 0), draft, torch.tensor([[1, 4]]), new, **kw)


def test_module_refusals():
    layer = Attention(32, 4, 2, head_dim=8)
    c = KVCache(1, 16, 2, 8, torch.float32, "cpu")
    begin_tree([c])
    cos, sin = torch.ones(4, 4), z(4, 4)
    x = z(1, 4, 32)
    with pytest.raises(ValueError, match="tree"):
        layer(x, cos, sin, kv_cache=c, key_padding_mask=torch.ones(1, 4).bool())
    with pytest.raises(ValueError, match="tree"):
        layer(x, cos, sin, kv_cache=c, doc_ids=z(1, 4).long())
    with pytest.raises(ValueError, match="overflow"):
        layer(z(1, 17, 32), cos, sin, kv_cache=c)
    with pytest.raises(RuntimeError, match="GPU"):
        layer(x, cos, sin, kv_cache=c)
    c.set_lengths([3])
    c.ragged = True
    with pytest.raises(ValueError, match="use_rope_tables"):
        layer(x, cos, sin, kv_cache=c)


@pytest.fixture
def no_device(monkeypatch):
    """The checks behind the test for a device, with the library's own refusals; what
    got past all of them would end at the stream."""
    def stream(t):
        raise AssertionError("nothing was refused")

    monkeypatch.setattr(ops, "_one_device", lambda *t: 0)
    monkeypatch.setattr(ops, "_on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", stream)


Q, KV, C = z(1, 2, 4, 64), z(1, 2, 2, 64), z(1, 2, 8, 64)
TAB, LENS = torch.ones(8, 32), z(1).int()


@pytest.mark.parametrize("change,kind", [
    (dict(parents=z(3).int()), ValueError), (dict(parents=z(2)), TypeError),
    (dict(parents=z(2, 2).int()), ValueError), (dict(counts=z(2).int()), ValueError),
    (dict(counts=z(1)), TypeError), (dict(q_norm_weight=torch.ones(64)), ValueError),
    (dict(q=Q.bfloat16()), TypeError), (dict(k=KV[:, :1]), ValueError),
    (dict(q=z(1, 257, 4, 64), k=z(1, 257, 2, 64), v=z(1, 257, 2, 64)), ValueError),
    (dict(kc=z(1, 8, 2, 64).transpose(1, 2)), ValueError), (dict(lens=LENS.long()), TypeError),
    (dict(lens=z(2).int()), TypeError), (dict(vc=z(1, 2, 9, 64)), ValueError),
    (dict(q=Q[0]), ValueError), (dict(cos=torch.ones(8, 16)), ValueError),
    (dict(cos=torch.ones(9, 32)), ValueError),
], ids=lambda x: "-".join(x) if isinstance(x, dict) else x.__name__)
def test_tree_argument_refusals(no_device, change, kind):
    a = dict(q=Q, k=KV, v=KV, kc=C, vc=C.clone(), lens=LENS, cos=TAB, sin=TAB) | change
    tensors = [a.pop(n) for n in ("q", "k", "v", "kc", "vc", "lens", "cos", "sin")]
    with pytest.raises(kind):
        ops.tree_decode_raw(*tensors, rope_row_offset=0, max_len=8, **a)


LOG, TOK, U = z(1, 3, 9), z(1, 3).long(), z(1, 3)


@pytest.mark.parametrize("change,kind", [
    (dict(logits=z(1, 3, 18)[..., ::2]), ValueError), (dict(tokens=TOK[:, :2]), ValueError),
    (dict(tokens=TOK.float()), TypeError), (dict(uniforms=U.double()), TypeError),
    (dict(draft_logits=LOG), ValueError), (dict(logits=LOG[0]), ValueError),
    (dict(draft_logits=LOG[:, :2], parents=z(3).int()), ValueError),
    (dict(draft_logits=LOG[:, :2], temperature=0), ValueError),
    (dict(draft_logits=LOG[:, :2].half()), ValueError), (dict(counts=z(2).int()), ValueError),
    (dict(logits=z(1, 257, 9), tokens=z(1, 257).long(), uniforms=z(1, 257)), ValueError),
    (dict(logits=LOG.double()), TypeError),
], ids=lambda x: "-".join(x) if isinstance(x, dict) else x.__name__)
def test_verify_argument_refusals(no_device, change, kind):
    a = dict(logits=LOG, tokens=TOK, uniforms=U) | change
    with pytest.raises(kind):
        ops.verify_drafts_raw(a.pop("logits"), a.pop("tokens"), a.pop("uniforms"), **a)


PATH, KEPT = z(1, 3).int(), z(1).int()


@pytest.mark.parametrize("change,kind", [
    (dict(k=[]), ValueError), (dict(v=[]), ValueError), (dict(lens=[LENS, LENS]), ValueError),
    (dict(lens=[LENS.long()]), TypeError), (dict(lens=[z(2).int()]), TypeError),
    (dict(path=PATH.long()), TypeError), (dict(kept=KEPT.long()), TypeError),
    (dict(path=z(2, 3).int()), ValueError), (dict(path=z(1, 257).int()), ValueError),
    (dict(v=[C.half()]), ValueError), (dict(v=[z(1, 8, 2, 64).transpose(1, 2)]), ValueError),
    (dict(v=[z(1, 2, 9, 64)]), ValueError), (dict(k=[C[0]], v=[C[0].clone()]), ValueError),
    (dict(), RuntimeError),
], ids=lambda x: "-".join(x) if isinstance(x, dict) else x.__name__)
def test_keep_argument_refusals(change, kind):
    a = dict(k=[C], v=[C.clone()], lens=[LENS], path=PATH, kept=KEPT) | change
    # (all tensors on the CPU: refused for that at the latest)
    with pytest.raises((kind, RuntimeError)):
        ops.cache_keep_raw(a["k"], a["v"], a["lens"], a["path"], a["kept"])


def test_keep_path_without_the_lengths(oracle):
    """The fill levels are read back where the caller does not know them."""
    caches = [KVCache(2, 16, 1, 8, torch.float32, "cpu") for _ in range(3)]
    for c in caches:
        c.set_lengths([4, 4])
    begin_tree(caches)
    keep_path(caches, z(2, 3).int(), torch.tensor([3, 1]))
    for c in caches:
        assert c.lens.tolist() == [7, 5] and c.seq_len == 7 and c.ragged and c.tree is None
    with pytest.raises(ValueError, match="lengths"):
        keep_path(caches, z(2, 3).int(), torch.tensor([3, 1]), [7])


def test_native_calls_answer_only_their_plain_form():
    """Tensors off the GPU, other objects and argument lists of another length are
    left to Python; nothing is read from them."""
    native = _lib.native()
    tree = [Q, KV, KV, C, C, LENS, TAB, TAB, None, None, None, None, 1e-5, 0, 8, 0, 0]
    verify = [LOG, TOK, U, None, None, None, 1.0, 0, 0]
    keep = [[C], [C], [LENS], [LENS], PATH, KEPT, 0, 0]
    for f, args in ((native.tree, tree), (native.verify, verify), (native.keep, keep)):
        assert f(*args) is None and f() is None and f(*args, 0) is None
        for i in range(len(args)):
            for bad in (None, 3, 1 << 70, "x", [], [None], float("nan")):
                assert f(*args[:i], bad, *args[i + 1:]) is None
    with pytest.raises(TypeError):
        native.bind(1)
    with pytest.raises(ValueError):
        native.bind(0, 0, 0, 0, 0)
    with pytest.raises(TypeError):
        native.bind("x", 0, 0, 0, 0)
