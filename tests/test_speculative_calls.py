"""Generation with drafts without a GPU: calls that its documentation allows, with the
oracle in place of the kernels."""

from __future__ import annotations

import pytest
import torch

from kempnerforge_amd import ops
from kempnerforge_amd.generate import generate, speculative_generate
from test_speculative import Bigram, oracle  # noqa: F401

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtypes,common", [((F32, BF), F32), ((BF, F32), F32), ((FH, BF), F32),
                                           ((BF, BF), BF)], ids=str)
@pytest.mark.parametrize("kw", [dict(temperature=0.8), dict(temperature=0.8, top_k=3),
                                dict(temperature=0), dict(temperature=0.8, tree=[-1, 0, 0, 1])],
                         ids=str)
def test_models_of_different_dtypes(oracle, monkeypatch, dtypes, common, kw):  # noqa: F811
    """As the kernels ask it, the draft's logits and the target's are of one type, which
    holds both: what was drawn is what is verified."""
    seen, verify = [], ops.verify_drafts_raw

    def check(logits, tokens, uniforms, *, draft_logits=None, **more):
        if draft_logits is not None:
            assert draft_logits.dtype == logits.dtype == common
            seen.append(logits)
        return verify(logits, tokens, uniforms, draft_logits=draft_logits, **more)

    monkeypatch.setattr(ops, "verify_drafts_raw", check)
    model, draft = (Bigram(5, i).to(d) for i, d in enumerate(dtypes))
    prompt = torch.tensor([[1, 2, 3], [0, 4, 4]])
    out = speculative_generate(model, draft, prompt, 9, **kw)
    assert out.shape == (2, 12)
    assert bool(seen) == (kw["temperature"] > 0 and "tree" not in kw)
    if kw["temperature"] == 0:
        assert torch.equal(out, generate(model, prompt, 9, temperature=0))


@pytest.mark.parametrize("training", [(True, True), (False, True), (True, False)], ids=str)
def test_the_models_modes_come_back(oracle, training):  # noqa: F811
    """After the result, and after a refusal: vocabularies that differ, a model without a
    distribution at once, or at a later step, an argument that the verification refuses."""
    def check(model, draft, kind=None, **kw):
        for m, on in zip((model, draft), training):
            m.train(on)
        if kind is None:
            speculative_generate(model, draft, torch.tensor([[1, 2]]), 6, temperature=0, **kw)
        else:
            with pytest.raises(kind):
                speculative_generate(model, draft, torch.tensor([[1, 2]]), 6, temperature=0, **kw)
        assert (model.training, draft.training) == training

    bad, late = Bigram(5, 0), Bigram(5, 0)
    with torch.no_grad():
        bad.table[:] = float("nan")
        late.table[:] = 0.0
        late.table[2, 3] = 1.0  # 2 is followed by 3, and 3 by nothing
        late.table[3] = float("nan")
    check(Bigram(5, 0), Bigram(5, 1))
    check(Bigram(5, 0), Bigram(5, 1), tree=[-1, 0, 0])
    check(Bigram(5, 0), Bigram(9, 1), ValueError)
    check(bad, Bigram(5, 1), RuntimeError)
    check(late, Bigram(5, 1), RuntimeError)
    check(late, Bigram(5, 1), RuntimeError, tree=[-1, 0, 0])


@pytest.mark.parametrize("lens", [None, [2, 1, 3]])
def test_no_new_tokens(oracle, lens):  # noqa: F811
    """generate's result: the prompts, padded on the right to the longest."""
    model, prompt = Bigram(5, 0), torch.tensor([[1, 2, 3, 4], [4, 3, 2, 1], [1, 1, 1, 1]])
    want = generate(model, prompt, 0, prompt_lens=lens, eos_token_id=0)
    got = speculative_generate(model, Bigram(5, 1), prompt, 0, prompt_lens=lens, eos_token_id=0)
    assert torch.equal(got, want)


@pytest.mark.parametrize("tree,forwards", [(None, (6, 14)), ([-1, 0, 0], (6, 11))], ids=str)
def test_forwards_of_a_call(oracle, tree, forwards):  # noqa: F811
    """The model runs for the prompts and once a step, and for nothing else (here every
    draft is refused, so that five steps follow the prompts' token).  The draft model runs
    for its vocabulary, the prompts, and in a step once a level of drafts and once more:
    chains of 2, 2, 2, 2 and then no drafts but the last token, 3 + 3 + 3 + 2 + 1, levels
    of one 2 + 2 + 2 + 2 + 1."""
    model, draft, calls = Bigram(5, 0), Bigram(5, 1), [0, 0]
    with torch.no_grad():
        model.table[:] = torch.eye(5)[[1, 2, 3, 4, 0]]  # counts up
        draft.table[:] = torch.eye(5)  # repeats
        if tree is not None:
            draft.table[:, [0, 1]] = 9.0  # of the next tokens 3, 4, 0, 1, 2 it has 0 and 1
            draft.table[:, 2] = 8.0
            model.table[:] = torch.eye(5)[[3, 3, 3, 4, 3]]  # 3, 4, 3, 4, ..

    def count(i):
        def hook(*_):
            calls[i] += 1
        return hook

    for i, m in enumerate((model, draft)):
        m.register_forward_hook(count(i))
    out = speculative_generate(model, draft, torch.tensor([[2]]), 6, temperature=0, tree=tree,
                               draft_len=2)
    want = [2, 3, 4, 0, 1, 2, 3] if tree is None else [2, 3, 4, 3, 4, 3, 4]
    assert out.tolist() == [want]
    assert tuple(calls) == forwards


@pytest.mark.parametrize("default", [BF, FH, torch.float64])
def test_whatever_the_default_dtype(oracle, monkeypatch, default):  # noqa: F811
    """The random numbers are float32, as the verification asks it."""
    verify = ops.verify_drafts_raw

    def check(logits, tokens, uniforms, **more):
        assert uniforms.dtype == F32
        return verify(logits, tokens, uniforms, **more)

    monkeypatch.setattr(ops, "verify_drafts_raw", check)
    torch.set_default_dtype(default)
    try:
        for kw in (dict(), dict(tree=[-1, 0, 0])):
            out = speculative_generate(Bigram(5, 0), Bigram(5, 1), torch.tensor([[1, 2]]), 6, **kw)
            assert out.shape == (1, 8)
    finally:
        torch.set_default_dtype(F32)
