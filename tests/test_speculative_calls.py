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
