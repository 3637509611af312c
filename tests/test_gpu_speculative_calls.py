"""Generation with drafts on the kernels: calls that its documentation allows."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce
from kempnerforge_amd.generate import _filtered, speculative_generate
from test_gpu_speculative import _lm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [dict(), dict(top_k=4)], ids=str)
def test_a_draft_model_of_another_dtype(kw):
    """A bfloat16 draft for a float32 model: the first two tokens' joint frequencies over
    8192 sequences within 5 standard deviations a cell of the model's own distribution
    (49 cells: by chance once in 35 000 runs, and the seed is fixed)."""
    announce(f"speculative dtypes {kw}")
    model, draft = _lm(4, vocab=7), _lm(5, vocab=7, n_layers=1).bfloat16()
    B, prompt = 4096, torch.randint(0, 7, (1, 5), device=DEV)
    with torch.no_grad():
        T = model(prompt)[0, -1].std().item()
    torch.manual_seed(7)
    count = torch.zeros(49, dtype=torch.long, device=DEV)
    for _ in range(2):
        out = speculative_generate(model, draft, prompt.expand(B, 5).contiguous(), 3,
                                   temperature=T, draft_len=2, **kw)
        count += torch.bincount(out[:, 5] * 7 + out[:, 6], minlength=49)

    def probs(tokens):
        with torch.no_grad():
            x = _filtered(model(tokens)[:, -1] / T, kw.get("top_k", 0), 1.0)
        return torch.softmax(x.double(), -1)

    second = probs(torch.cat([prompt.expand(7, 5), torch.arange(7, device=DEV)[:, None]], 1))
    p = (probs(prompt)[0][:, None] * second).reshape(-1)
    n = count.sum()
    assert p.max() < 0.7 and (p > 0.01).sum() > 5
    z = ((count - n * p) / (n * p * (1 - p)).sqrt().clamp_min(1.0)).abs().max().item()
    print(f"[speculative dtypes {kw}] worst z {z:.2f}", flush=True)
    assert z < 5
    # and the other way round
    out = speculative_generate(draft, model, prompt, 9, temperature=T, draft_len=3, **kw)
    assert out.shape == (1, 14)
