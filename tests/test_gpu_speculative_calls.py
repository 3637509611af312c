"""Generation with drafts on the kernels: calls that its documentation allows."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce
from kempnerforge_amd import _lib
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


def _bad(t):
    """Forms of a tensor that the kernels do not read."""
    yield t.cpu()
    yield t.to(torch.float64)
    yield t[..., :-1] if t.shape[-1] > 1 else t.expand(*t.shape[:-1], 2)
    yield t[None]
    wide = torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)
    yield wide[..., 0]
    yield t.as_subclass(type("Sub", (torch.Tensor,), {}))
    yield t.tolist()


def test_native_calls_refuse_every_other_form():
    """With all other arguments in their plain form, each argument in another one is
    answered with None (and nothing is launched: the caches stay)."""
    announce("native call forms")
    B, N, Hq, Hkv, D, S, V = 2, 3, 4, 2, 64, 16, 9
    i32, bf = torch.int32, torch.bfloat16
    new = lambda *s, dtype=bf: torch.zeros(*s, dtype=dtype, device=DEV)  # noqa: E731
    par = torch.tensor([-1, 0, 0], dtype=i32, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    kc, vc = new(B, Hkv, S, D), new(B, Hkv, S, D)
    tree = [new(B, N, Hq, D), new(B, N, Hkv, D), new(B, N, Hkv, D), kc, vc, new(B, dtype=i32),
            new(S, D // 2, dtype=torch.float32), new(S, D // 2, dtype=torch.float32), par,
            torch.full((B,), N, dtype=i32, device=DEV), new(D, dtype=torch.float32),
            new(D, dtype=torch.float32), 1e-5, 0, S, 0, stream]
    verify = [new(B, N, V), new(B, N, dtype=torch.int64), new(B, N, dtype=torch.float32), None,
              torch.full((B,), N, dtype=i32, device=DEV), new(B, N - 1, V), 1.0, 0, stream]
    keep = [[kc], [vc], [new(B, dtype=i32)], [new(B, dtype=i32)], new(B, N, dtype=i32),
            new(B, dtype=i32), 0, stream]
    native = _lib.native()
    for f, args in ((native.tree, tree), (native.verify, verify), (native.keep, keep)):
        last = len(args) - 1  # (the stream: any number is one)
        for i, a in enumerate(args[:last]):
            if isinstance(a, torch.Tensor):
                bad = list(_bad(a))
                if f is native.verify and i in (0, 5):  # (their rows may have any strides)
                    bad.append(new(*a.shape[:-1], 2 * V)[..., ::2])
            elif isinstance(a, list):
                bad = [[x] for x in _bad(a[0])] + [tuple(a), a * 2, [], [None], None]
            elif a is None:
                bad = [new(N + 1, dtype=i32), 5, "x"]
            else:
                bad = [None, "x", 1 << 70, torch.tensor(1)] + ([7] if i >= last - 1 else [])
            for x in bad:
                got = f(*args[:i], x, *args[i + 1:])
                assert got is None, (f.__name__, i, x if not torch.is_tensor(x) else x.shape)
        assert f(*args) is not None
    torch.cuda.synchronize()
