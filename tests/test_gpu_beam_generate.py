"""Beam search, samples of a prompt and batches behind a system prompt on the GPU: branch
caches through the model, against recomputation without caches."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce, half_ulp
from kempnerforge_amd import Attention, KVCache, reorder_branches
from kempnerforge_amd.generate import beam_generate, generate
from oracle import attention_ref as ref
from spec_util import tree_bound
from test_gpu_branch import reference
from test_gpu_generate import TinyLM

pytestmark = pytest.mark.gpu
INF = float("inf")


def _model(dtype=torch.float32, qk_norm=False, vocab=53, seed=0, **kw):
    torch.manual_seed(seed)
    if dtype == torch.float32:
        return TinyLM(vocab=vocab, qk_norm=qk_norm, **kw).to(DEV)
    return TinyLM(vocab=vocab, dim=1024, n_heads=8, n_kv=2, qk_norm=qk_norm, **kw).to(DEV, dtype)


def _beams(model, prompt, n, W, eos, penalty):
    """Beam search over one prompt (a list) by recomputation without caches, in 64 bits
    behind the logits: (score, tokens) of the finished and the unfinished, best first."""
    live, done = [(0.0, [])], []
    for step in range(1, n + 1):
        rows = torch.tensor([prompt + seq for _, seq in live], device=DEV)
        with torch.no_grad():
            logp = torch.log_softmax(model(rows)[:, -1].double(), -1).cpu()
        total = torch.tensor([s for s, _ in live], dtype=torch.float64)[:, None] + logp
        V = logp.shape[1]
        best = total.flatten().sort(descending=True, stable=True)
        cand = [(v, live[i // V][1] + [i % V]) for v, i in
                zip(best.values[:2 * W].tolist(), best.indices[:2 * W].tolist())]
        done += [(s / step ** penalty, seq) for s, seq in cand[:W] if seq[-1] == eos]
        done = sorted(done, key=lambda x: -x[0])[:W]
        live = [(s, seq) for s, seq in cand if seq[-1] != eos][:W]
    return sorted(done + [(s / n ** penalty, seq) for s, seq in live], key=lambda x: -x[0])


@pytest.mark.parametrize("qk_norm,beams,eos,penalty", [(False, 4, None, 1.0), (True, 3, 7, 1.0),
                                                       (False, 5, 11, 0.0), (False, 1, 2, 1.0),
                                                       (True, 17, 5, 2.0)])
def test_beam_search_matches_recomputation(qk_norm, beams, eos, penalty):
    """float32.  A logit is the last of seven products of 256 terms in a row (projections,
    output and head over two layers).  The roundings of 256 terms are independent, 16 steps
    of 2^-24 together, of terms that are 16 times the sum's size together: 256 steps of the
    logits' magnitude a product, in either of the two evaluations, and a continuation's
    score adds n of them (divided by n^penalty).  The tokens are the same wherever scores
    differ by more."""
    announce(f"beam search {qk_norm} {beams} {eos} {penalty}")
    model = _model(qk_norm=qk_norm)
    prompts, n = [[1, 2, 3, 4, 5, 6, 7], [9, 8, 7, 6, 5, 4, 3]], 10
    out, scores = beam_generate(model, torch.tensor(prompts, device=DEV), n, beams=beams,
                                num_return=min(beams, 3), eos_token_id=eos, length_penalty=penalty)
    with torch.no_grad():
        top = model(torch.tensor(prompts, device=DEV)).abs().max().item()
    for b, prompt in enumerate(prompts):
        want = _beams(model, prompt, n, beams, eos, penalty)
        for r in range(min(beams, 3)):
            tol = 2 * 7 * 256 * 2.0 ** -24 * top * n / n ** penalty
            assert abs(scores[b, r].item() - want[r][0]) < tol, (b, r)
            near = [w for w in want if abs(w[0] - want[r][0]) < 2 * tol]
            row = out[b, r, len(prompt):].tolist()
            assert any(row[:len(seq)] == seq for _, seq in near), (b, r)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ragged_prompts_match_each_alone(dtype):
    announce(f"beam search ragged {dtype}")
    model = _model(dtype, seed=1)
    lens, n = [3, 17, 9], 8 if dtype == torch.float32 else 2
    prompt = torch.randint(0, 53, (3, 17), device=DEV)
    out, scores = beam_generate(model, prompt, n, beams=4, num_return=2, prompt_lens=lens)
    for b, k in enumerate(lens):
        alone, s = beam_generate(model, prompt[b:b + 1, :k], n, beams=4, num_return=2)
        # (as above, a mean over n tokens; 16-bit types: a few steps of 2^-8 of logits whose
        # own rounding is half a one)
        with torch.no_grad():
            top = model(prompt).float().abs().max().item()
        tol = top * (2 * 7 * 256 * 2.0 ** -24 if dtype == torch.float32 else 8 * 2.0 ** -8)
        assert (scores[b] - s[0]).abs().max().item() < tol
        if dtype == torch.float32:
            assert torch.equal(out[b, :, :k + n], alone[0]), b


@pytest.mark.parametrize("lens", [None, [4, 9]])
def test_samples_equal_repeated_prompts(lens):
    """The same random numbers on the same distributions (float32, to 1e-6)."""
    announce(f"samples {lens}")
    model = _model(seed=2)
    prompt = torch.randint(0, 53, (2, 9), device=DEV)
    torch.manual_seed(5)
    a = generate(model, prompt, 12, temperature=0.7, top_k=20, num_samples=4, prompt_lens=lens)
    torch.manual_seed(5)
    b = generate(model, prompt.repeat_interleave(4, 0), 12, temperature=0.7, top_k=20,
                 prompt_lens=None if lens is None else [n for n in lens for _ in range(4)])
    assert torch.equal(a, b)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_questions_behind_a_system_prompt(qk_norm):
    """A system prompt, then right-padded questions of different lengths in one forward,
    then single tokens: the logits of each sequence alone over one cache (float32; the
    tolerance as in the search's test)."""
    announce(f"system prompt {qk_norm}")
    dtype = torch.float32
    model = _model(dtype, qk_norm, seed=3)
    cfg = model.config
    system = torch.randint(0, 53, (1, 70), device=DEV)
    lens, W = [5, 33, 1, 20], 4
    asked = torch.randint(0, 53, (W, 33), device=DEV)
    more = torch.randint(0, 53, (W, 3), device=DEV)

    def caches(B, rows):
        return [KVCache(B, rows, cfg.n_kv_heads, cfg.head_dim, dtype, DEV)
                for _ in range(cfg.n_layers)]

    with torch.no_grad():
        first = caches(1, 70)
        model(system, kv_caches=first)
        for c in first:
            c.use_rope_tables(model._rope_cos.to(DEV), model._rope_sin.to(DEV))
        own = [c.branch(W, 40) for c in first]
        got = [model(asked, kv_caches=own)]
        for c in own:
            c.set_lengths(lens)
        for i in range(3):
            got.append(model(more[:, i:i + 1], kv_caches=own)[:, 0])
        for b, n in enumerate(lens):
            alone = caches(1, 120)
            want = [model(torch.cat([system, asked[b:b + 1, :n]], 1), kv_caches=alone)[0, 70:]]
            for i in range(3):
                want.append(model(more[b:b + 1, i:i + 1], kv_caches=alone)[0, 0])
            for g, w in zip([got[0][b, :n]] + [x[b] for x in got[1:]], want):
                tol = 2 * 7 * 256 * 2.0 ** -24 * w.abs().max().item()
                assert (g - w).abs().max().item() <= tol, b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_a_layer_against_64_bits(dtype, qk_norm):
    """Attention with a branch cache, many tokens and then one: its projections' own values
    through the 64-bit restatement, the output projection's sum of 1024 products in 32
    bits (as many steps of 2^-24 of their magnitudes) of outputs that are off by the
    kernel's bound, rounded once more."""
    announce(f"branch layer {dtype} {qk_norm}")
    torch.manual_seed(6)
    layer = Attention(1024, 8, 2, qk_norm=qk_norm).to(DEV, dtype)
    cos, sin = (t.to(DEV) for t in ref.rope_tables(128, 128, 1e4))
    base = KVCache(2, 70, 2, 128, dtype, DEV)
    norms = {}
    with torch.no_grad():
        if qk_norm:
            for m in (layer.q_norm, layer.k_norm):
                m.weight.copy_(1 + 0.1 * torch.randn(128))
            norms = dict(more=2.0 ** -16, q_norm=layer.q_norm.weight.cpu(),
                         k_norm=layer.k_norm.weight.cpu())
        layer(torch.randn(2, 70, 1024, device=DEV).to(dtype), cos[:70], sin[:70], kv_cache=base)
        base.set_lengths([70, 41])
        base.use_rope_tables(cos, sin)
        own = base.branch(3, 40)
        for N in (33, 1):
            x = torch.randn(6, N, 1024, device=DEV).to(dtype)
            q, k, v = (p(x).view(6, N, -1, 128).cpu() for p in (layer.q_proj, layer.k_proj,
                                                                layer.v_proj))
            kc, vc, lens = own.k.cpu(), own.v.cpu(), own.lens.tolist()
            out = layer(x, cos[own.seq_len:own.seq_len + N], sin[own.seq_len:own.seq_len + N],
                        kv_cache=own)
            assert own.lens.tolist() == [n + N for n in lens]
            want, mag = reference(q, k, v, base.k.cpu(), base.v.cpu(), kc, vc, cos.cpu(), sin.cpu(),
                                  own.k, own.v, [70, 41], lens, None, **norms)
            dot = 1.4 * 1.4 * 128 ** 0.5 if qk_norm else 12.0
            off = tree_bound(want, mag, dtype, 128, 104, dot=dot,
                             moved=2.0 ** -16 * dot if qk_norm else 0.0).flatten(2)
            wo = layer.o_proj.weight.cpu().double()
            y = want.flatten(2) @ wo.T
            bound = (off @ wo.abs().T + 1024 * 2.0 ** -24 * (want.flatten(2).abs() @ wo.abs().T)
                     + half_ulp(y, dtype))
            worst = ((out.cpu().double() - y).abs() / bound).max().item()
            print(f"[layer] worst error / bound {worst:.3f}", flush=True)
            assert worst <= 1.0, (N, worst)


def test_a_step_captured_and_replayed():
    """One beam step (a layer's attention, the selection, the caches' move) in a graph,
    against the same calls made eagerly."""
    announce("beam step graph")
    from kempnerforge_amd import ops

    model = _model(torch.bfloat16, seed=4)
    cfg, G, W, V = model.config, 2, 4, 53
    prompt = torch.randint(0, 53, (G, 30), device=DEV)
    with torch.no_grad():
        base = [KVCache(G, 30, cfg.n_kv_heads, cfg.head_dim, torch.bfloat16, DEV)
                for _ in range(cfg.n_layers)]
        model(prompt, kv_caches=base)
        layer, own = model.layers[0], [c.branch(W, 16) for c in base]
        cos, sin = model._rope_cos.to(DEV), model._rope_sin.to(DEV)
        for c in own:
            c.use_rope_tables(cos, sin)
            c.seq_len = 36
        x = torch.randn(G * W, 1, 1024, device=DEV).bfloat16()
        scores = -torch.rand(G, W, device=DEV)

        def step():
            for c in own:
                c._seq_len = 6
            h = layer(x, cos, sin, kv_cache=own[0])
            best, parents, tokens = ops.beam_select_raw(model.head(h).view(G, W, V), scores,
                                                        select=W)
            reorder_branches(own, parents)
            own[0].lens.sub_(1)
            return best, parents, tokens

        state = [t for c in own for t in (c.k, c.v, c.lens)]

        def fill(seed):
            g = torch.Generator(device=DEV).manual_seed(seed)
            for c in own:
                c.k.normal_(generator=g)
                c.v.normal_(generator=g)
                c.lens.fill_(6)
            x.normal_(generator=g)
            scores.uniform_(-3, 0, generator=g)

        fill(0)
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
            fill(rep)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in (*out, *state)]
            fill(rep)
            want = [*step(), *state]
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want)), rep


def test_two_streams_at_once():
    """Two beam steps' calls on two streams, each with its own workspaces."""
    announce("branch two streams")
    from kempnerforge_amd import ops
    from test_gpu_branch import I32, inputs

    runs = []
    for seed in range(2):
        x = [t.to(DEV) for t in inputs(torch.bfloat16, 2, 6, 1, 32, 8, 128, 3000, 200, seed=seed)]
        lens = I32([10 * b for b in range(12)])
        runs.append((x, I32([2900, 40 + seed]), lens, torch.cuda.Stream()))

    def call(r):
        x, plens, lens, _ = r
        q, k, v, kp, vp, kc, vc, cos, sin = x
        return ops.branch_decode_raw(q, k, v, kp, vp, plens, kc, vc, lens, cos, sin,
                                     rope_row_offset=0, max_prefix=3000, max_len=200)

    want = [call(r) for r in runs]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for r in runs:
            with torch.cuda.stream(r[3]):
                got.append([call(r) for _ in range(3)])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(o, w) for o in g)
