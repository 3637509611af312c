"""A speculative step through the module and its caches, and generation with
drafts: the operators together, as a user's program runs them."""

from __future__ import annotations

import pytest
import torch

from gpu_util import DEV, announce, seeded
from kempnerforge_amd import Attention, KVCache, begin_tree, keep_path, ops
from kempnerforge_amd.generate import _filtered, generate, speculative_generate
from kempnerforge_amd.position import precompute_rope_frequencies
from test_gpu_generate import TinyLM

pytestmark = pytest.mark.gpu

TREE = [-1, 0, 0, 0, 1, 1, 2, 3, 4, 4, 6]


def _lm(seed, **kw):
    torch.manual_seed(seed)
    return TinyLM(**kw).to(DEV)


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("tree", [None, TREE, [-1, 0], [-1] + list(range(7))])
def test_greedy_equals_generate(tree, qk_norm):
    """At temperature 0 in float32 the tokens are generate's, whatever the drafts are
    worth: another model's, or the model's own (all accepted)."""
    announce(f"speculative greedy {tree} {qk_norm}")
    model, other = _lm(0, qk_norm=qk_norm), _lm(1, n_layers=1, qk_norm=qk_norm)
    prompt = torch.randint(0, 97, (3, 11), device=DEV)
    want = generate(model, prompt, 24, temperature=0)
    for draft in (other, model):
        got = speculative_generate(model, draft, prompt, 24, temperature=0, tree=tree, draft_len=5)
        assert torch.equal(got, want)
    assert model.training and other.training  # as they were


@pytest.mark.parametrize("tree", [None, TREE])
def test_ragged_prompts_and_eos(tree):
    announce(f"speculative ragged {tree}")
    model, draft = _lm(2, vocab=13), _lm(3, vocab=13, n_layers=1)
    lens = [3, 17, 9, 1]
    prompt = torch.randint(1, 13, (4, 17), device=DEV)
    got = speculative_generate(model, draft, prompt, 30, temperature=0, tree=tree,
                               prompt_lens=lens, eos_token_id=0)
    for b, n in enumerate(lens):
        alone = generate(model, prompt[b:b + 1, :n], 30, temperature=0, eos_token_id=0)[0]
        assert torch.equal(got[b, :alone.numel()], alone), b
        assert (got[b, alone.numel():] == 0).all()


@pytest.mark.parametrize("kw", [dict(), dict(tree=[-1, 0, 0, 1]), dict(top_k=4),
                                dict(top_p=0.7, tree=[-1, 0, 0, 1])], ids=str)
def test_samples_follow_the_model(kw):
    """The joint frequencies of the first two emitted tokens over 8192 sequences of one
    prompt against the model's own distribution, within 5 standard deviations a cell
    (49 cells: by chance once in 35 000 runs, and the seed is fixed)."""
    announce(f"speculative distribution {kw}")
    model, draft = _lm(4, vocab=7), _lm(5, vocab=7, n_layers=1)
    B, prompt = 4096, torch.randint(0, 7, (1, 5), device=DEV)
    with torch.no_grad():  # a temperature at which the logits leave a choice
        T = model(prompt)[0, -1].std().item()
    torch.manual_seed(7)
    count = torch.zeros(49, dtype=torch.long, device=DEV)
    for _ in range(2):
        out = speculative_generate(model, draft, prompt.expand(B, 5).contiguous(), 3,
                                   temperature=T, draft_len=2, **kw)
        count += torch.bincount(out[:, 5] * 7 + out[:, 6], minlength=49)

    def probs(tokens):
        with torch.no_grad():
            x = _filtered(model(tokens)[:, -1] / T, kw.get("top_k", 0), kw.get("top_p", 1.0))
        return torch.softmax(x.double(), -1)

    first = probs(prompt)[0]
    second = probs(torch.cat([prompt.expand(7, 5), torch.arange(7, device=DEV)[:, None]], 1))
    p = (first[:, None] * second).reshape(-1)
    n = count.sum()
    assert p.max() < 0.7 and (p > 0.01).sum() > 5
    assert count[p == 0].sum() == 0
    z = ((count - n * p) / (n * p * (1 - p)).sqrt().clamp_min(1.0)).abs().max().item()
    print(f"[speculative distribution {kw}] worst z {z:.2f}", flush=True)
    assert z < 5


@pytest.mark.parametrize("tree", [None, TREE])
def test_bfloat16_steps_emit_their_own_argmax(tree):
    """head_dim 128 in bfloat16: every emitted token is the most likely one of the
    logits of the step that scored its predecessor, and those are finite.  (Not
    compared with a forward over the whole sequence: this model's second layer has
    scores near 1e5, where bfloat16's half step of a query, 2^-9, is 200 in the
    exponent, so that any other order of rounding picks other keys.)"""
    announce(f"speculative bf16 {tree}")
    torch.manual_seed(8)
    model = TinyLM(dim=1024, n_heads=8, n_kv=2).to(DEV, torch.bfloat16)
    prompt = torch.randint(0, 97, (4, 9), device=DEV)
    seen = []  # per forward of all layers: fill levels, tokens, parents, best tokens
    draft = TinyLM(dim=1024, n_heads=8, n_kv=2).to(DEV, torch.bfloat16)
    draft.load_state_dict(model.state_dict())

    def record(module, args, kwargs, out):
        caches = kwargs.get("kv_caches")
        if caches is not None and caches[0].tree is not None:
            assert out.isfinite().all()
            seen.append((caches[0].lens.tolist(), args[0].tolist(), out.argmax(-1).tolist()))

    model.register_forward_hook(record, with_kwargs=True)
    out = speculative_generate(model, draft, prompt, 16, temperature=0, tree=tree)
    checked = 0
    for lens, tokens, best in seen:
        n = len(tokens[0])
        par = list(range(-1, n - 1)) if tree is None else tree[:n]
        for b in range(4):
            row, at, pos = out[b].tolist(), 0, lens[b]
            if pos + 1 >= len(row):
                continue  # finished
            assert tokens[b][0] == row[pos]
            while at is not None and pos + 1 < len(row):
                assert best[b][at] == row[pos + 1], (b, pos)
                checked += 1
                at = next((c for c in range(n) if par[c] == at and tokens[b][c] == row[pos + 1]),
                          None)
                pos += 1
    assert checked == 4 * 15  # all but the first of each sequence, which the prompt gave


@pytest.mark.parametrize("dtype,head_dim", [(torch.float32, 64), (torch.bfloat16, 128),
                                            (torch.float32, 32)])
def test_one_layer_step_by_step(dtype, head_dim):
    """A tree step of one Attention layer: each node's output is what a fresh cache
    gives for the tokens of its own path, and after keep_path the cache decodes on
    as if the accepted tokens had been fed one by one."""
    announce(f"module tree step {dtype} {head_dim}")
    torch.manual_seed(9)
    Hq, Hkv = 4, 2
    layer = Attention(Hq * head_dim, Hq, Hkv, head_dim=head_dim, qk_norm=True).to(DEV, dtype)
    cos, sin = (t.to(DEV) for t in precompute_rope_frequencies(head_dim, 64))
    B, S, N = 2, 13, len(TREE)
    x = seeded((B, S + N + 1, Hq * head_dim), 0, dtype).to(DEV)
    parents = torch.tensor(TREE, device=DEV)

    def cache():
        return KVCache(B, 40, Hkv, head_dim, dtype, DEV)

    def feed(c, xs, at):
        return layer(xs, cos[at:at + xs.shape[1]], sin[at:at + xs.shape[1]], kv_cache=c)

    tol = 1e-5 if dtype == torch.float32 else 4e-2
    with torch.no_grad():
        c = cache()
        feed(c, x[:, :S], 0)
        begin_tree([c], parents)
        out = feed(c, x[:, S:S + N], S)
        assert c.seq_len == S and c.lens.tolist() == [S, S]
        for i in range(N):
            chain, j = [], i
            while j >= 0:
                chain.insert(0, j)
                j = TREE[j]
            ref = cache()
            feed(ref, x[:, :S], 0)
            for d, j in enumerate(chain):
                one = feed(ref, x[:, S + j:S + j + 1], S + d)
            err = (out[:, i:i + 1].float() - one.float()).abs().max().item()
            assert err <= tol * max(1.0, one.float().abs().max().item()), (i, err)
        # accept nodes 0, 2, 6 and 10 in row 0, and 0, 1 in row 1
        path = torch.full((B, N), -1, dtype=torch.int32, device=DEV)
        path[0, :4] = torch.tensor([0, 2, 6, 10], dtype=torch.int32)
        path[1, :2] = torch.tensor([0, 1], dtype=torch.int32)
        kept = torch.tensor([4, 2], dtype=torch.int32, device=DEV)
        keep_path([c], path, kept)
        assert c.tree is None and c.seq_len == S + 4 and c.ragged
        assert c.lens.tolist() == [S + 4, S + 2]
        c.use_rope_tables(cos, sin)
        nxt = x[:, S + N:]
        got = layer(nxt, cos[:1], sin[:1], kv_cache=c)
        for b, chain in enumerate(([0, 2, 6, 10], [0, 1])):
            ref = KVCache(1, 40, Hkv, head_dim, dtype, DEV)
            layer(x[b:b + 1, :S], cos[:S], sin[:S], kv_cache=ref)
            for d, j in enumerate(chain):
                feed(ref, x[b:b + 1, S + j:S + j + 1], S + d)
            one = feed(ref, nxt[b:b + 1], S + len(chain))
            err = (got[b:b + 1].float() - one.float()).abs().max().item()
            assert err <= tol * max(1.0, one.float().abs().max().item()), (b, err)


class _Step:
    """The three operators over a model's caches, as a serving loop runs them: two
    layers' attention, the verification, the move."""

    def __init__(self, seed, B, N, V, tree, layers=2, dtype=torch.bfloat16):
        Hq, Hkv, D, S = 8, 2, 128, 400
        dev = lambda t: t.to(DEV)  # noqa: E731
        self.q = [dev(seeded((B, N, Hq, D), seed + i, dtype)) for i in range(layers)]
        self.k = [dev(seeded((B, N, Hkv, D), seed + 10 + i, dtype)) for i in range(layers)]
        self.kc = [dev(seeded((B, Hkv, S, D), seed + 20 + i, dtype)) for i in range(layers)]
        self.vc = [dev(seeded((B, Hkv, S, D), seed + 30 + i, dtype)) for i in range(layers)]
        self.lens = [dev(torch.tensor([37 * (b + 1) for b in range(B)], dtype=torch.int32))
                     for _ in range(layers)]
        self.parents = None if tree is None else dev(torch.tensor(tree, dtype=torch.int32))
        self.head = dev(seeded((Hq * D, V), seed + 40, dtype))
        self.tokens = dev(torch.randint(0, V, (B, N), generator=torch.Generator().manual_seed(seed)))
        self.u = dev(torch.rand(B, N, generator=torch.Generator().manual_seed(seed + 1)))
        self.cos, self.sin = (dev(t) for t in precompute_rope_frequencies(D, S))

    def state(self):
        return self.kc + self.vc + self.lens

    def __call__(self):
        x = 0
        for i in range(len(self.q)):
            x = x + ops.tree_decode_raw(self.q[i], self.k[i], self.k[i], self.kc[i], self.vc[i],
                                        self.lens[i], self.cos, self.sin, rope_row_offset=0,
                                        max_len=400, parents=self.parents)
        logits = x.flatten(2) @ self.head
        path, kept, token = ops.verify_drafts_raw(logits, self.tokens, self.u, temperature=40.0,
                                                  parents=self.parents)
        ops.cache_keep_raw(self.kc, self.vc, self.lens, path, kept)
        return path, kept, token


STEPS = [(0, 3, 11, 4, TREE), (100, 2, 5, 3, None)]  # (few tokens, so that drafts are accepted)


def _eager(runs):
    """Outputs of `runs` steps one after the other, and the state they leave."""
    steps = [_Step(*cfg) for cfg in STEPS]
    outs = [[[t.clone() for t in s()] for _ in range(runs)] for s in steps]
    torch.cuda.synchronize()
    return steps, outs


def test_whole_steps_captured_and_replayed():
    """Each step's graph replayed in turn with the other's and with eager calls between:
    tokens, caches and lengths as from eager steps."""
    announce("speculative step graphs")
    runs = 4
    want_steps, want = _eager(runs)
    assert any(k > 1 for outs in want for o in outs for k in o[1].tolist())
    steps = [_Step(*cfg) for cfg in STEPS]
    other = _Step(7, 4, 20, 100, None)
    graphs, outs = [], []
    for s in steps:
        saved = [t.clone() for t in s.state()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for t, x in zip(s.state(), saved):
            t.copy_(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s())
        graphs.append(g)
    for r in range(runs):
        for i, g in enumerate(graphs):
            g.replay()
            if r % 2:
                other()
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want[i][r]):
                assert torch.equal(a, b), (r, i)
    for s, w in zip(steps, want_steps):
        for a, b in zip(s.state(), w.state()):
            assert torch.equal(a, b)


def test_steps_on_two_streams_at_once():
    announce("speculative steps on two streams")
    runs = 6
    want_steps, want = _eager(runs)
    steps = [_Step(*cfg) for cfg in STEPS]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[] for _ in steps]
    for _ in range(runs):
        for i, (s, st) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(st):
                got[i].append([t.clone() for t in s()])
    torch.cuda.synchronize()
    for i in range(len(steps)):
        for a, b in zip(got[i], want[i]):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        for a, b in zip(steps[i].state(), want_steps[i].state()):
            assert torch.equal(a, b)


def test_plain_and_other_forms_of_a_call_agree():
    """Arguments that Python converts (other integer types, strided views, a tensor's
    subclass, numbers as tensors) give the bits of the plain form."""
    announce("speculative call forms")
    s = _Step(3, 3, 11, 7, TREE, layers=1)
    s2 = _Step(3, 3, 11, 7, TREE, layers=1)

    class Sub(torch.Tensor):
        pass

    wide = torch.empty(3, 11, 8, 200, dtype=torch.bfloat16, device=DEV)
    wide[..., :128] = s2.q[0]
    kw = dict(rope_row_offset=0, max_len=400)
    counts = torch.tensor([11, 4, 0], dtype=torch.int32, device=DEV)
    a = ops.tree_decode_raw(s.q[0], s.k[0], s.k[0], s.kc[0], s.vc[0], s.lens[0], s.cos, s.sin,
                            parents=s.parents, counts=counts, **kw)
    b = ops.tree_decode_raw(wide[..., :128], s2.k[0].as_subclass(Sub), s2.k[0], s2.kc[0], s2.vc[0],
                            s2.lens[0], s2.cos.double(), s2.sin, parents=s2.parents.long(),
                            counts=counts.long(), rope_row_offset=0,
                            max_len=torch.tensor(400))
    assert torch.equal(a, b) and torch.equal(s.kc[0], s2.kc[0]) and torch.equal(s.vc[0], s2.vc[0])
    logits = (a.flatten(2) @ s.head).float()
    a = ops.verify_drafts_raw(logits, s.tokens, s.u, temperature=1.0, parents=s.parents,
                              counts=counts)
    b = ops.verify_drafts_raw(logits, s.tokens.int(), s.u.t().contiguous().t(), temperature=True,
                              parents=s.parents.expand(3, 11), counts=counts.long())
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    lens = [torch.zeros(3, dtype=torch.int32, device=DEV) for _ in range(2)]
    ops.cache_keep_raw(s.kc, s.vc, s.lens, a[0], a[1], lens_out=lens[:1])
    ops.cache_keep_raw(tuple(s2.kc), s2.vc, s2.lens, a[0].t().contiguous().t(), a[1],
                       lens_out=lens[1:])
    assert torch.equal(*lens) and torch.equal(s.kc[0], s2.kc[0])


def test_refusals_keep_their_errors_on_the_device():
    """What the host's checks refuse (all before any launch), with tensors on the GPU."""
    announce("speculative host refusals")
    s = _Step(3, 3, 11, 7, None, layers=1)
    args = [s.q[0], s.k[0], s.k[0], s.kc[0], s.vc[0], s.lens[0], s.cos, s.sin]
    before = [t.clone() for t in s.state()]
    for kw, kind in ((dict(max_len=401), RuntimeError), (dict(max_len=0), RuntimeError),
                     (dict(max_len=(1 << 32) + 8), RuntimeError),
                     (dict(max_len=8 - (1 << 32)), RuntimeError),
                     (dict(max_len=400, parents=s.tokens), ValueError),
                     (dict(max_len=400, counts=s.u[0]), TypeError),
                     (dict(max_len=400, parents=torch.zeros(11).int()), RuntimeError),
                     (dict(max_len=400, q_norm_weight=torch.ones(128, device=DEV)), ValueError)):
        if "parents" in kw and kw["parents"] is s.tokens:
            kw["parents"] = s.tokens[:, :5]
        with pytest.raises(kind):
            ops.tree_decode_raw(*args, rope_row_offset=0, **kw)
    logits = torch.zeros(3, 11, 7, device=DEV)
    for kw, kind in ((dict(temperature=-1.0), RuntimeError),
                     (dict(temperature=float("nan")), RuntimeError),
                     (dict(draft_logits=logits), ValueError),
                     (dict(draft_logits=logits[:, 1:], temperature=0), ValueError)):
        with pytest.raises(kind):
            ops.verify_drafts_raw(logits, s.tokens, s.u, **kw)
    path, kept = torch.zeros(3, 11, device=DEV).int(), torch.zeros(3, device=DEV).int()
    for a in (([s.kc[0]], [s.kc[0]], s.lens, path, kept), (s.kc, s.vc, s.lens, path, kept.long()),
              (s.kc * 2, s.vc * 2, s.lens * 2, path, kept), (s.kc, s.vc, [s.lens[0][:2]], path, kept)):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            ops.cache_keep_raw(*a)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(s.state(), before))


def test_a_draft_row_without_a_distribution_is_refused():
    """Its token is refused and the next one drawn from the target's row."""
    announce("verify bad draft rows")
    B, N, V = 3, 4, 50
    g = torch.Generator().manual_seed(0)
    logits, u = torch.randn(B, N, V, generator=g), torch.rand(B, N, generator=g)
    tokens = torch.randint(0, V, (B, N), generator=g)
    drafts = torch.randn(B, N - 1, V, generator=g)
    drafts[0, 0], drafts[1, 0], drafts[2, 0] = float("nan"), -float("inf"), float("inf")
    dev = [t.to(DEV) for t in (logits, tokens, u)]
    path, kept, token = ops.verify_drafts_raw(*dev, draft_logits=drafts.to(DEV))
    one = ops.verify_drafts_raw(dev[0][:, :1], dev[1][:, :1].contiguous(),
                                dev[2][:, :1].contiguous())
    assert kept.tolist() == [1, 1, 1] and torch.equal(token, one[2])
