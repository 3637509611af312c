"""Autoregressive generation over the gfx950 KV-cache decode, with ragged batches.

``sample`` and ``generate`` keep the signatures and results of
``kempnerforge/model/generate.py:15-124`` (temperature, top-k, top-p sampling;
prefill, then one token per step through the model with one ``KVCache`` per
layer).  Three additions, all off by default:

* ``prompt_lens``: prompts of different lengths in one batch, right-padded in
  ``prompt_tokens``.  The prefill runs on the padded batch, then every layer's
  cache gets the per-sequence lengths and the model's full RoPE tables, so each
  sequence continues from its own last prompt token at its own position (the
  padding is overwritten as the sequence grows and is never attended).  The
  reference can only batch prompts of one length.
* ``eos_check_every``: how often the all-sequences-finished test reads back to
  the host.  The reference reads it every step (a device synchronisation per
  token); every N steps keeps the GPU queue full, and the output is cut at the
  step where the last sequence finished, so it is the same as the reference's
  (up to N - 1 decode steps are computed and discarded).

* ``num_samples``: several continuations of each prompt.  The prompt is prefilled and
  its keys and values are kept and read once for all of them (``BranchKVCache``).

``beam_generate`` (no counterpart in the reference) keeps the most likely continuations
of each prompt, likewise behind one copy of it.

``speculative_generate`` (no counterpart in the reference) emits tokens of the same
distribution several at a time: a smaller model drafts a chain or a tree of them,
one forward of the model scores all, and the accepted path is kept.

The model is the reference's ``Transformer`` contract: ``model(tokens,
kv_caches=...)`` returns logits ``(batch, seq, vocab)``, ``model.config`` has
``max_seq_len``, ``n_layers``, ``n_kv_heads``, ``head_dim`` and ``rope_theta``,
and the attention layers are ``kempnerforge_amd.Attention``.
"""

from __future__ import annotations

import contextlib

import torch

from kempnerforge_amd import ops
from kempnerforge_amd.attention import KVCache, begin_tree, keep_path, reorder_branches
from kempnerforge_amd.position import precompute_rope_frequencies


def sample(logits: torch.Tensor, temperature: float = 1.0, top_k: int = 0,
           top_p: float = 1.0) -> torch.Tensor:
    """Next token ids ``(batch,)`` from logits ``(batch, vocab)``: greedy at
    temperature 0, else temperature, top-k, then nucleus filtering and a
    multinomial draw (``kempnerforge/model/generate.py:15-56``)."""
    if temperature == 0:
        return logits.argmax(dim=-1)
    logits = _filtered(logits / temperature, top_k, top_p)
    return torch.multinomial(logits.softmax(dim=-1), num_samples=1).squeeze(-1)


def _filtered(logits: torch.Tensor, top_k: int, top_p: float) -> torch.Tensor:
    """Rows ``(rows, vocab)`` of scaled logits with -inf at the tokens that top-k and
    nucleus filtering leave out."""
    if top_k > 0:
        top_k = min(top_k, logits.shape[-1])
        threshold = logits.topk(top_k, dim=-1).values[:, -1:]
        logits = logits.where(logits >= threshold, torch.full_like(logits, float("-inf")))
    if top_p < 1.0:
        sorted_logits, sorted_indices = logits.sort(dim=-1, descending=True)
        probs = sorted_logits.softmax(dim=-1)
        # drop tokens whose preceding cumulative mass already reaches top_p
        drop = (probs.cumsum(dim=-1) - probs) >= top_p
        sorted_logits[drop] = float("-inf")
        logits = torch.zeros_like(logits).scatter_(1, sorted_indices, sorted_logits)
    return logits


def _rope_tables(model, total_len: int, device):
    cos = getattr(model, "_rope_cos", None)
    sin = getattr(model, "_rope_sin", None)
    if cos is None or sin is None or cos.shape[0] < total_len:
        cfg = model.config
        cos, sin = precompute_rope_frequencies(cfg.head_dim, max(total_len, cfg.max_seq_len),
                                               theta=getattr(cfg, "rope_theta", 10000.0))
    return cos.to(device), sin.to(device)


def _prefill(model, prompt_tokens, prompt_lens, rows: int, total_len: int):
    """Caches of ``rows`` tokens that hold the prompts, and the logits behind each."""
    cfg, device = model.config, prompt_tokens.device
    batch = prompt_tokens.shape[0]
    dtype = next(model.parameters()).dtype
    caches = [KVCache(batch, rows, cfg.n_kv_heads, cfg.head_dim, dtype, device)
              for _ in range(cfg.n_layers)]
    logits = model(prompt_tokens, kv_caches=caches)
    if prompt_lens is None:
        return caches, logits[:, -1, :]
    last = torch.tensor([n - 1 for n in prompt_lens], device=device)
    cos, sin = _rope_tables(model, total_len, device)
    for c in caches:
        c.set_lengths(prompt_lens)
        c.use_rope_tables(cos, sin)
    return caches, logits[torch.arange(batch, device=device), last]


@torch.no_grad()
def generate(
    model,
    prompt_tokens: torch.Tensor,
    max_new_tokens: int,
    *,
    temperature: float = 1.0,
    top_k: int = 0,
    top_p: float = 1.0,
    eos_token_id: int | None = None,
    prompt_lens: list[int] | None = None,
    eos_check_every: int = 1,
    num_samples: int = 1,
) -> torch.Tensor:
    """Prompt plus generated tokens, ``(batch * num_samples, prompt_len + generated)``
    (a prompt's samples one after the other).

    Without ``prompt_lens`` this is the reference's ``generate``
    (``kempnerforge/model/generate.py:59-124``).  With it, sequence ``b``'s
    prompt is ``prompt_tokens[b, :prompt_lens[b]]``; the result holds, per row,
    the prompt followed directly by that sequence's generated tokens, padded on
    the right with ``eos_token_id`` (or 0) up to the longest row.
    """
    if eos_check_every < 1:
        raise ValueError("eos_check_every must be >= 1")
    if num_samples < 1:
        raise ValueError("num_samples must be >= 1")
    was_training = model.training
    model.eval()
    device = prompt_tokens.device
    batch, prompt_len = prompt_tokens.shape
    cfg = model.config
    total_len = prompt_len + max_new_tokens
    if total_len > cfg.max_seq_len:
        raise ValueError(
            f"prompt ({prompt_len}) + max_new_tokens ({max_new_tokens}) = {total_len} "
            f"exceeds model max_seq_len ({cfg.max_seq_len})"
        )
    if prompt_lens is not None:
        prompt_lens = [int(n) for n in prompt_lens]
        if len(prompt_lens) != batch or min(prompt_lens) < 1 or max(prompt_lens) > prompt_len:
            raise ValueError("prompt_lens needs one length in [1, prompt_len] per sequence")
    caches, next_logits = _prefill(model, prompt_tokens, prompt_lens,
                                   prompt_len if num_samples > 1 else total_len, total_len)
    if num_samples > 1 and max_new_tokens > 0:
        caches = [c.branch(num_samples, max_new_tokens) for c in caches]
    if num_samples > 1:
        next_logits = next_logits.repeat_interleave(num_samples, dim=0)
        prompt_tokens = prompt_tokens.repeat_interleave(num_samples, dim=0)
        batch *= num_samples
        if prompt_lens is not None:
            prompt_lens = [n for n in prompt_lens for _ in range(num_samples)]

    generated = []
    done = torch.zeros(batch, dtype=torch.bool, device=device)
    pending = []  # per step since the last check: all sequences finished?
    for step in range(max_new_tokens):
        token = sample(next_logits, temperature, top_k, top_p)
        generated.append(token)
        if eos_token_id is not None:
            done = done | (token == eos_token_id)
            pending.append(done.all())
            if len(pending) == eos_check_every or step + 1 == max_new_tokens:
                hits = torch.stack(pending).nonzero()
                if hits.numel():
                    # the reference stops right after the step that finished the batch
                    generated = generated[: step + 1 - len(pending) + int(hits[0, 0]) + 1]
                    break
                pending = []
        if step + 1 == max_new_tokens:
            break  # the reference's last forward only feeds a cache that is dropped
        next_logits = model(token.unsqueeze(1), kv_caches=caches)[:, -1, :]

    if was_training:
        model.train()
    gen = torch.stack(generated, dim=1) if generated else prompt_tokens[:, :0]
    if prompt_lens is None:
        return torch.cat([prompt_tokens, gen], dim=1)
    pad = eos_token_id if eos_token_id is not None else 0
    width = max(prompt_lens) + gen.shape[1]
    out = torch.full((batch, width), pad, dtype=prompt_tokens.dtype, device=device)
    for b, n in enumerate(prompt_lens):
        out[b, :n] = prompt_tokens[b, :n]
        out[b, n:n + gen.shape[1]] = gen[b]
    return out


@torch.no_grad()
def beam_generate(
    model,
    prompt_tokens: torch.Tensor,
    max_new_tokens: int,
    *,
    beams: int = 4,
    num_return: int = 1,
    length_penalty: float = 1.0,
    eos_token_id: int | None = None,
    prompt_lens: list[int] | None = None,
    eos_check_every: int = 1,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``num_return`` best continuations of each prompt by beam search: tokens
    ``(batch, num_return, width)``, best first, and their scores ``(batch, num_return)``
    float32.

    A continuation's score is its summed log-probability divided by its length (its
    ``eos_token_id`` counts) to the power of ``length_penalty``.  Each step keeps the
    ``beams`` most likely unfinished continuations of each prompt; one that ends, and is
    among the ``beams`` best of all the step's, is set aside with its score, the best
    ``beams`` of these are kept, and after ``max_new_tokens`` the unfinished ones join
    them.  The search ends early where no unfinished one can reach the worst of
    ``beams`` finished ones any more (read back every ``eos_check_every`` steps).

    The prompts are prefilled once; their keys and values are read once for all beams
    (``kf_attn_branch``), the step's candidates picked in one call (``kf_beam_select``),
    and the beams' own cache rows moved in one launch (``kf_kv_cache_reorder``).
    ``prompt_lens`` as in :func:`generate`.  Rows hold the prompt, directly followed by
    the continuation, padded on the right with ``eos_token_id`` (or 0); a continuation
    that the vocabulary does not give (fewer than ``num_return``) has the score -inf and
    no tokens."""
    batch, prompt_len = prompt_tokens.shape
    if not 1 <= beams <= ops.BEAM_MAX:
        raise ValueError(f"beams must lie in [1, {ops.BEAM_MAX}] (got {beams})")
    if not 1 <= num_return <= beams:
        raise ValueError(f"num_return must lie in [1, beams] (got {num_return})")
    if max_new_tokens < 1 or eos_check_every < 1:
        raise ValueError("max_new_tokens and eos_check_every must be >= 1")
    limit = model.config.max_seq_len
    if prompt_len + max_new_tokens > limit:
        raise ValueError(
            f"prompt ({prompt_len}) + max_new_tokens ({max_new_tokens}) = "
            f"{prompt_len + max_new_tokens} exceeds model max_seq_len ({limit})"
        )
    if prompt_lens is not None:
        prompt_lens = [int(n) for n in prompt_lens]
        if len(prompt_lens) != batch or min(prompt_lens) < 1 or max(prompt_lens) > prompt_len:
            raise ValueError("prompt_lens needs one length in [1, prompt_len] per sequence")
    with _evaluating(model):
        scores, rows, lengths = _beam_search(model, prompt_tokens, prompt_lens, max_new_tokens,
                                             beams, length_penalty, eos_token_id, eos_check_every)
    scores, best = scores.topk(num_return, dim=1)
    rows = rows.gather(1, best[..., None].expand(-1, -1, max_new_tokens)).cpu()
    lengths = lengths.gather(1, best).tolist()
    starts = prompt_lens if prompt_lens is not None else [prompt_len] * batch
    pad = eos_token_id if eos_token_id is not None else 0
    width = max(n + max(row) for n, row in zip(starts, lengths))
    out = torch.full((batch, num_return, width), pad, dtype=prompt_tokens.dtype)
    host_prompt = prompt_tokens.cpu()
    for b, n in enumerate(starts):
        out[b, :, :n] = host_prompt[b, :n]
        for r, k in enumerate(lengths[b]):
            out[b, r, n:n + k] = rows[b, r, :k].to(out.dtype)
    return out.to(prompt_tokens.device), scores


def _beam_search(model, prompt_tokens, prompt_lens, max_new_tokens, beams, length_penalty,
                 eos_token_id, eos_check_every):
    """Scores ``[batch, 2 beams]``, tokens and lengths of the finished continuations and
    of the unfinished ones at the end."""
    device, (batch, prompt_len) = prompt_tokens.device, prompt_tokens.shape
    caches, logits = _prefill(model, prompt_tokens, prompt_lens, prompt_len,
                              prompt_len + max_new_tokens)
    caches = [c.branch(beams, max_new_tokens) for c in caches]
    inf = float("inf")
    scores = torch.zeros(batch, 1, device=device, dtype=torch.float32)
    rows = torch.zeros(batch, 1, max_new_tokens, dtype=torch.int64, device=device)
    rank = torch.arange(2 * beams, device=device)
    done_scores = torch.full((batch, beams), -inf, device=device, dtype=torch.float32)
    done_rows = torch.zeros(batch, beams, max_new_tokens, dtype=torch.int64, device=device)
    done_lens = torch.zeros(batch, beams, dtype=torch.int64, device=device)
    # what an unfinished continuation of summed log-probability s can still reach: s / this
    longest = float(max_new_tokens) ** length_penalty
    for step in range(1, max_new_tokens + 1):
        # (first step: one sequence a prompt)
        best, parents, tokens = ops.beam_select_raw(
            logits.reshape(batch, scores.shape[1], -1), scores, select=2 * beams)
        rows = rows.gather(1, parents.clamp_min(0).long()[..., None].expand(-1, -1, max_new_tokens))
        rows[:, :, step - 1] = tokens.clamp_min(0)
        ends = torch.zeros_like(tokens, dtype=torch.bool)
        if eos_token_id is not None:
            ends = tokens == eos_token_id
            ended = torch.where(ends & (rank < beams), best / float(step) ** length_penalty, -inf)
            done_scores, at = torch.cat([done_scores, ended], 1).topk(beams, dim=1)
            done_rows = torch.cat([done_rows, rows], 1).gather(
                1, at[..., None].expand(-1, -1, max_new_tokens))
            done_lens = torch.cat([done_lens, torch.full_like(tokens, step)], 1).gather(1, at)
        # the best that go on, in order (at most one candidate a beam ends)
        live = torch.sort(ends.to(torch.int8), dim=1, stable=True).indices[:, :beams]
        scores = torch.where(ends, -inf, best).gather(1, live)
        tokens, parents = tokens.gather(1, live), parents.gather(1, live)
        rows = rows.gather(1, live[..., None].expand(-1, -1, max_new_tokens))
        if step == max_new_tokens:
            break
        if eos_token_id is not None and step % eos_check_every == 0:
            reach = scores.amax(1) / (longest if length_penalty >= 0
                                      else float(step + 1) ** length_penalty)
            if bool((reach <= done_scores.amin(1)).all()):
                scores = torch.full_like(scores, -inf)
                break
        if step > 1:
            reorder_branches(caches, parents.contiguous())
        logits = model(tokens.clamp_min(0).view(-1, 1).to(prompt_tokens.dtype),
                       kv_caches=caches)[:, -1, :]
    left = scores / float(step) ** length_penalty
    lens = torch.where(torch.isinf(left), 0, step).to(torch.int64)
    done_lens = torch.where(torch.isinf(done_scores), 0, done_lens)
    return (torch.cat([done_scores, left], 1), torch.cat([done_rows, rows], 1),
            torch.cat([done_lens, lens], 1))



def _tree_levels(tree) -> tuple[list[int], list[int], list[int]]:
    """A draft tree given as its parents, level by level: (parents, rank of each node
    among its siblings, first node of each level with the node count at the end)."""
    parents = [int(p) for p in tree]
    if not 2 <= len(parents) <= ops.TREE_MAX_NODES:
        raise ValueError(f"a draft tree has 2 to {ops.TREE_MAX_NODES} nodes (got {len(parents)})")
    if parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(parents) if i):
        raise ValueError("tree must name the parent of each node, before it; node 0 has -1")
    depth, rank, children = [0], [0], [0] * len(parents)
    for p in parents[1:]:
        depth.append(depth[p] + 1)
        rank.append(children[p])
        children[p] += 1
    if depth != sorted(depth):
        raise ValueError("tree must list its nodes level by level")
    starts = [i for i, d in enumerate(depth) if i == 0 or d > depth[i - 1]]
    return parents, rank, starts + [len(parents)]


class _Stream:
    """One model and its caches over the sequences that are being generated."""

    def __init__(self, model, prompt, prompt_lens, rows: int):
        cfg, device = model.config, prompt.device
        dtype = next(model.parameters()).dtype
        self.model = model
        self.caches = [KVCache(prompt.shape[0], rows, cfg.n_kv_heads, cfg.head_dim, dtype, device)
                       for _ in range(cfg.n_layers)]
        logits = model(prompt, kv_caches=self.caches)
        last = torch.tensor([n - 1 for n in prompt_lens], device=device)
        self.logits = logits[torch.arange(prompt.shape[0], device=device), last]
        cos, sin = _rope_tables(model, min(rows, cfg.max_seq_len), device)
        for c in self.caches:
            c.set_lengths(prompt_lens)
            c.use_rope_tables(cos, sin)

    def __call__(self, tokens):
        return self.model(tokens, kv_caches=self.caches)

    def rewind(self, lens: torch.Tensor, lengths: list[int]) -> None:
        """Fill levels of another stream over the same sequences."""
        for c in self.caches:
            c.lens.copy_(lens)
            c._seq_len, c.ragged = max(lengths), len(set(lengths)) > 1


@contextlib.contextmanager
def _evaluating(*models):
    """The models in eval mode; as they were afterwards, however that comes."""
    modes = [(m, m.training) for m in models]
    for m in models:
        m.eval()
    try:
        yield
    finally:
        for m, was_training in modes:
            m.train(was_training)


@torch.no_grad()
def speculative_generate(
    model,
    draft_model,
    prompt_tokens: torch.Tensor,
    max_new_tokens: int,
    *,
    draft_len: int = 4,
    tree: list[int] | None = None,
    temperature: float = 1.0,
    top_k: int = 0,
    top_p: float = 1.0,
    eos_token_id: int | None = None,
    prompt_lens: list[int] | None = None,
) -> torch.Tensor:
    """:func:`generate` with drafts of ``draft_model``: tokens of the same
    distribution (at temperature 0 the same tokens, up to the rounding of the
    model's logits), several per forward of ``model``.

    Without ``tree`` the draft model samples a chain of ``draft_len`` tokens.  With
    it (the parent of each node, level by level, node 0 the last token with -1) the
    drafts are its most likely tokens after each node, a child per rank.  Each step
    runs the draft model along the chain (or down the levels), scores all drafts in
    one forward of ``model`` (``kf_attn_tree``), verifies them
    (``kf_verify_drafts``) and keeps the accepted path's cache rows
    (``kf_kv_cache_keep``); it reads the accepted tokens back once.  A sequence near
    its ``max_new_tokens`` drafts no deeper than it can use.

    Both models share the vocabulary and follow :func:`generate`'s contract; their dtypes
    may differ (a chain is then drawn and verified in the type that holds both).  Returns
    each prompt followed directly by its tokens, rows padded on the right with
    ``eos_token_id`` (or 0) to the longest; a row ends with its first
    ``eos_token_id`` or after ``max_new_tokens``."""
    batch, prompt_len = prompt_tokens.shape
    if draft_len < 1 or draft_len + 1 > ops.TREE_MAX_NODES:
        raise ValueError(f"draft_len must lie in [1, {ops.TREE_MAX_NODES - 1}] (got {draft_len})")
    if tree is None:
        parents, rank, starts = None, None, list(range(draft_len + 2))
    else:
        parents, rank, starts = _tree_levels(tree)
    limit = min(model.config.max_seq_len, draft_model.config.max_seq_len)
    if prompt_len + max_new_tokens > limit:
        raise ValueError(
            f"prompt ({prompt_len}) + max_new_tokens ({max_new_tokens}) = "
            f"{prompt_len + max_new_tokens} exceeds the models' max_seq_len ({limit})"
        )
    if prompt_lens is None:
        prompt_lens = [prompt_len] * batch
    prompt_lens = [int(n) for n in prompt_lens]
    if len(prompt_lens) != batch or min(prompt_lens) < 1 or max(prompt_lens) > prompt_len:
        raise ValueError("prompt_lens needs one length in [1, prompt_len] per sequence")
    emitted: list[list[int]] = [[] for _ in range(batch)]
    if max_new_tokens > 0:
        with _evaluating(model, draft_model):
            emitted = _emit(model, draft_model, prompt_tokens, prompt_lens, max_new_tokens, parents,
                            rank, starts, temperature, top_k, top_p, eos_token_id)
    pad = eos_token_id if eos_token_id is not None else 0
    width = max(n + len(e) for n, e in zip(prompt_lens, emitted))
    out = torch.full((batch, width), pad, dtype=prompt_tokens.dtype)
    host_prompt = prompt_tokens.cpu()
    for b, (n, e) in enumerate(zip(prompt_lens, emitted)):
        out[b, :n] = host_prompt[b, :n]
        out[b, n:n + len(e)] = torch.tensor(e, dtype=out.dtype)
    return out.to(prompt_tokens.device)


def _emit(model, draft_model, prompt_tokens, prompt_lens, max_new_tokens, parents, rank, starts,
          temperature, top_k, top_p, eos_token_id) -> list[list[int]]:
    """The tokens of :func:`speculative_generate`, a list per sequence; the drafts' tree as
    :func:`_tree_levels` gives it (a chain: no parents)."""
    device = prompt_tokens.device
    batch, prompt_len = prompt_tokens.shape
    chain = parents is None
    # Rows behind the last token for its drafts.  (Positions stay below limit.)
    rows = prompt_len + max_new_tokens + starts[-1]
    target = _Stream(model, prompt_tokens, prompt_lens, rows)
    vocab = target.logits.shape[-1]
    # The draft model's vocabulary before any token of the other's reaches it (token 0 is in
    # both): what lies past its embedding would be read out of range.
    draft_vocab = draft_model(prompt_tokens.new_zeros(1, 1)).shape[-1]
    if vocab != draft_vocab:
        raise ValueError(f"the models' vocabularies differ ({vocab}, {draft_vocab})")
    draft = _Stream(draft_model, prompt_tokens, prompt_lens, rows)

    # A sampled chain's drafts are drawn from the rows that they are verified against, in a
    # type that holds both models' logits.
    dtype = target.logits.dtype
    if chain:
        dtype = torch.promote_types(dtype, draft.logits.dtype)

    def dist(logits):
        """(logits, temperature) of the distribution that is sampled."""
        logits = logits.to(dtype)
        if temperature == 0 or (top_k <= 0 and top_p >= 1.0):
            return logits, temperature
        flat = _filtered((logits / temperature).reshape(-1, vocab), top_k, top_p)
        return flat.view(logits.shape), 1.0

    def uniforms(n):
        """Random numbers for n nodes a sequence, whatever torch's default dtype."""
        return torch.rand(batch, n, device=device, dtype=torch.float32)

    def draw(logits, temp):
        """A token per row, by a verification of no drafts; -1 for a row that is no
        distribution."""
        return ops.verify_drafts_raw(logits[:, None], root, uniforms(1), temperature=temp)[2]

    root = prompt_tokens.new_zeros(batch, 1)
    token = draw(*dist(target.logits))
    emitted = [[t] for t in token.tolist()]
    if min(e[0] for e in emitted) < 0:
        raise RuntimeError("the model's logits are no distribution (NaN, or -inf throughout)")
    lengths = list(prompt_lens)
    if not chain:
        parents = torch.tensor(parents, dtype=torch.int32, device=device)
        rank = torch.tensor(rank, device=device)

    def left(b):
        """How many more tokens sequence b takes."""
        row = emitted[b]
        return 0 if row[-1] == eos_token_id else max_new_tokens - len(row)

    while any(left(b) for b in range(batch)):
        # levels of drafts that each sequence can use (finished ones: no node at all)
        deep = [min(left(b), len(starts) - 1) for b in range(batch)]
        use = [starts[d] for d in deep]
        n, levels = max(use), max(deep)
        counts = torch.tensor(use, dtype=torch.int32, device=device)
        tokens = token.new_zeros(batch, n)
        tokens[:, 0] = token
        tree_parents, draft_logits = None, None
        if chain:
            rowlist = []
            for j in range(1, n):
                logits, temp = dist(draft(tokens[:, j - 1:j])[:, -1])
                rowlist.append(logits)
                # (a draft that is no distribution ends its path in the verification)
                tokens[:, j] = draw(logits, temp).clamp_min(0)
            draft(tokens[:, n - 1:])  # (its key and value, for when all are accepted)
            if temperature > 0 and n > 1:
                draft_logits = torch.stack(rowlist, dim=1)
        else:
            tree_parents = parents[:n]
            for d in range(1, levels):
                lo, hi, end = starts[d - 1], starts[d], starts[d + 1]
                begin_tree(draft.caches, parents[:hi], counts.clamp_max(hi))
                logits = draft(tokens[:, :hi])[:, lo:hi]
                at, want = parents[hi:end].long() - lo, rank[hi:end]
                # (a rank past the vocabulary repeats its last token: refused again)
                best = logits.topk(min(vocab, len(rank)), dim=-1).indices
                tokens[:, hi:end] = best[:, at, want.clamp_max(best.shape[-1] - 1)]
            begin_tree(draft.caches, tree_parents, counts)
            draft(tokens)
        begin_tree(target.caches, tree_parents, counts)
        logits, temp = dist(target(tokens))
        path, kept, token = ops.verify_drafts_raw(
            logits, tokens, uniforms(n), temperature=temp, parents=tree_parents, counts=counts,
            draft_logits=draft_logits)
        accepted = tokens.gather(1, path.clamp_min(0).long())
        # the step's one read-back: per sequence, how many, the path's tokens, the next
        host = torch.cat([kept[:, None].long(), accepted, token[:, None]], dim=1).tolist()
        for b, (k, *row) in enumerate(host):
            if use[b] == 0:
                continue
            if k == 0 or row[-1] < 0:
                raise RuntimeError("the model's logits are no distribution (NaN, or -inf "
                                   "throughout)")
            lengths[b] += k
            for t in row[1:k] + row[-1:]:
                if left(b):
                    emitted[b].append(t)
        keep_path(target.caches, path, kept, lengths)
        if chain:
            draft.rewind(target.caches[0].lens, lengths)
        else:
            keep_path(draft.caches, path, kept, lengths)
        token = token.clamp_min(0)  # (a finished sequence has no next token; any will do)

    return emitted
