"""Speculative decoding over the KV cache: the operators whose speed is measured.

Three operators make one step of it.  ``tree_decode_raw`` appends a tree (or a
chain) of drafted tokens to the cache and attends each of them to the cached
prefix and to its own ancestors; ``verify_drafts_raw`` walks the tree against
the target's logits with given random numbers and draws the token after the
accepted path; ``cache_keep_raw`` moves the accepted path's cache rows together
in every layer.  ``listed`` gives the fixed cases, ``draw`` more of the same
ranges; ``prepare`` makes a case's inputs on the GPU, ``run`` is one pass (in
plain torch, or through the framework's calls where ``own`` is true), ``exact``
the same results in 64 bits, ``work`` what a pass cannot do without.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 500000.0
# share of the drafted tokens that the target's distributions favour (the token
# each row of logits prefers has about this probability)
FAVOURED = 0.75


def _tree(name, B, L, N, Hq, Hkv, D, dtype="bf16", shape="chain", ragged=False, qk_norm=False):
    return {"name": name, "kind": "tree", "B": B, "L": L, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D,
            "dtype": dtype, "shape": shape, "ragged": ragged, "qk_norm": qk_norm}


def _verify(name, B, N, V, dtype="bf16", shape="chain", ragged=False, temperature=1.0,
            drafts=False):
    return {"name": name, "kind": "verify", "B": B, "N": N, "V": V, "dtype": dtype,
            "shape": shape, "ragged": ragged, "temperature": temperature, "drafts": drafts}


def _keep(name, layers, B, L, N, Hkv, D, dtype="bf16", shape="tree2"):
    return {"name": name, "kind": "keep", "layers": layers, "B": B, "L": L, "N": N, "Hkv": Hkv,
            "D": D, "dtype": dtype, "shape": shape}


def listed():
    return [
        # One interactive generation, 8B layer, four drafted tokens in a chain
        # after the last one: the smallest call of a real model.
        _tree("tree_single", 1, 1000, 5, 32, 8, 128),
        # A serving batch with ragged caches, each sequence's 16 nodes a binary
        # tree of its own size.
        _tree("tree_batch", 32, 8192, 16, 32, 8, 128, shape="tree2", ragged=True),
        # Long contexts of a 70B layer with the widest tree: the largest.
        _tree("tree_long", 4, 16384, 64, 64, 8, 128, shape="tree4"),
        # One rank's heads of a 13B layer under 4-way tensor parallelism, five
        # query heads per KV head, an odd number of nodes, in float16.
        _tree("tree_tp4_fp16", 8, 4001, 27, 10, 2, 128, "fp16", "random"),
        # The debug configuration's layer in float32.
        _tree("tree_debug_fp32", 2, 250, 9, 4, 2, 64, "fp32", "tree2"),
        # The next 200 tokens of four conversations of different lengths: a
        # chain as long as a prompt.
        _tree("tree_turn", 4, 2048, 200, 32, 8, 128, ragged=True),
        # Four drafted tokens with the draft model's own distributions, float32
        # logits of a 32000-token vocabulary.
        _verify("verify_single", 1, 5, 32000, "fp32", drafts=True),
        # Trees of 64 nodes for 16 sequences over a large vocabulary: the largest.
        _verify("verify_batch", 16, 64, 131072, "bf16", "tree4", True, 0.7),
        # Greedy decoding: the tokens have to be the most likely ones; a
        # vocabulary of odd size, so that the rows are not aligned.
        _verify("verify_greedy", 8, 27, 50001, "fp16", "tree2", temperature=0.0),
        # The accepted path of one sequence's tree in all layers of an 8B model.
        _keep("keep_single", 32, 1, 4096, 16, 8, 128),
        # The same for a batch whose trees are wide.
        _keep("keep_batch", 32, 16, 1024, 64, 8, 128, shape="tree4"),
    ]


# (Hq, Hkv, D) of the configurations the repository names
HEADS = [(32, 8, 128), (64, 8, 128), (16, 2, 128), (12, 2, 128), (10, 2, 128), (8, 2, 128),
         (12, 12, 64), (4, 2, 64), (16, 16, 64), (32, 8, 64)]
SHAPES = ["chain", "tree2", "tree3", "tree4", "random"]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "verify", "verify", "keep"])
    Hq, Hkv, D = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    shape = rng.choice(SHAPES)
    if kind == "tree":
        N = _log_int(rng, 1, 256 if shape == "chain" else 64)
        L = _log_int(rng, 33, 4096 if dtype == "fp32" else 16384)
        # (queries x keys, bounded by the largest listed case's)
        most = (4 * 64 * 16384 * 64) // (Hq * N * L) if dtype != "fp32" else 33554432 // (Hq * N * L)
        B = rng.randint(1, max(1, min(32, most, 262144 // L)))
        return {"kind": kind, "B": B, "L": L, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D,
                "dtype": dtype, "shape": shape, "ragged": rng.random() < 0.5,
                "qk_norm": rng.random() < 0.25}
    if kind == "verify":
        N, V = _log_int(rng, 1, 64), _log_int(rng, 300, 131072)
        B = rng.randint(1, max(1, min(64, (16 * 64 * 131072) // (N * V * (2 if dtype == "fp32" else 1)))))
        temperature = rng.choice([0.0, 0.6, 1.0, 1.3])
        drafts = shape == "chain" and temperature > 0 and rng.random() < 0.6
        return {"kind": kind, "B": B, "N": N, "V": V, "dtype": dtype, "shape": shape,
                "ragged": rng.random() < 0.5, "temperature": temperature, "drafts": drafts}
    layers, N = rng.choice([2, 16, 32, 40]), _log_int(rng, 2, 64)
    L = _log_int(rng, 100, 4096)
    B = rng.randint(1, max(1, min(16, 16 * 1024 * 8 * 32 * 128 // ((L + N) * Hkv * layers * D))))
    return {"kind": kind, "layers": layers, "B": B, "L": L, "N": N, "Hkv": Hkv, "D": D,
            "dtype": dtype, "shape": shape}


# ------------------------------------------------------------------ layouts
def _parents(case, seed):
    """Parent of each node, -1 for the first: ``[N]`` ints, one shape for the
    batch ("random": ``[B][N]``, every sequence its own)."""
    N, shape = case["N"], case["shape"]
    if shape == "chain":
        return list(range(-1, N - 1))
    if shape == "random":
        g = torch.Generator().manual_seed(7919 * seed + N)
        u = torch.rand(case["B"], N, generator=g).tolist()
        # one of the last few nodes, so that the trees are deeper than wide
        return [[-1] + [i - 1 - int(u[b][i] * min(i, 4)) for i in range(1, N)]
                for b in range(case["B"])]
    w = int(shape[4:])
    return [-1] + [(i - 1) // w for i in range(1, N)]


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _counts(case, seed):
    """Nodes in use per sequence, or None for all of them."""
    if not case.get("ragged"):
        return None
    g = torch.Generator().manual_seed(104729 * seed + case["N"])
    n = [1 + int(float(torch.rand((), generator=g)) * case["N"]) for _ in range(case["B"])]
    n[0] = case["N"]
    return n


def _cache_lengths(case, seed):
    """Tokens cached per sequence before the step: one length, or (ragged) from
    an eighth of it on."""
    B, L = case["B"], case["L"]
    if not case.get("ragged", True):
        return [L] * B
    g = torch.Generator().manual_seed(1000003 * seed + L)
    lens = [L // 8 + int(float(torch.rand((), generator=g)) * (L - L // 8)) for _ in range(B)]
    lens[0] = L
    return lens


def _int32(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ prepare
def _tables(D, rows):
    inv = THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, kind, B, N = DTYPES[case["dtype"]], case["kind"], case["B"], case["N"]
    parents = _parents(case, seed)
    st = {"kind": kind, "parents": None if case["shape"] == "chain" else _int32(parents)}

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    if kind == "tree":
        Hq, Hkv, D, S = case["Hq"], case["Hkv"], case["D"], case["L"] + N
        st["cos"], st["sin"] = _tables(D, S)
        st |= {"q": rand(B, N, Hq, D), "k": rand(B, N, Hkv, D), "v": rand(B, N, Hkv, D),
               "k_cache": rand(B, Hkv, S, D), "v_cache": rand(B, Hkv, S, D), "max_len": S,
               "lens": _int32(_cache_lengths(case, seed)), "counts": _int32(_counts(case, seed)),
               "q_norm": None, "k_norm": None}
        if case["qk_norm"]:
            st["q_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32)
            st["k_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32)
        return st
    if kind == "verify":
        V, T = case["V"], case["temperature"]
        t = T if T > 0 else 1.0
        # a peaked distribution a row: one token holds FAVOURED of the mass, the
        # others' logits are normal
        logits = 3.0 * t * torch.randn(B, N, V, generator=g, device=DEV)
        top = torch.randint(V, (B, N, 1), generator=g, device=DEV)
        rest = math.log(V) + 4.5 + math.log(FAVOURED / (1 - FAVOURED))
        logits.scatter_(2, top, rest * t)
        tokens = torch.randint(V, (B, N), generator=g, device=DEV)
        st["drafts"] = None
        par = torch.tensor(parents, device=DEV).broadcast_to(B, N)
        if case["drafts"] and N > 1:
            # the draft model sees about the same; its tokens are drawn from it
            near = logits[:, :-1] + 0.5 * t * torch.randn(B, N - 1, V, generator=g, device=DEV)
            st["drafts"] = near.to(dt)
            p = torch.softmax(st["drafts"].float() / t, dim=-1)
            u = torch.rand(B, N - 1, 1, generator=g, device=DEV)
            tokens[:, 1:] = (p.cumsum(-1) < u).sum(-1).clamp_max(V - 1)
        elif N > 1:
            # the draft model's most likely tokens after each node, in order:
            # the target's favourite first, or second
            same = par[:, 1:, None] == par[:, None, 1:]
            rank = torch.tril(same, -1).sum(-1)
            fav = top.squeeze(-1).gather(1, par[:, 1:])
            late = torch.rand(B, N, generator=g, device=DEV).gather(1, par[:, 1:]) < 0.2
            hit = rank == late.long()
            tokens[:, 1:] = torch.where(hit, fav, tokens[:, 1:])
        st |= {"logits": logits.to(dt), "tokens": tokens, "temperature": T,
               "uniforms": torch.rand(B, N, generator=g, device=DEV),
               "counts": _int32(_counts(case, seed))}
        return st
    # keep: the path that a verification accepted, nodes of one tree in order
    n_layers, Hkv, D, S = case["layers"], case["Hkv"], case["D"], case["L"] + N
    st["k_all"], st["v_all"] = rand(n_layers, B, Hkv, S, D), rand(n_layers, B, Hkv, S, D)
    st["path"], st["kept"] = (_int32(x) for x in _path(case, seed))
    lens = _cache_lengths(case, seed)
    st["lens"] = [_int32(lens) for _ in range(n_layers)]
    st["lens_out"] = [torch.zeros(B, dtype=torch.int32, device=DEV) for _ in range(n_layers)]
    st["k_caches"], st["v_caches"] = list(st["k_all"]), list(st["v_all"])
    return st


def _path(case, seed):
    """Accepted nodes per sequence (-1 behind the last) and how many they are."""
    B, N = case["B"], case["N"]
    par = _parents(case, seed)
    g = torch.Generator().manual_seed(15485863 * seed + N)
    paths, kept = [], []
    for b in range(B):
        p, path = par[b] if isinstance(par[0], list) else par, [0]
        while True:
            kids = [i for i in range(N) if p[i] == path[-1]]
            if not kids or float(torch.rand((), generator=g)) > 0.85:
                break
            path.append(kids[int(float(torch.rand((), generator=g)) * len(kids))])
        kept.append(len(path))
        paths.append(path + [-1] * (N - len(path)))
    return paths, kept


# ------------------------------------------------------------------ run
def run(state):
    if own:
        return _run_own(state)
    return {"tree": _plain_tree, "verify": _plain_verify, "keep": _plain_keep}[state["kind"]](state)


def _run_own(st):
    from kempnerforge_amd import ops

    if st["kind"] == "tree":
        out = ops.tree_decode_raw(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"],
                                  st["lens"], st["cos"], st["sin"], rope_row_offset=0,
                                  max_len=st["max_len"], parents=st["parents"],
                                  counts=st["counts"], q_norm_weight=st["q_norm"],
                                  k_norm_weight=st["k_norm"])
        return {"out": out, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if st["kind"] == "verify":
        path, kept, token = ops.verify_drafts_raw(
            st["logits"], st["tokens"], st["uniforms"], temperature=st["temperature"],
            parents=st["parents"], counts=st["counts"], draft_logits=st["drafts"])
        return {"path": path, "kept": kept, "token": token}
    ops.cache_keep_raw(st["k_caches"], st["v_caches"], st["lens"], st["path"], st["kept"],
                       lens_out=st["lens_out"])
    return {"k_all": st["k_all"], "v_all": st["v_all"], "lens": st["lens_out"][0],
            "lens_last": st["lens_out"][-1]}


# ------------------------------------------------------------------ the plain forms
def _ancestors(parents, B, N):
    """``[B, N, N]``: 1 where node j is node i or one of its ancestors (the
    inverse of I - P for the parent matrix P, exact: all its entries are 0 or
    1), and the parents as ``[B, N]``."""
    if parents is None:
        parents = torch.arange(-1, N - 1, device=DEV)
    par = parents.long().broadcast_to(B, N)
    eye = torch.eye(N, device=DEV)
    link = (par[:, :, None] == torch.arange(N, device=DEV)).float()
    anc = torch.linalg.solve_triangular(eye - link, eye.expand(B, N, N), upper=False)
    return anc, par


def _rotated(x, cos, sin):
    """RoPE of ``x [B, N, H, D]`` by ``cos, sin [B, N, D/2]``, half-split pairs."""
    half = x.shape[-1] // 2
    c, s = cos[:, :, None], sin[:, :, None]
    x1, x2 = x[..., :half], x[..., half:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def _normed(x, w, eps=1e-5):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _plain_tree(st):
    q, kc, vc = st["q"], st["k_cache"], st["v_cache"]
    B, N, Hq, D = q.shape
    Hkv, S = kc.shape[1], kc.shape[2]
    lens = st["lens"].long()
    anc, _ = _ancestors(st["parents"], B, N)
    node = torch.arange(N, device=DEV)
    used = node < (lens.new_full((B,), N) if st["counts"] is None else st["counts"])[:, None]
    pos = lens[:, None] + anc.sum(-1).long() - 1
    c, s = st["cos"][pos], st["sin"][pos]
    qr = _rotated(_normed(q.float(), st["q_norm"]), c, s)
    kr = _rotated(_normed(st["k"].float(), st["k_norm"]), c, s)
    # rows of unused nodes are written back as they are
    slot = (lens[:, None] + node)[:, None, :, None].expand(B, Hkv, N, D)
    keep = used[:, None, :, None]
    for cache, new in ((kc, kr), (vc, st["v"])):
        rows = torch.where(keep, new.transpose(1, 2).to(cache.dtype), cache.gather(2, slot))
        cache.scatter_(2, slot, rows)
    # prefix keys, then ancestors among the nodes
    key = torch.arange(S, device=DEV) - lens[:, None]
    inside = (key >= 0) & (key < N)
    among = anc.bool().gather(2, key.clamp(0, N - 1)[:, None, :].expand(B, N, S))
    see = (key < 0)[:, None] | (inside[:, None] & among)
    # rows of a KV head: (query head of the group, node)
    qg = qr.view(B, N, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    scores = (qg * D ** -0.5) @ kc.float().transpose(2, 3)
    scores = scores.view(B, Hkv, -1, N, S).masked_fill_(~see[:, None, None], -math.inf)
    scores = (scores - scores.amax(-1, keepdim=True)).exp_()
    scores = scores / scores.sum(-1, keepdim=True)
    o = scores.view(B, Hkv, -1, S) @ vc.float()
    o = o.view(B, Hkv, -1, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)
    out = torch.where(used[:, :, None, None], o, 0.0).to(q.dtype)
    return {"out": out, "k_cache": kc, "v_cache": vc}


def _plain_verify(st):
    logits, tokens, u, T = st["logits"], st["tokens"], st["uniforms"].double(), st["temperature"]
    B, N, V = logits.shape
    anc, par = _ancestors(st["parents"], B, N)
    node = torch.arange(N, device=DEV)
    used = node < (tokens.new_full((B,), N) if st["counts"] is None else st["counts"])[:, None]
    up = par.clamp_min(0)
    # nodes of one parent, and which of them come earlier
    sib = (par[:, :, None] == par[:, None, :]) & (node[:, None] > node)
    if T == 0:
        best = logits.argmax(-1)
        taken = tokens == best.gather(1, up)
    else:
        x = logits.float() / T
        lse = torch.logsumexp(x, dim=-1)
        flat = up * V + tokens
        p = (x.view(B, -1).gather(1, flat) - lse.gather(1, up)).double().exp()
        if st["drafts"] is not None:
            # accepted with probability p / q
            y = st["drafts"].float() / T
            q = (y.gather(2, tokens[:, 1:, None])[..., 0] - torch.logsumexp(y, dim=-1)).double().exp()
            taken = u * torch.nn.functional.pad(q, (1, 0), value=1.0) < p
        else:
            # a sibling is tried on what its refused elder siblings leave; a
            # repeated token has nothing left
            again = sib & (tokens[:, :, None] == tokens[:, None, :])
            first = ~again.any(-1)
            left = 1.0 - (sib.double() @ (p * first)[..., None])[..., 0]
            taken = first & (u * left < p)
    taken &= used
    # the first taken child of each parent, reached when all its ancestors are
    chosen = taken & ~(sib & taken[:, None, :]).any(-1)
    chosen[:, 0] = used[:, 0]
    missing = (anc.bool() & ~chosen[:, None, :]).any(-1)
    reached = ~missing
    kept = reached.sum(-1)
    order = torch.where(reached, node, N).sort(-1).values
    path = torch.where(order < N, order, -1)
    last = path.gather(1, (kept - 1).clamp_min(0)[:, None])
    if T == 0:
        token = best.gather(1, last.clamp_min(0))
    else:
        # the token after the path: from the last node's distribution, less what
        # its refused children took of it, at the point u[:, 0] of its sum
        row = last.clamp_min(0)
        w = logits.gather(1, row[..., None].expand(B, 1, V))[:, 0].double() / T
        w = (w - w.logsumexp(-1, keepdim=True)).exp()
        refused = (par == row) & used & (node > 0)
        if st["drafts"] is not None:
            at = row.clamp_max(N - 2)[..., None].expand(B, 1, V)
            d = st["drafts"].gather(1, at)[:, 0].double() / T
            d = (d - d.logsumexp(-1, keepdim=True)).exp()
            w = torch.where(refused.any(-1, keepdim=True), (w - d).clamp_min(0.0), w)
        else:
            gone = torch.where(refused, tokens, V)
            w = torch.nn.functional.pad(w, (0, 1)).scatter(1, gone, 0.0)[:, :V]
        cum = w.cumsum(-1)
        token = (cum <= u[:, :1] * cum[:, -1:]).sum(-1, keepdim=True).clamp_max(V - 1)
    token = torch.where(kept[:, None] > 0, token, -1)[:, 0]
    return {"path": path.int(), "kept": kept.int(), "token": token}


def _plain_keep(st):
    k, v, lens, path, kept = st["k_all"], st["v_all"], st["lens"][0].long(), st["path"], st["kept"]
    n_layers, B, H, S, D = k.shape
    N = path.shape[1]
    j = torch.arange(N, device=DEV)
    # the rows behind the path are written back as they are
    src = lens[:, None] + torch.where(j < kept[:, None], path.long(), j)
    dst = lens[:, None] + j
    src, dst = (x[None, :, None, :, None].expand(n_layers, B, H, N, D) for x in (src, dst))
    k.scatter_(3, dst, k.gather(3, src))
    v.scatter_(3, dst, v.gather(3, src))
    new = st["lens"][0] + kept
    torch._foreach_copy_(st["lens_out"], [new] * n_layers)
    return {"k_all": k, "v_all": v, "lens": st["lens_out"][0], "lens_last": st["lens_out"][-1]}


# ------------------------------------------------------------------ work
def work(case):
    B, N = case["B"], case["N"]
    el = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "tree":
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        used = _counts(case, 0) or [N] * B
        par = _parents(case, 0)
        # (query, key) pairs: the prefix, and each node's ancestors and itself
        pairs = keys = 0
        for b, (n, L) in enumerate(zip(used, _cache_lengths(case, 0))):
            d = _depths(par[b] if isinstance(par[0], list) else par)
            pairs += n * L + sum(x + 1 for x in d[:n])
            keys += L
        nodes = sum(used)
        # in: cache rows, q, k, v; out: the nodes' cache rows and the output
        return {"bytes": el * (2 * keys * Hkv * D + 2 * nodes * Hq * D + 4 * nodes * Hkv * D),
                "flops": 4 * D * Hq * pairs}
    if case["kind"] == "verify":
        V = case["V"]
        used, par = _counts(case, 0) or [N] * B, _parents(case, 0)
        rows = 0.0
        for b, n in enumerate(used):
            # the rows of the accepted nodes, about FAVOURED of them a level
            deep = max(_depths(par[b] if isinstance(par[0], list) else par)[:n])
            rows += sum(FAVOURED ** i for i in range(deep + 1))
        rows = int(rows * (2 if case["drafts"] and N > 1 else 1))
        return {"bytes": rows * V * el + B * N * 16 + B * 16, "flops": 4 * rows * V}
    par, rows = _path(case, 0)
    moved = sum(sum(i != n for i, n in enumerate(p[:k])) for p, k in zip(par, rows))
    per = 2 * 2 * el * case["layers"] * case["Hkv"] * case["D"]  # K and V, read and written
    return {"bytes": moved * per + 8 * case["layers"] * B + 4 * B * (N + 1), "flops": 0}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"tree": _exact_tree, "verify": _exact_verify,
                "keep": _exact_keep}[case["kind"]](case, seed, st)


def _row_parents(case, seed, b):
    par = _parents(case, seed)
    return par[b] if isinstance(par[0], list) else par


def _exact_tree(case, seed, st):
    B, N, Hq, Hkv, D = (case[x] for x in ("B", "N", "Hq", "Hkv", "D"))
    rep, half = Hq // Hkv, D // 2
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    out = torch.zeros(B, N, Hq, D, dtype=torch.float64, device=DEV)
    used = _counts(case, seed) or [N] * B

    def turn(x, w, at):  # [n, H, D]
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        z = torch.complex(x[..., :half], x[..., half:])
        z = z * torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]
        return torch.cat([z.real, z.imag], -1)

    for b, L in enumerate(_cache_lengths(case, seed)):
        n, par = used[b], _row_parents(case, seed, b)
        depth = _depths(par)[:n]
        at = torch.tensor([L + d for d in depth], device=DEV)
        kc[b, :, L:L + n] = turn(st["k"][b, :n].double(), st["k_norm"], at).transpose(0, 1)
        vc[b, :, L:L + n] = st["v"][b, :n].double().transpose(0, 1)
        q = turn(st["q"][b, :n].double(), st["q_norm"], at) / math.sqrt(D)
        hide = np.ones((n, n), dtype=bool)
        for i in range(n):
            j = i
            while j >= 0:
                hide[i, j] = False
                j = par[j]
        hide = torch.from_numpy(hide).to(DEV)
        for h in range(Hkv):
            qh = q[:, h * rep:(h + 1) * rep].reshape(n * rep, D)
            s = (qh @ kc[b, h, :L + n].T).view(n, rep, L + n)
            s[:, :, L:].masked_fill_(hide[:, None], -math.inf)
            p = torch.softmax(s, -1).view(n * rep, L + n)
            out[b, :n, h * rep:(h + 1) * rep] = (p @ vc[b, h, :L + n]).view(n, rep, D)
    return {"out": out, "k_cache": kc, "v_cache": vc}


def _exact_verify(case, seed, st):
    B, N, V, T = case["B"], case["N"], case["V"], case["temperature"]
    used = _counts(case, seed) or [N] * B
    tok, u = st["tokens"].cpu().numpy(), st["uniforms"].double().cpu().numpy()
    paths, kept, token = np.full((B, N), -1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.int64)

    def dist(x):
        x = x.double().cpu().numpy() / T
        e = np.exp(x - x.max())
        return e / e.sum()

    for b in range(B):
        par, here, path = _row_parents(case, seed, b), 0, [0]
        while True:
            kids = [i for i in range(1, used[b]) if par[i] == here]
            row = st["logits"][b, here]
            if T == 0:
                best = int(np.argmax(row.double().cpu().numpy()))
                step = next((i for i in kids if tok[b, i] == best), None)
            else:
                w, step = dist(row), None
                for i in kids:
                    c = tok[b, i]
                    if st["drafts"] is not None:
                        q = dist(st["drafts"][b, here])
                        if u[b, i] * q[c] < w[c]:
                            step = i
                            break
                        w = np.maximum(w - q, 0.0)
                    else:
                        if w[c] > 0 and u[b, i] * w.sum() < w[c]:
                            step = i
                            break
                        w[c] = 0.0
            if step is None:
                break
            here = step
            path.append(step)
        if T == 0:
            token[b] = best
        else:
            cum = np.cumsum(w)
            token[b] = min(V - 1, int(np.sum(cum <= u[b, 0] * cum[-1])))
        kept[b] = len(path)
        paths[b, :len(path)] = path
    return {"path": paths, "kept": kept, "token": token}


def _exact_keep(case, seed, st):
    k, v = st["k_all"].double(), st["v_all"].double()
    paths, kept = _path(case, seed)
    lens = _cache_lengths(case, seed)
    for b, L in enumerate(lens):
        for j, i in enumerate(paths[b][:kept[b]]):  # ascending: row j was moved already
            k[:, b, :, L + j] = k[:, b, :, L + i]
            v[:, b, :, L + j] = v[:, b, :, L + i]
    new = np.array(lens, np.int32) + np.array(kept, np.int32)
    return {"k_all": k, "v_all": v, "lens": new, "lens_last": new}
