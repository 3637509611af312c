"""Several continuations of one prompt: the operators whose speed is measured.

Beam search, several samples of a prompt, and a batch behind one system prompt keep
a long prefix once for all their sequences.  ``branch_decode_raw`` appends new tokens
to each sequence's own cache and attends them to the prefix of their group and to
their own rows; ``beam_select_raw`` picks the best of all beams' next tokens;
``cache_reorder_raw`` gives every beam the cache rows of the beam that it continues,
in all layers.  ``listed`` gives the fixed cases, ``draw`` more of the same ranges;
``prepare`` makes a case's inputs on the GPU, ``run`` is one pass (in plain torch, or
through the framework's calls where ``own`` is true), ``exact`` the same results in
64 bits, ``work`` what a pass cannot do without.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 500000.0


def _branch(name, G, W, P, L, N, Hq, Hkv, D, dtype="bf16", ragged=False, qk_norm=False):
    """G prefixes of up to P tokens, W sequences behind each with up to L tokens of
    their own and N new ones."""
    return {"name": name, "kind": "branch", "G": G, "W": W, "P": P, "L": L, "N": N, "Hq": Hq,
            "Hkv": Hkv, "D": D, "dtype": dtype, "ragged": ragged, "qk_norm": qk_norm}


def _select(name, G, W, V, K, dtype="bf16", dead=False):
    return {"name": name, "kind": "select", "G": G, "W": W, "V": V, "K": K, "dtype": dtype,
            "dead": dead}


def _reorder(name, layers, G, W, L, Hkv, D, dtype="bf16", ragged=False):
    return {"name": name, "kind": "reorder", "layers": layers, "G": G, "W": W, "L": L, "Hkv": Hkv,
            "D": D, "dtype": dtype, "ragged": ragged}


def listed():
    return [
        # Beam search of four beams over one prompt, an 8B layer: the smallest call of
        # a real model.
        _branch("branch_beams", 1, 4, 1000, 40, 1, 32, 8, 128),
        # Sixteen sampled answers to each of four long prompts, a 70B layer; the
        # answers have different lengths.
        _branch("branch_samples", 4, 16, 8192, 512, 1, 64, 8, 128, ragged=True),
        # A serving batch behind one system prompt, each sequence with its own
        # conversation so far.
        _branch("branch_system", 1, 128, 4096, 2048, 1, 32, 8, 128, ragged=True),
        # The users' first questions behind a system prompt, right-padded to the
        # longest: many new tokens at once, the most operations.
        _branch("branch_questions", 1, 8, 4096, 0, 200, 32, 8, 128, ragged=True),
        # One rank's heads of a 13B layer under 4-way tensor parallelism, five beams,
        # in float16.
        _branch("branch_tp4_fp16", 3, 5, 4001, 77, 1, 10, 2, 128, "fp16"),
        # The debug configuration's layer in float32.
        _branch("branch_debug_fp32", 2, 3, 250, 31, 1, 4, 2, 64, "fp32"),
        # Four beams of one prompt, float32 logits of a 32000-token vocabulary, the
        # best eight (so that four are left where some end).
        _select("select_single", 1, 4, 32000, 8, "fp32"),
        # Eight beams of 32 prompts over a large vocabulary: the largest.
        _select("select_batch", 32, 8, 131072, 16),
        # A vocabulary of odd size, so that the rows are not aligned, and five beams.
        _select("select_odd", 8, 5, 50001, 5, "fp16", dead=True),
        # All layers of an 8B model, four beams that have 100 tokens of their own.
        _reorder("reorder_single", 32, 1, 4, 100, 8, 128),
        # The same for eight beams of eight prompts, later in their answers.
        _reorder("reorder_batch", 32, 8, 8, 256, 8, 128),
    ]


# (Hq, Hkv, D) of the configurations the repository names
HEADS = [(32, 8, 128), (64, 8, 128), (16, 2, 128), (12, 2, 128), (10, 2, 128), (8, 2, 128),
         (12, 12, 64), (4, 2, 64), (16, 16, 64), (32, 8, 64)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["branch", "branch", "branch", "select", "select", "reorder"])
    Hq, Hkv, D = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind == "branch":
        N = 1 if rng.random() < 0.7 else _log_int(rng, 2, 200)
        P = _log_int(rng, 17, 16384)
        L = _log_int(rng, 1, 2048)
        W = _log_int(rng, 1, 128)
        # (queries x keys and cache elements, bounded by the largest listed cases')
        pairs, most = Hq * D * N * W * (P + L + N), 8 * 200 * 32 * 4196 * 128
        elements = 128 * 8 * 1024 * 128
        if dtype == "fp32":
            most, elements = most // 4, elements // 2
        while W > 1 and (pairs > most or W * (Hkv * (L + N) + Hq * N) * D > elements):
            W //= 2
            pairs = Hq * D * N * W * (P + L + N)
        each = D * (Hkv * (P + W * (L + N)) + W * Hq * N)
        G = rng.randint(1, max(1, min(8, most // pairs, elements // each)))
        return {"kind": kind, "G": G, "W": W, "P": P, "L": L, "N": N, "Hq": Hq, "Hkv": Hkv, "D": D,
                "dtype": dtype, "ragged": rng.random() < 0.5, "qk_norm": rng.random() < 0.25}
    if kind == "select":
        W, V = rng.randint(1, 16), _log_int(rng, 300, 131072)
        el = 2 if dtype == "fp32" else 1
        G = _log_int(rng, 1, max(1, min(64, (32 * 8 * 131072) // (W * V * el))))
        return {"kind": kind, "G": G, "W": W, "V": V, "K": W * rng.choice([1, 2, 2]),
                "dtype": dtype, "dead": W > 1 and rng.random() < 0.3}
    layers, L, W = rng.choice([2, 16, 32, 40]), _log_int(rng, 1, 1024), rng.randint(2, 16)
    most = 32 * 64 * 256 * 8 * 128 // (layers * W * L * Hkv * D * (2 if dtype == "fp32" else 1))
    while most < 1 and L > 1:
        L, most = L // 2, 32 * 64 * 256 * 8 * 128 // (layers * W * (L // 2) * Hkv * D * 2)
    G = rng.randint(1, max(1, min(16, most)))
    return {"kind": kind, "layers": layers, "G": G, "W": W, "L": L, "Hkv": Hkv, "D": D,
            "dtype": dtype, "ragged": rng.random() < 0.3}


# ------------------------------------------------------------------ layouts
def _some(seed, salt, n, lo, hi):
    """n whole numbers from lo to hi, the first of them hi."""
    g = torch.Generator().manual_seed(1000003 * seed + salt)
    v = [lo + int(float(torch.rand((), generator=g)) * (hi + 1 - lo)) for _ in range(n)]
    return [hi] + v[1:]


def _lengths(case, seed):
    """Prefix tokens per group, own tokens and new tokens per sequence."""
    G, B, P, L, N = case["G"], case["G"] * case["W"], case["P"], case["L"], case["N"]
    if not case["ragged"]:
        return [P] * G, [L] * B, [N] * B
    return (_some(seed, 1, G, P // 4, P), _some(seed, 2, B, L // 8, L),
            _some(seed, 3, B, 1, N))


def _own_lengths(case, seed):
    B, L = case["G"] * case["W"], case["L"]
    return _some(seed, 4, B, L // 2, L) if case["ragged"] else [L] * B


def _parents(case, seed):
    """The beam of its group that each beam continues: the better beams more often."""
    G, W = case["G"], case["W"]
    g = torch.Generator().manual_seed(15485863 * seed + W)
    u = torch.rand(G, W, generator=g).square() * W
    return u.long().clamp_max(W - 1).tolist()


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------ prepare
def _tables(D, rows):
    inv = THETA ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, kind, G, W = DTYPES[case["dtype"]], case["kind"], case["G"], case["W"]
    B = G * W

    def rand(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)

    if kind == "branch":
        N, P, S = case["N"], case["P"], case["L"] + case["N"]
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        prefix, lens, counts = _lengths(case, seed)
        st = {"kind": kind, "q": rand(B, N, Hq, D), "k": rand(B, N, Hkv, D),
              "v": rand(B, N, Hkv, D), "k_prefix": rand(G, Hkv, P, D),
              "v_prefix": rand(G, Hkv, P, D), "k_cache": rand(B, Hkv, S, D),
              "v_cache": rand(B, Hkv, S, D), "prefix_lens": _int32(prefix), "lens": _int32(lens),
              "counts": _int32(counts) if case["ragged"] else None, "max_prefix": P,
              "max_len": S, "q_norm": None, "k_norm": None}
        st["cos"], st["sin"] = _tables(D, P + S)
        if case["qk_norm"]:
            st["q_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32)
            st["k_norm"] = 1 + 0.1 * rand(D, dtype=torch.float32)
        return st
    if kind == "select":
        V = case["V"]
        # a few tokens of each beam hold most of the mass
        logits = 2.5 * torch.randn(B, V, generator=g, device=DEV)
        top = torch.randint(V, (B, 12), generator=g, device=DEV)
        boost = math.log(V) + 3.0 + 2.0 * torch.randn(B, 12, generator=g, device=DEV)
        logits.scatter_(1, top, boost)
        scores = -12.0 * torch.rand(G, W, generator=g, device=DEV)
        scores = scores.sort(dim=1, descending=True).values
        if case["dead"]:
            scores[:, -1] = -math.inf
        return {"kind": kind, "logits": logits.view(G, W, V).to(dt), "scores": scores,
                "K": case["K"]}
    n_layers, Hkv, D, L = case["layers"], case["Hkv"], case["D"], case["L"]
    k, v = rand(n_layers, B, Hkv, L + 1, D), rand(n_layers, B, Hkv, L + 1, D)
    return {"kind": kind, "k_all": k, "v_all": v, "k_caches": list(k), "v_caches": list(v),
            "lens": _int32(_own_lengths(case, seed)), "parents": _int32(_parents(case, seed))}


# ------------------------------------------------------------------ run
def run(state):
    if own:
        return _run_own(state)
    return {"branch": _plain_branch, "select": _plain_select,
            "reorder": _plain_reorder}[state["kind"]](state)


def _run_own(st):
    from kempnerforge_amd import ops

    if st["kind"] == "branch":
        out = ops.branch_decode_raw(
            st["q"], st["k"], st["v"], st["k_prefix"], st["v_prefix"], st["prefix_lens"],
            st["k_cache"], st["v_cache"], st["lens"], st["cos"], st["sin"], rope_row_offset=0,
            max_prefix=st["max_prefix"], max_len=st["max_len"], counts=st["counts"],
            q_norm_weight=st["q_norm"], k_norm_weight=st["k_norm"])
        return {"out": out, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    if st["kind"] == "select":
        scores, parents, tokens = ops.beam_select_raw(st["logits"], st["scores"], select=st["K"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    ops.cache_reorder_raw(st["k_caches"], st["v_caches"], st["lens"], st["parents"])
    return {"k_all": st["k_all"], "v_all": st["v_all"]}


# ------------------------------------------------------------------ the plain forms
def _rotated(x, cos, sin):
    """RoPE of ``x [B, N, H, D]`` by ``cos, sin [B, N, D/2]``, half-split pairs."""
    half = x.shape[-1] // 2
    c, s = cos[:, :, None], sin[:, :, None]
    x1, x2 = x[..., :half], x[..., half:]
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1)


def _normed(x, w, eps=1e-5):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _plain_branch(st):
    q, kc, vc, kp, vp = st["q"], st["k_cache"], st["v_cache"], st["k_prefix"], st["v_prefix"]
    B, N, Hq, D = q.shape
    G, Hkv, P, S = kp.shape[0], kp.shape[1], kp.shape[2], kc.shape[2]
    W, rep = B // G, Hq // Hkv
    lens, plens = st["lens"].long(), st["prefix_lens"].long()
    node = torch.arange(N, device=DEV)
    used = node < (lens.new_full((B,), N) if st["counts"] is None else st["counts"])[:, None]
    pos = plens.repeat_interleave(W)[:, None] + lens[:, None] + node
    c, s = st["cos"][pos], st["sin"][pos]
    qr = _rotated(_normed(q.float(), st["q_norm"]), c, s) * D ** -0.5
    kr = _rotated(_normed(st["k"].float(), st["k_norm"]), c, s)
    # rows of unused tokens are written back as they are
    row = (lens[:, None] + node).clamp_max(S - 1)
    slot = row[:, None, :, None].expand(B, Hkv, N, D)
    keep = used[:, None, :, None]
    for cache, new in ((kc, kr), (vc, st["v"])):
        rows = torch.where(keep, new.transpose(1, 2).to(cache.dtype), cache.gather(2, slot))
        cache.scatter_(2, slot, rows)
    # the prefix: all rows of a group's KV head against its keys at once
    qh = qr.view(B, N, Hkv, rep, D).transpose(1, 2)  # [B, Hkv, N, rep, D]
    qg = qh.view(G, W, Hkv, N, rep, D).transpose(1, 2).reshape(G, Hkv, W * N * rep, D)
    far = qg @ kp.float().transpose(2, 3)
    hide = torch.arange(P, device=DEV) >= plens[:, None]
    far.masked_fill_(hide[:, None, None], -math.inf)
    # a sequence's own rows: token i sees those up to its own
    near = qh.reshape(B, Hkv, N * rep, D) @ kc.float().transpose(2, 3)
    late = torch.arange(S, device=DEV) > lens[:, None, None] + node[:, None]  # [B, N, S]
    near.view(B, Hkv, N, rep, S).masked_fill_(late[:, None, :, None], -math.inf)
    near = near.view(G, W, Hkv, N * rep, S).transpose(1, 2).reshape(G, Hkv, W * N * rep, S)
    top = torch.maximum(far.amax(-1, keepdim=True), near.amax(-1, keepdim=True))
    far, near = (far - top).exp_(), (near - top).exp_()
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    o = far @ vp.float()
    near = near.view(G, Hkv, W, N * rep, S).transpose(1, 2).reshape(B, Hkv, N * rep, S)
    # (rows behind a sequence's last weigh nothing)
    o2 = near @ vc.float()
    o2 = o2.view(G, W, Hkv, N * rep, D).transpose(1, 2).reshape(G, Hkv, W * N * rep, D)
    o = (o + o2) / total
    o = o.view(G, Hkv, W, N, rep, D).permute(0, 2, 3, 1, 4, 5).reshape(B, N, Hq, D)
    out = torch.where(used[:, :, None, None], o, 0.0).to(q.dtype)
    return {"out": out, "k_cache": kc, "v_cache": vc}


def _plain_select(st):
    logits, scores, K = st["logits"], st["scores"], st["K"]
    G, W, V = logits.shape
    # in 64 bits: two candidates may lie next to each other
    x = logits.double()
    total = scores.double()[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))
    total = total.view(G, W * V)
    # equals go to the lowest place: all above the K-th largest, then the first of
    # its equals
    edge = total.topk(K, dim=-1).values[:, -1:]
    above, equal = total > edge, total == edge
    left = K - above.sum(-1, keepdim=True)
    chosen = above | (equal & (equal.cumsum(-1) <= left))
    place = torch.arange(W * V, device=DEV)
    at = torch.where(chosen, place, W * V).topk(K, dim=-1, largest=False).values.sort(-1).values
    best, order = total.gather(1, at).sort(dim=-1, descending=True, stable=True)
    at = at.gather(1, order)
    return {"scores": best.float(), "parents": (at // V).int(), "tokens": at % V}


def _plain_reorder(st):
    k, v, lens, parents = st["k_all"], st["v_all"], st["lens"].long(), st["parents"].long()
    n_layers, B, H, S, D = k.shape
    G, W = parents.shape
    src = (torch.arange(G, device=DEV)[:, None] * W + parents).view(-1)
    moved = torch.arange(S, device=DEV) < lens[src][:, None]
    for x in (k, v):
        x.copy_(torch.where(moved[None, :, None, :, None], x.index_select(1, src), x))
    return {"k_all": k, "v_all": v}


# ------------------------------------------------------------------ work
def work(case):
    el = 4 if case["dtype"] == "fp32" else 2
    G, W = case["G"], case["W"]
    if case["kind"] == "branch":
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        prefix, lens, counts = _lengths(case, 0)
        # (query, key) pairs; keys of the prefixes (once each) and of the sequences
        pairs = sum(n * (prefix[b // W] + L) + n * (n + 1) // 2
                    for b, (L, n) in enumerate(zip(lens, counts)))
        keys, new = sum(prefix) + sum(lens), sum(counts)
        # in: cache rows, q, k, v; out: the new cache rows and the output
        return {"bytes": el * (2 * keys * Hkv * D + 2 * new * Hq * D + 4 * new * Hkv * D),
                "flops": 4 * D * Hq * pairs}
    if case["kind"] == "select":
        rows = G * (W - 1 if case["dead"] else W)
        return {"bytes": rows * case["V"] * el + G * (4 * W + 16 * case["K"]),
                "flops": 4 * rows * case["V"]}
    lens, rows = _own_lengths(case, 0), 0
    for g, parents in enumerate(_parents(case, 0)):
        moves = [(p, w) for w, p in enumerate(parents) if p != w]
        rows += sum(lens[g * W + p] for p, _ in moves)           # written
        rows += sum(lens[g * W + p] for p in {p for p, _ in moves})  # read
    return {"bytes": max(1, 2 * el * case["layers"] * case["Hkv"] * case["D"] * rows) + 8 * G * W,
            "flops": 0}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"branch": _exact_branch, "select": _exact_select,
                "reorder": _exact_reorder}[case["kind"]](case, seed, st)


def _exact_branch(case, seed, st):
    G, W, N, Hq, Hkv, D = (case[x] for x in ("G", "W", "N", "Hq", "Hkv", "D"))
    rep, half = Hq // Hkv, D // 2
    prefix, lens, counts = _lengths(case, seed)
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    out = torch.zeros(G * W, N, Hq, D, dtype=torch.float64, device=DEV)

    def turn(x, w, at):  # [n, H, D]
        if w is not None:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        z = torch.complex(x[..., :half], x[..., half:])
        z = z * torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]
        return torch.cat([z.real, z.imag], -1)

    for g in range(G):
        kp, vp = (st[x][g, :, :prefix[g]].double() for x in ("k_prefix", "v_prefix"))
        for b in range(g * W, (g + 1) * W):
            n, L = counts[b], lens[b]
            at = torch.arange(prefix[g] + L, prefix[g] + L + n, device=DEV)
            kc[b, :, L:L + n] = turn(st["k"][b, :n].double(), st["k_norm"], at).transpose(0, 1)
            vc[b, :, L:L + n] = st["v"][b, :n].double().transpose(0, 1)
            q = turn(st["q"][b, :n].double(), st["q_norm"], at) / math.sqrt(D)
            hide = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
            for h in range(Hkv):
                keys = torch.cat([kp[h], kc[b, h, :L + n]])
                s = (q[:, h * rep:(h + 1) * rep].reshape(n * rep, D) @ keys.T).view(n, rep, -1)
                s[:, :, prefix[g] + L:].masked_fill_(hide[:, None], -math.inf)
                p = torch.softmax(s, -1).view(n * rep, -1)
                o = p @ torch.cat([vp[h], vc[b, h, :L + n]])
                out[b, :n, h * rep:(h + 1) * rep] = o.view(n, rep, D)
    return {"out": out, "k_cache": kc, "v_cache": vc}


def _exact_select(case, seed, st):
    G, K, V = case["G"], case["K"], case["V"]
    scores = np.zeros((G, K))
    parents, tokens = np.zeros((G, K), np.int32), np.zeros((G, K), np.int64)
    start = st["scores"].double().cpu().numpy()
    for g in range(G):
        x = st["logits"][g].double().cpu().numpy()
        top = x.max(axis=1, keepdims=True)
        total = x - top - np.log(np.exp(x - top).sum(axis=1, keepdims=True)) + start[g][:, None]
        flat = total.reshape(-1)
        edge = np.partition(flat, -K)[-K]
        some = np.flatnonzero(flat >= edge)
        some = some[np.argsort(-flat[some], kind="stable")][:K]
        scores[g], parents[g], tokens[g] = flat[some], some // V, some % V
    return {"scores": scores, "parents": parents, "tokens": tokens}


def _exact_reorder(case, seed, st):
    k, v = st["k_all"].double(), st["v_all"].double()
    W, lens, was = case["W"], _own_lengths(case, seed), (k.clone(), v.clone())
    for g, parents in enumerate(_parents(case, seed)):
        for w, p in enumerate(parents):
            n = lens[g * W + p]
            for x, old in zip((k, v), was):
                x[:, g * W + w, :, :n] = old[:, g * W + p, :, :n]
    return {"k_all": k, "v_all": v}
