"""What the speed of the cache and position operators is measured on.

``listed()`` holds the fixed cases, ``draw(rng)`` gives another one of the same
ranges.  ``prepare`` makes what a program has in hand before the call (inputs on
the GPU), ``run`` is one pass: the operators in their plain form, or with
``own`` the calls a program makes of the framework.  ``work`` gives the bytes
and operations a pass cannot do without, ``exact`` the same outputs from the
definition in float64.

Case kinds
  tree      attention of drafted tokens, which form a tree, over a KV cache that
            holds their own keys behind every sequence's prefix
  weights   attention that also adds up, per key, the softmax weight it was
            given: decode steps over a cache, and whole prompts
  evict     a cache cut down to the keys of the largest accumulated weight
  rotary    rotation of q and k by positions of one or several axes, alone or
            with its gradients
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _tree(name, dtype, batch, heads, kv_heads, tokens, capacity, head_dim, shortest, form):
    """``form``: "shared" (one tree of parents for the batch), "parents" (a tree
    for every sequence, of fewer tokens than the batch's widest), "mask" (a
    boolean matrix for every sequence)."""
    c = dict(kind="tree", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, tokens=tokens,
             capacity=capacity, head_dim=head_dim, shortest=shortest, form=form)
    return dict(c, name=name) if name else c


def _weights(name, dtype, batch, heads, kv_heads, q_len, capacity, head_dim, shortest, mask):
    """``mask``: "lengths" (a cache of sequences of different fill), "causal" (a
    prompt, ``q_len == capacity``) or "none"."""
    c = dict(kind="weights", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, q_len=q_len,
             capacity=capacity, head_dim=head_dim, shortest=shortest, mask=mask)
    return dict(c, name=name) if name else c


def _evict(name, dtype, batch, kv_heads, capacity, head_dim, shortest, keep, sinks, recent):
    c = dict(kind="evict", dtype=dtype, batch=batch, kv_heads=kv_heads, capacity=capacity, head_dim=head_dim,
             shortest=shortest, keep=keep, sinks=sinks, recent=recent)
    return dict(c, name=name) if name else c


def _rotary(name, dtype, batch, length, heads, kv_heads, head_dim, sections, far, interleaved, shared, backward):
    """``sections``: rotated features of every axis, "32+48+48"; ``far``: the
    largest position."""
    c = dict(kind="rotary", dtype=dtype, batch=batch, length=length, heads=heads, kv_heads=kv_heads,
             head_dim=head_dim, sections=sections, far=far, interleaved=interleaved, shared=shared,
             backward=backward)
    return dict(c, name=name) if name else c


def listed():
    return [
        # A small float32 model (the library's default dtype) drafting five tokens: launch and latency bound.
        _tree("f32_tree_small", "f32", 2, 4, 4, 5, 512, 64, 200, "shared"),
        # One chat with a fixed draft tree against a cache of middle size.
        _tree("bf16_tree_single", "bf16", 1, 32, 8, 26, 4096, 128, 4070, "shared"),
        # A serving batch, caches of different fill, every sequence with a draft tree of its own size.
        _tree("bf16_tree_ragged", "bf16", 16, 32, 8, 16, 8192, 128, 512, "parents"),
        # Wide drafts, whose masks the drafting model hands over.
        _tree("f16_tree_wide", "f16", 8, 32, 8, 61, 4096, 128, 1500, "mask"),
        # One token of one chat, whose cache will be cut down by the weights its keys were given.
        _weights("bf16_weights_single", "bf16", 1, 32, 8, 1, 4096, 128, 4096, "lengths"),
        # One token for every sequence of a serving batch: the largest cache.
        _weights("bf16_weights_ragged", "bf16", 32, 32, 8, 1, 8192, 128, 512, "lengths"),
        # The prompt that filled such a cache.
        _weights("bf16_weights_prompt", "bf16", 1, 16, 4, 4096, 4096, 128, 4096, "causal"),
        # One chat's cache cut to half.
        _evict("bf16_evict_single", "bf16", 1, 8, 4096, 128, 4096, 2048, 4, 32),
        # A serving batch's caches of different fill cut to half their capacity.
        _evict("bf16_evict_ragged", "bf16", 16, 8, 8192, 128, 1000, 4096, 4, 256),
        # One new token for every sequence of a serving batch, far into its text.
        _rotary("bf16_rotary_step", "bf16", 32, 1, 32, 8, 128, "128", 1000000, True, False, False),
        # A video's patches: time, height and width.
        _rotary("bf16_rotary_video", "bf16", 1, 12288, 16, 16, 128, "32+48+48", 64, True, False, False),
        # A training step on text with images, one spectrum of frequencies dealt to the three axes.
        _rotary("bf16_rotary_train", "bf16", 2, 4096, 16, 4, 128, "32+48+48", 4096, False, True, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    # float32 products run at about a sixteenth of the 16-bit rate
    return max(w["bytes"], w["flops"] * (16 if case["dtype"] == "f32" else 1) / 300)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        if _cost(case) <= most:
            return case


def _draw(rng):
    kind = rng.choice(("tree", "tree", "weights", "prompt", "evict", "rotary", "rotary"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    head_dim = rng.choice((64, 64, 80, 96, 128, 128, 128, 256))
    if dtype == "f32" and kind in ("tree", "weights", "prompt") and head_dim in (80, 96):
        head_dim = 64
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 8))
    batch = _log_int(rng, 1, 32)
    if kind == "tree":
        tokens = _log_int(rng, 1, 128)
        capacity = _log_int(rng, 256, 32768)
        shortest = rng.randint(0, capacity - tokens)
        return _tree(None, dtype, batch, heads, kv_heads, tokens, capacity, head_dim, shortest,
                     rng.choice(("shared", "parents", "mask")))
    if kind == "weights":
        capacity = _log_int(rng, 256, 32768)
        return _weights(None, dtype, batch, heads, kv_heads, rng.choice((1, 1, 1, 2, 5, 8)), capacity, head_dim,
                        rng.randint(1, capacity), "lengths")
    if kind == "prompt":
        length = _log_int(rng, 64, 4096)
        mask = rng.choice(("causal", "causal", "lengths", "none"))
        return _weights(None, dtype, min(batch, 4), heads, kv_heads, length, length, head_dim,
                        rng.randint(1, length) if mask == "lengths" else length, mask)
    if kind == "evict":
        capacity = _log_int(rng, 64, 32768)
        keep = max(1, int(capacity * rng.uniform(0.1, 0.9)))
        sinks = min(rng.choice((0, 1, 4)), keep)
        recent = min(rng.choice((0, 16, 33, 256)), keep - sinks)
        return _evict(None, dtype, batch, kv_heads, capacity, head_dim, rng.randint(1, capacity), keep, sinks, recent)
    axes = rng.choice((1, 2, 3))
    pairs = [max(1, head_dim // (2 * axes) - rng.choice((0, 0, 0, 3))) for _ in range(axes)]
    far = _log_int(rng, 64, 1000000)
    return _rotary(None, dtype, min(batch, 8), _log_int(rng, 1, 16384), heads, kv_heads, head_dim,
                   "+".join(str(2 * p) for p in pairs), far, rng.random() < 0.5, rng.random() < 0.5,
                   rng.random() < 0.5)


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------

def _spread(shortest, longest, batch):
    """Lengths spread evenly from ``longest`` down to ``shortest``."""
    if batch == 1:
        return [longest]
    return [round(longest - (longest - shortest) * i / (batch - 1)) for i in range(batch)]


def _lengths(gen, shortest, longest, batch):
    """Those lengths in a random order."""
    L = torch.tensor(_spread(shortest, longest, batch), dtype=torch.int32).cuda()
    return L[torch.randperm(batch, generator=gen, device="cuda")]


def _sizes(case):
    """Drafted tokens of every sequence of a "parents" case."""
    return _spread(max(1, case["tokens"] // 2), case["tokens"], case["batch"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32)

    s = {"case": case}
    kind, B, D = case["kind"], case["batch"], case["head_dim"]
    if kind == "rotary":
        T, A = case["length"], len(case["sections"].split("+"))
        s["q"], s["k"] = normal(B, T, case["heads"], D), normal(B, T, case["kv_heads"], D)
        s["sections"] = tuple(int(x) for x in case["sections"].split("+"))
        s["table"] = _table(case)
        s["positions"] = (uniform(B, T, A) * (case["far"] + 1)).to(torch.int32)
        if case["backward"]:
            s["dq"], s["dk"] = normal(B, T, case["heads"], D), normal(B, T, case["kv_heads"], D)
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    S, Hkv = case["capacity"], case["kv_heads"]
    s["k"], s["v"] = normal(B, S, Hkv, D), normal(B, S, Hkv, D)
    s["scale"] = 1.0 / math.sqrt(D)
    if kind == "evict":
        s["lengths"] = _lengths(gen, case["shortest"], S, B)
        # a few keys carry most of the weight; some were never looked at (equal zeros)
        w = -torch.log(uniform(B, Hkv, S).clamp_min(1e-6)) ** 2
        s["weights"] = torch.where(uniform(B, Hkv, S) < 0.05, torch.zeros_like(w), -w)
        return s
    if kind == "weights":
        s["q"] = normal(B, case["q_len"], case["heads"], D)
        s["weights"] = uniform(B, Hkv, S)
        if case["mask"] == "lengths":
            s["lengths"] = _lengths(gen, case["shortest"], S, B)
        return s
    T = case["tokens"]
    s["q"] = normal(B, T, case["heads"], D)
    s["lengths"] = _lengths(gen, case["shortest"], S - T, B)  # keys of the prefix
    lead = () if case["form"] == "shared" else (B,)
    # token t's parent: one of the eight tokens before it, or the prefix (-1)
    t = torch.arange(T, device="cuda").expand(lead + (T,))
    parents = t - 1 - (uniform(*lead, T) * (t + 1).clamp_max(8)).long()
    if case["form"] == "parents":
        sizes = torch.tensor(_sizes(case), device="cuda")[:, None]
        parents = torch.where(t < sizes, parents, torch.full_like(parents, -2))  # -2: no token here
    s["parents"] = parents.to(torch.int32)
    if case["form"] == "mask":
        s["tree_mask"] = _ancestors(s.pop("parents"))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _ancestors(parents):
    """Boolean ``[..., T, T]``: whether column j is token i or an ancestor of it,
    by squaring the relation "is, or is the parent of"."""
    T = parents.shape[-1]
    t = torch.arange(T, device=parents.device)
    here = parents >= -1
    seen = ((parents[..., None] == t) | ((t[:, None] == t) & here[..., None])).float()
    for _ in range(max(1, (T - 1).bit_length())):
        seen = (torch.matmul(seen, seen) > 0).float()
    return seen > 0


def _attend(q, k, v, scale, keep):
    """float32 attention: ``q [B, T, Hq, D]``, ``k, v [B, S, Hkv, D]``, ``keep``
    boolean, broadcast to ``[B, Hkv, G, T, S]`` -> output and weights.  Rows
    that keep nothing give zeros."""
    B, T, Hq, D = q.shape
    S, Hkv = k.shape[1:3]
    # a KV head's query heads share one product
    rows = q.float().reshape(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    keys, values = (x.float().permute(0, 2, 1, 3) for x in (k, v))
    s = torch.matmul(rows, keys.transpose(-1, -2)).reshape(B, Hkv, Hq // Hkv, T, S) * scale
    if keep is not None:
        s = torch.where(keep, s, torch.full((), float("-inf"), device=s.device))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(p.reshape(B, Hkv, -1, S), values).reshape(B, Hkv, Hq // Hkv, T, D)
    return out.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(q.dtype), p


def _plain_tree(s):
    S = s["k"].shape[1]
    seen = s["tree_mask"] if "tree_mask" in s else _ancestors(s["parents"])
    T = seen.shape[-1]
    L = s["lengths"][:, None, None].long()
    j = torch.arange(S, device="cuda")[None, None, :] - L  # drafted token of every slot
    B = L.shape[0]
    rows = seen.expand(B, T, T)
    tail = torch.gather(rows, 2, j.clamp(0, T - 1).expand(B, T, S)) & (j >= 0) & (j < T)
    prefix = j < 0
    if "parents" in s:  # a slot without a token keeps nothing
        prefix = prefix & (s["parents"].expand(B, T)[..., None] >= -1)
    return _attend(s["q"], s["k"], s["v"], s["scale"], (tail | prefix)[:, None, None])[0]


def _plain_weights(s):
    case, S = s["case"], s["k"].shape[1]
    j = torch.arange(S, device="cuda")
    keep = None
    if case["mask"] == "lengths":
        keep = (j < s["lengths"][:, None])[:, None, None, None, :]
    elif case["mask"] == "causal":
        keep = j <= j[:, None]
    out, p = _attend(s["q"], s["k"], s["v"], s["scale"], keep)
    return {"out": out, "weights": s["weights"] + p.sum((2, 3))}


def _plain_evict(s):
    case, w = s["case"], s["weights"]
    keep, S = case["keep"], w.shape[-1]
    j = torch.arange(S, device="cuda")
    L = s["lengths"][:, None, None]
    rank = torch.where((j < case["sinks"]) | (j >= L - case["recent"]), torch.full_like(w, float("inf")), w)
    rank = torch.where(j < L, rank, torch.full_like(w, float("-inf")))
    index = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    index = torch.sort(torch.where(index < L, index, S), dim=-1).values  # in order, free places last
    free = index == S
    at = index.clamp_max(S - 1).permute(0, 2, 1)[..., None]
    k, v = (torch.gather(x, 1, at.expand(-1, -1, -1, x.shape[-1])) for x in (s["k"], s["v"]))
    gone = free.permute(0, 2, 1)[..., None]
    return {"k": torch.where(gone, torch.zeros_like(k), k), "v": torch.where(gone, torch.zeros_like(v), v),
            "weights": torch.where(free, torch.zeros_like(w[..., :1]), torch.gather(w, 2, index.clamp_max(S - 1))),
            "lengths": s["lengths"].clamp_max(keep), "index": torch.where(free, -1, index).to(torch.int32)}


def _table(case):
    """What a program that rotates by itself keeps: axis and frequency
    (float64) of every rotated pair, its first and its second feature."""
    sections = [int(x) for x in case["sections"].split("+")]
    width, at = sum(sections), 0
    axis, power, first, second = [], [], [], []
    for a, d in enumerate(sections):
        for i in range(d // 2):
            axis.append(a)
            power.append((at // 2 + i) * 2 / width if case["shared"] else i * 2 / d)
        at += d
    at = 0
    for d in ((width,) if case["shared"] else sections):
        for i in range(d // 2):
            first.append(at + (2 * i if case["interleaved"] else i))
            second.append(at + (2 * i + 1 if case["interleaved"] else i + d // 2))
        at += d
    frequency = 10000.0 ** -torch.tensor(power, dtype=torch.float64)
    return tuple(x.cuda() for x in (torch.tensor(axis), frequency, torch.tensor(first), torch.tensor(second)))


def _rotate(x, cos, sin, first, second):
    y = x.float().clone()
    x0, x1 = y[..., first], y[..., second]
    y[..., first] = x0 * cos - x1 * sin
    y[..., second] = x1 * cos + x0 * sin
    return y.to(x.dtype)


def _plain_rotary(s):
    case = s["case"]
    axis, frequency, *pairs = s["table"]
    angles = (s["positions"].double()[..., axis] * frequency)[:, :, None]
    cos, sin = torch.cos(angles).float(), torch.sin(angles).float()
    out = {n: _rotate(s[n].detach(), cos, sin, *pairs) for n in ("q", "k")}
    if case["backward"]:  # the transposed rotation, by the opposite angle
        out.update({n: _rotate(s[n], cos, -sin, *pairs) for n in ("dq", "dk")})
    return out


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"tree": _plain_tree, "weights": _plain_weights, "evict": _plain_evict, "rotary": _plain_rotary}[kind](s)
    return _own(s)


def _own(s):
    from probjax_amd import attention, masks

    case = s["case"]
    kind = case["kind"]
    if kind == "tree":
        return attention.tree_attention(s["q"], s["k"], s["v"], parents=s.get("parents"),
                                        tree_mask=s.get("tree_mask"), kv_lengths=s["lengths"], sm_scale=s["scale"])
    if kind == "weights":
        mask = (masks.KVLenMask(s["lengths"]) if case["mask"] == "lengths"
                else masks.CausalMask() if case["mask"] == "causal" else None)
        out, weights = attention.attention_with_key_weights(s["q"], s["k"], s["v"], s["weights"], mask=mask,
                                                            sm_scale=s["scale"])
        return {"out": out, "weights": weights}
    if kind == "evict":
        r = attention.evict_keys(s["k"], s["v"], s["weights"], case["keep"], kv_lengths=s["lengths"],
                                 sinks=case["sinks"], recent=case["recent"])
        return {"k": r.k, "v": r.v, "weights": r.key_weights, "lengths": r.kv_lengths, "index": r.index}
    q, k = attention.rotary(s["q"], s["k"], s["positions"], sections=s["sections"],
                            interleaved=case["interleaved"], shared_spectrum=case["shared"])
    if not case["backward"]:
        return {"q": q, "k": k}
    dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------

def work(case):
    size, kind, B, D = SIZE[case["dtype"]], case["kind"], case["batch"], case["head_dim"]
    if kind == "rotary":
        values = B * case["length"] * (case["heads"] + case["kv_heads"]) * D * (2 if case["backward"] else 1)
        pairs = sum(int(x) for x in case["sections"].split("+")) / (2 * D)
        return {"bytes": 2 * size * values + 4 * B * case["length"] * len(case["sections"].split("+")),
                "flops": 6 * values * pairs}
    S, Hkv = case["capacity"], case["kv_heads"]
    if kind == "evict":
        kept = sum(min(n, case["keep"]) for n in _spread(case["shortest"], S, B))
        looked = sum(_spread(case["shortest"], S, B))
        slots = B * case["keep"] * Hkv
        # weights looked at; K and V of the kept keys read, of every place written; weights and indices written
        return {"bytes": 4 * Hkv * looked + 2 * size * D * (kept * Hkv + slots) + 8 * slots, "flops": Hkv * looked}
    if kind == "weights":
        T, H = case["q_len"], case["heads"]
        keys = sum(_spread(case["shortest"], S, B))
        scores = B * T * (T + 1) / 2 if case["mask"] == "causal" else T * keys
        return {"bytes": size * (2 * keys * Hkv * D + 2 * B * T * H * D) + 8 * B * Hkv * S,
                "flops": 4 * H * D * scores + H * scores}
    T, H = case["tokens"], case["heads"]
    sizes = _sizes(case) if case["form"] == "parents" else [T] * B
    prefix = _spread(case["shortest"], S - T, B)
    keys = sum(prefix) + sum(sizes)
    tree = {"shared": 4 * T, "parents": 4 * B * T, "mask": B * T * T}[case["form"]]
    scores = sum(sizes) * sum(prefix) / B + sum(n * n / 2 for n in sizes)
    return {"bytes": size * (2 * keys * Hkv * D + (sum(sizes) + B * T) * H * D) + tree, "flops": 4 * H * D * scores}


# ---------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------

def _attend64(q, k, v, scale, keep):
    """One KV head of one sequence: ``q [G, T, D]``, ``k, v [n, D]``, ``keep
    [T, n]`` -> output and weights, empty rows zero."""
    x = torch.matmul(q, k.t().contiguous()) * scale
    if keep is not None:
        x = x.masked_fill(~keep, float("-inf"))
    p = torch.nan_to_num(torch.softmax(x, dim=-1), nan=0.0)
    return torch.matmul(p, v), p


def _exact_attention(s):
    case = s["case"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    B, T, Hq, D = q.shape
    S, Hkv = k.shape[1:3]
    G = Hq // Hkv
    out = torch.zeros_like(q)
    weights = s["weights"].double().clone() if "weights" in s else None
    lengths = s["lengths"].tolist() if "lengths" in s else [S] * B
    for b in range(B):
        n, keep = lengths[b], None
        if case["kind"] == "tree":
            keep = torch.ones((T, n + T), dtype=torch.bool, device="cuda")
            keep[:, n:] = False
            if "tree_mask" in s:
                keep[:, n:] = s["tree_mask"][b]
            else:
                parents = s["parents"].expand(B, T)[b].tolist()
                for t in range(T):
                    if parents[t] < -1:
                        keep[t] = False
                        continue
                    a = t
                    while a >= 0:
                        keep[t, n + a] = True
                        a = parents[a]
            n = n + T
        elif case["mask"] == "causal":
            keep = torch.ones((T, S), dtype=torch.bool, device="cuda").tril()
        for h in range(Hkv):
            g = slice(h * G, (h + 1) * G)
            o, p = _attend64(q[b, :, g].transpose(0, 1).contiguous(), k[b, :n, h].contiguous(),
                             v[b, :n, h].contiguous(), s["scale"], keep)
            out[b, :, g] = o.transpose(0, 1)
            if weights is not None:
                weights[b, h, :n] += p.sum((0, 1))
    return out if weights is None else {"out": out, "weights": weights}


def _exact_rotary(s):
    """Every pair as a complex number, turned by exp(i position frequency)."""
    case, sections = s["case"], s["sections"]
    width = sum(sections)
    turns, at = [], 0
    for a, d in enumerate(sections):
        i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
        f = torch.exp(-math.log(10000.0) * ((at // 2 + i) * 2 / width if case["shared"] else i * 2 / d))
        turns.append(s["positions"][..., a:a + 1].double() * f)
        at += d
    turns = [torch.cat(turns, -1)] if case["shared"] else turns
    out = {}
    for n, sign in (("q", 1), ("k", 1)) + ((("dq", -1), ("dk", -1)) if case["backward"] else ()):
        x, parts = s[n].detach().double(), []
        for t, y in zip(turns, x[..., :width].split([2 * t.shape[-1] for t in turns], -1)):
            y = y.unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
            y = y if case["interleaved"] else y.transpose(-1, -2)
            z = torch.view_as_complex(y.contiguous()) * torch.polar(torch.ones_like(t), sign * t)[:, :, None]
            y = torch.view_as_real(z)
            parts.append((y if case["interleaved"] else y.transpose(-1, -2)).flatten(-2))
        out[n] = torch.cat(parts + [x[..., width:]], -1)
    return out


def _exact_evict(s):
    """Head by head: protected keys first, then by weight, then by place."""
    case = s["case"]
    B, Hkv, S = s["weights"].shape
    keep, D = case["keep"], case["head_dim"]
    w = s["weights"].double().cpu().numpy()
    index = np.full((B, Hkv, keep), -1)
    for b, n in enumerate(s["lengths"].tolist()):
        j = np.arange(n)
        open_ = (j >= case["sinks"]) & (j < n - case["recent"])
        for h in range(Hkv):
            best = np.lexsort((j, -w[b, h, :n], open_))[:keep]
            index[b, h, :len(best)] = np.sort(best)
    at = torch.from_numpy(index).cuda()
    out = {"weights": torch.zeros((B, Hkv, keep), dtype=torch.float64, device="cuda"),
           "k": torch.zeros((B, keep, Hkv, D), dtype=torch.float64, device="cuda")}
    out["v"] = torch.zeros_like(out["k"])
    for b, n in enumerate(s["lengths"].tolist()):
        m = min(n, keep)
        for h in range(Hkv):
            out["weights"][b, h, :m] = s["weights"][b, h, at[b, h, :m]].double()
            for x in ("k", "v"):
                out[x][b, :m, h] = s[x][b, at[b, h, :m], h].double()
    return {**out, "lengths": s["lengths"].clamp_max(keep), "index": at.to(torch.int32)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(s)
    if case["kind"] == "evict":
        return _exact_evict(s)
    return _exact_attention(s)
