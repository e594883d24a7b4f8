"""What the speed of the paged cache's operators is measured on.

``listed()`` holds the fixed cases, ``draw(rng)`` gives another one of the same
ranges.  ``prepare`` makes what a program has in hand before the call (inputs on
the GPU, the cache and its page table), ``run`` is one pass: the operators in
their plain form, or with ``own`` the calls a program makes of the framework.
``work`` gives the bytes and operations a pass cannot do without, ``exact`` the
same outputs from the definition in float64.

A paged cache is a pool of pages ``[pages, page, kv_heads, head_dim]`` for K and
one for V, and for every sequence a row of page numbers (-1: none).  In 8 bits
the pools hold e4m3 codes, and every row (one token's key or value of one head)
has a power of two that its codes are multiplied by, held as ``exponent + 127``
in ``[pages, kv_heads, page]`` bytes.

Case kinds
  write   new keys and values appended to their sequences, in 8 bits or copied
  read    the sequences' keys and values gathered into ``[B, L, H, D]`` tensors
  decode  attention of every sequence's newest tokens over its cache
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "e4m3": 1}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _write(name, dtype, cache, batch, tokens, shortest, before, kv_heads, head_dim, page, fused):
    """``before``: keys the longest sequence holds; ``shortest``: new tokens of the
    sequence with the fewest; ``fused``: k and v are slices of one projection."""
    c = dict(kind="write", dtype=dtype, cache=cache, batch=batch, tokens=tokens, shortest=shortest, before=before,
             kv_heads=kv_heads, head_dim=head_dim, page=page, fused=fused)
    return dict(c, name=name) if name else c


def _read(name, dtype, cache, batch, capacity, shortest, kv_heads, head_dim, page, layout):
    c = dict(kind="read", dtype=dtype, cache=cache, batch=batch, capacity=capacity, shortest=shortest,
             kv_heads=kv_heads, head_dim=head_dim, page=page, layout=layout)
    return dict(c, name=name) if name else c


def _decode(name, dtype, cache, batch, tokens, heads, kv_heads, capacity, shortest, head_dim, page, layout):
    """``layout``: a page's order in memory, "tokens" ``[page, H, D]`` or "heads"
    ``[H, page, D]``."""
    c = dict(kind="decode", dtype=dtype, cache=cache, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads,
             capacity=capacity, shortest=shortest, head_dim=head_dim, page=page, layout=layout)
    return dict(c, name=name) if name else c


def listed():
    return [
        # One token for every sequence of a serving batch, written in 8 bits: launch and latency bound.
        _write("write_step_e4m3", "bf16", "e4m3", 32, 1, 1, 1000, 8, 128, 64, True),
        # A batch of prompts of different length into an empty cache, in 8 bits.
        _write("write_prompts_e4m3", "bf16", "e4m3", 8, 4096, 300, 0, 8, 128, 64, True),
        # A second turn's prompts behind the first one's, wide heads, kept in their own type.
        _write("write_prompts_bf16", "bf16", "bf16", 4, 2048, 2048, 1111, 4, 256, 32, False),
        # A small float32 model's sequences read back.
        _read("read_small_f32", "f32", "f32", 2, 1008, 517, 4, 64, 48, "tokens"),
        # A serving batch's caches read back for the next turn's prompts.
        _read("read_batch_e4m3", "bf16", "e4m3", 16, 8192, 1000, 8, 128, 64, "tokens"),
        # One token of a small float32 model (the library's default dtype).
        _decode("decode_small_f32", "f32", "f32", 2, 1, 4, 4, 512, 200, 64, 16, "tokens"),
        # One token of one chat.
        _decode("decode_single_bf16", "bf16", "bf16", 1, 1, 32, 8, 4096, 4090, 128, 16, "tokens"),
        # One token for every sequence of a serving batch, caches of different fill.
        _decode("decode_batch_bf16", "bf16", "bf16", 32, 1, 32, 8, 8192, 512, 128, 64, "tokens"),
        # The same batch with its cache in 8 bits.
        _decode("decode_batch_e4m3", "bf16", "e4m3", 32, 1, 32, 8, 8192, 512, 128, 64, "tokens"),
        # One token of one very long text, in 8 bits, pages ordered by head.
        _decode("decode_long_e4m3", "bf16", "e4m3", 1, 1, 32, 8, 131072, 131000, 128, 128, "heads"),
        # Five drafted tokens for every sequence, in 8 bits.
        _decode("decode_drafts_e4m3", "f16", "e4m3", 16, 5, 32, 8, 4096, 900, 128, 16, "tokens"),
        # Heads and pages that are no powers of two.
        _decode("decode_odd_f16", "f16", "f16", 7, 1, 12, 4, 2900, 333, 96, 20, "tokens"),
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
    kind = rng.choice(("write", "read", "decode", "decode", "decode"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    cache = rng.choice((dtype, "e4m3"))
    head_dim = rng.choice((64, 64, 80, 96, 112, 128, 128, 128, 192, 256))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    page = rng.choice((16, 16, 32, 64, 64, 128, 256, 1, 8, 20, 100))
    batch = _log_int(rng, 1, 32)
    layout = rng.choice(("tokens", "heads"))
    if kind == "write":
        tokens = rng.choice((1, 2, 5, _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)))
        return _write(None, dtype, cache, batch, tokens, rng.randint(1, tokens), _log_int(rng, 1, 4096), kv_heads,
                      head_dim, page, rng.random() < 0.5)
    if kind == "read":
        capacity = _log_int(rng, 64, 16384)
        return _read(None, dtype, cache, batch, capacity, rng.randint(1, capacity), kv_heads, head_dim, page, layout)
    tokens = rng.choice((1, 1, 1, 1, 2, 5, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 7, 8, 16))
    capacity = _log_int(rng, 64, 131072)
    return _decode(None, dtype, cache, batch, tokens, heads, kv_heads, capacity,
                   rng.randint(min(tokens, capacity), capacity), head_dim, page, layout)


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------

def _spread(shortest, longest, batch):
    """Lengths spread evenly from ``longest`` down to ``shortest``."""
    if batch == 1:
        return [longest]
    return [round(longest - (longest - shortest) * i / (batch - 1)) for i in range(batch)]


def _pages(case):
    """Most pages of a sequence."""
    longest = case["before"] + case["tokens"] if case["kind"] == "write" else case["capacity"]
    return -(-longest // case["page"])


def _in_8_bits(x):
    """``x [pages, page, H, D]`` as e4m3 codes and exponents ``[pages, H, page]``."""
    codes, exponents = _encode(x)
    return codes, exponents.permute(0, 2, 1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, kind, B = DTYPES[case["dtype"]], case["kind"], case["batch"]
    H, D, page, N = case["kv_heads"], case["head_dim"], case["page"], _pages(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    def order(n):
        return torch.randperm(n, generator=gen, device="cuda")

    s = {"case": case}
    if kind == "write":
        s["lengths"] = torch.tensor(_spread(case["before"] // 2, case["before"], B), dtype=torch.int32).cuda()[order(B)]
        s["new"] = torch.tensor(_spread(case["shortest"], case["tokens"], B), dtype=torch.int32).cuda()[order(B)]
        used = s["lengths"] + case["tokens"]
        if case["fused"]:
            s["k"], s["v"] = normal(B, case["tokens"], 4 * H, D)[:, :, 2 * H:].split(H, dim=2)
        else:
            s["k"], s["v"] = normal(B, case["tokens"], H, D), normal(B, case["tokens"], H, D)
    else:
        s["lengths"] = torch.tensor(_spread(case["shortest"], case["capacity"], B), dtype=torch.int32).cuda()[order(B)]
        used = s["lengths"]
    # pages of one pool in no order; none behind a sequence's end
    slots = torch.arange(N, device="cuda") * page
    s["table"] = torch.where(slots < used[:, None], order(B * N).view(B, N), -1).to(torch.int32)
    for n in ("k", "v"):
        pool = normal(B * N, page, H, D)
        if case["cache"] == "e4m3":
            pool, s[n + "_exponents"] = _in_8_bits(pool)
        if case.get("layout") == "heads":
            pool = pool.view(torch.uint8) if case["cache"] == "e4m3" else pool
            pool = pool.transpose(1, 2).contiguous().transpose(1, 2).view(DTYPES[case["cache"]])
        s[n + "_pool"] = pool
    if kind == "decode":
        s["q"] = normal(B, case["tokens"], case["heads"], D)
        s["scale"] = 1.0 / math.sqrt(D)
    if own:  # what a program makes once and keeps: the cache, around the pools and the table
        from probjax_amd import attention

        s["cache"] = attention.PagedCache(s["k_pool"], s["v_pool"], s["table"], s.get("k_exponents"),
                                          s.get("v_exponents"))
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------

def _encode(x):
    """Rows ``[..., D]`` as e4m3 codes and ``exponent + 127`` ``[...]`` (uint8): the
    least power of two that brings the row's largest value to at most 448.  A value
    that would read back past the range of the rows' type is held at 240."""
    most = 61440.0 if x.dtype == torch.float16 else 1.875 * 2.0 ** 127
    x = x.float()
    finite = torch.isfinite(x)
    bits = torch.where(finite, x.abs(), 0.0).amax(-1).view(torch.int32)
    # 448 is 1.75 * 2^8: its fraction's bits are 0x600000
    exponent = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp_min(1)
    back = ((254 - exponent) << 23).view(torch.float32)
    codes = torch.where(finite, x.clamp(-most, most) * back[..., None], float("nan")).to(torch.float8_e4m3fn)
    return codes, exponent.to(torch.uint8)


def _gather(s, n):
    """All pages of every sequence ``[B, N * page, H, D]``, in float32."""
    case, table = s["case"], s["table"].long().clamp_min(0)
    pool = s[n + "_pool"]
    if case["cache"] != "e4m3":
        return pool[table].float().flatten(1, 2)
    x = pool.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
    scale = (s[n + "_exponents"][table].int() << 23).view(torch.float32)  # [B, N, H, page]
    return (x * scale.permute(0, 1, 3, 2)[..., None]).flatten(1, 2)


def _plain_write(s):
    case = s["case"]
    T, page = case["tokens"], case["page"]
    t = torch.arange(T, device="cuda")
    at = s["lengths"].long()[:, None] + t
    there = (t < s["new"][:, None])[..., None]  # [B, T, 1]
    pages, slot = torch.gather(s["table"].long(), 1, at // page), at % page
    out = {}
    for n in ("k", "v"):
        pool, x = s[n + "_pool"], s[n]
        if case["cache"] == "e4m3":
            x, exponent = _encode(x)
            exponents = s[n + "_exponents"]
            old = exponents[pages, :, slot]
            exponents[pages, :, slot] = torch.where(there, exponent, old)
            out[n + "_exponents"] = exponents
            codes, x = pool.view(torch.uint8), x.view(torch.uint8)
        else:
            codes = pool
        codes[pages, slot] = torch.where(there[..., None], x, codes[pages, slot])
        out[n] = pool
    return {**out, "lengths": s["lengths"] + s["new"]}


def _plain_read(s):
    case = s["case"]
    L, dtype = case["capacity"], DTYPES[case["dtype"]]
    there = (torch.arange(L, device="cuda") < s["lengths"][:, None])[..., None, None]
    return {n: torch.where(there, _gather(s, n)[:, :L], 0.0).to(dtype) for n in ("k", "v")}


def _plain_decode(s):
    case = s["case"]
    q = s["q"].float()
    B, T, Hq, D = q.shape
    H = case["kv_heads"]
    q = q.view(B, T, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D)
    k = _gather(s, "k").permute(0, 2, 3, 1).contiguous()  # [B, H, D, S]
    x = torch.matmul(q, k) * s["scale"]
    del k
    sees = s["lengths"][:, None] - (T - 1 - torch.arange(T, device="cuda"))  # keys that token t sees
    hidden = torch.arange(x.shape[-1], device="cuda") >= sees[..., None]  # [B, T, S]
    x = x.view(B, H, Hq // H, T, -1).masked_fill(hidden[:, None, None], float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    v = _gather(s, "v").permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p.view(B, H, -1, p.shape[-1]), v).view(B, H, Hq // H, T, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D).to(s["q"].dtype)


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode}[kind](s)
    from probjax_amd import attention

    cache = s["cache"]
    if kind == "write":
        lengths = attention.write_pages(cache, s["k"], s["v"], kv_lengths=s["lengths"], new_lengths=s["new"])
        out = {"k": s["k_pool"], "v": s["v_pool"], "lengths": lengths}
        if s["case"]["cache"] == "e4m3":
            out.update(k_exponents=s["k_exponents"], v_exponents=s["v_exponents"])
        return out
    if kind == "read":
        k, v = attention.read_pages(cache, kv_lengths=s["lengths"], length=s["case"]["capacity"], dtype=DTYPES[s["case"]["dtype"]])
        return {"k": k, "v": v}
    return attention.paged_decode(s["q"], cache, kv_lengths=s["lengths"], sm_scale=s["scale"])


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------

def work(case):
    B, H, D, N = case["batch"], case["kv_heads"], case["head_dim"], _pages(case)
    size, held = SIZE[case["dtype"]], SIZE[case["cache"]]
    row = D * held + (1 if case["cache"] == "e4m3" else 0)  # of one key or value in the cache
    if case["kind"] == "write":
        rows = 2 * H * sum(_spread(case["shortest"], case["tokens"], B))
        return {"bytes": rows * (D * size + row) + 12 * B, "flops": 2 * rows * D}
    keys = sum(_spread(case["shortest"], case["capacity"], B))
    if case["kind"] == "read":
        return {"bytes": 2 * H * (keys * row + B * case["capacity"] * D * size) + 4 * B * N, "flops": 2 * H * keys * D}
    T, Hq = case["tokens"], case["heads"]
    return {"bytes": 2 * H * keys * row + 2 * B * T * Hq * D * size + 4 * B * N, "flops": 4 * T * Hq * D * keys}


# ---------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------

def _e4m3_values():
    """The value of every code: sign, 4 bits of exponent (bias 7), 3 of fraction;
    all ones is NaN."""
    values = []
    for code in range(256):
        e, f = code >> 3 & 15, code & 7
        x = float("nan") if code & 127 == 127 else f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        values.append(-x if code & 128 else x)
    return torch.tensor(values, dtype=torch.float64).cuda()


def _sequence64(s, n, b, length):
    """The first ``length`` keys or values of sequence b, slot by slot: ``[length, H, D]``."""
    page = s["case"]["page"]
    at = torch.arange(length, device="cuda")
    where = s["table"][b].long()[at // page], at % page
    x = s[n + "_pool"]
    if s["case"]["cache"] != "e4m3":
        return x[where].double()
    exponents = s[n + "_exponents"].permute(0, 2, 1)[where].double() - 127
    return _e4m3_values()[x.view(torch.uint8)[where].long()] * torch.exp2(exponents)[..., None]


def _encode64(x):
    """e4m3 values and exponents of rows ``[..., D]``, by the definition."""
    most = 61440.0 if x.dtype == torch.float16 else 1.875 * 2.0 ** 127
    x = x.double()
    m, e = torch.frexp(x.abs().amax(-1) / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp_min(-126)  # least e with amax <= 448 * 2^e
    y = x.clamp(-most, most) * torch.exp2(-e.double())[..., None]
    step = torch.exp2((torch.frexp(y.abs())[1] - 1).clamp_min(-6).double() - 3)
    return torch.round(y / step) * step, e + 127  # (round: ties to even)


def _exact_write(s):
    case = s["case"]
    page, out = case["page"], {}
    lengths, new = s["lengths"].tolist(), s["new"].tolist()
    for n in ("k", "v"):
        pool = s[n + "_pool"]
        quantised = case["cache"] == "e4m3"
        pool = _e4m3_values()[pool.view(torch.uint8).long()] if quantised else pool.double()
        exponents = s[n + "_exponents"].clone() if quantised else None
        for b, (before, more) in enumerate(zip(lengths, new)):
            at = torch.arange(before, before + more, device="cuda")
            pages, slot = s["table"][b].long()[at // page], at % page
            x = s[n][b, :more]
            if quantised:
                x, e = _encode64(x)
                exponents.permute(0, 2, 1)[pages, slot] = e.to(torch.uint8)
            pool[pages, slot] = x.double()
        out[n] = pool
        if quantised:
            out[n + "_exponents"] = exponents
    return {**out, "lengths": torch.tensor([x + y for x, y in zip(lengths, new)], dtype=torch.int32)}


def _exact_read(s):
    case = s["case"]
    out = {}
    for n in ("k", "v"):
        x = torch.zeros((case["batch"], case["capacity"], case["kv_heads"], case["head_dim"]), dtype=torch.float64,
                        device="cuda")
        for b, length in enumerate(s["lengths"].tolist()):
            x[b, :length] = _sequence64(s, n, b, length)
        out[n] = x
    return out


def _exact_decode(s):
    q = s["q"].double()
    B, T, Hq, D = q.shape
    H = s["case"]["kv_heads"]
    out = torch.zeros_like(q)
    for b, length in enumerate(s["lengths"].tolist()):
        k, v = _sequence64(s, "k", b, length), _sequence64(s, "v", b, length)
        sees = torch.ones((T, length), dtype=torch.bool, device="cuda").tril(length - T)
        for h in range(Hq):
            g = h * H // Hq
            x = torch.matmul(k[:, g], q[b, :, h].t().contiguous()).t() * s["scale"]
            p = torch.softmax(x.masked_fill(~sees, float("-inf")), dim=-1)
            out[b, :, h] = torch.matmul(p, v[:, g])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "decode": _exact_decode}[case["kind"]](s)
