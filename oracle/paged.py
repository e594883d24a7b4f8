"""A paged KV cache in float64 (oracle): rows in 8 bits, appending, reading back,
attention of the newest tokens.  No counterpart in the reference.  Pinned in
``tests/test_oracle_paged.py``."""

import numpy as np

from .cache_ops import attend


def e4m3_value(code):
    """The value of one e4m3 code: 4 bits of exponent (bias 7), 3 of fraction; all
    ones is NaN, there are no infinities."""
    e, f = code >> 3 & 15, code & 7
    if code & 127 == 127:
        return np.nan
    x = f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
    return -x if code & 128 else x


E4M3 = np.array([e4m3_value(c) for c in range(256)])

# Largest magnitude whose code reads back inside the range of the type it came in.
MOST = {"f16": 240 * 2.0 ** 8, "bf16": 240 * 2.0 ** 120, "f32": 240 * 2.0 ** 120}


def row_exponents(x):
    """``exponent + 127`` of rows ``[..., D]``: the least, from 1 on, with the largest
    finite value at most ``448 * 2^exponent``."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1, initial=0.0)
    e = np.full(a.shape, -126)
    for _ in range(400):
        more = a > 448.0 * np.exp2(e.astype(np.float64))
        if not more.any():
            break
        e = e + more
    return (e + 127).astype(np.uint8)


def encode(x, name):
    """``(codes, exponents)`` of rows ``[..., D]`` of type ``name``: every value to the
    nearest code, ties to the even one, by search."""
    x = np.asarray(x, np.float64)
    exponents = row_exponents(x)
    y = np.clip(x, -MOST[name], MOST[name]) * np.exp2(127.0 - exponents)[..., None]
    up = E4M3[:127]
    at = np.clip(np.searchsorted(up, np.abs(y)), 1, 126)
    low, high = np.abs(y) - up[at - 1], up[at] - np.abs(y)
    code = np.where((low < high) | ((low == high) & (at % 2 == 1)), at - 1, at)
    code = code | np.where(np.signbit(y), 128, 0)
    return np.where(np.isfinite(x), code, 127).astype(np.uint8), exponents


def decode(codes, exponents):
    return E4M3[codes] * np.exp2(exponents.astype(np.float64) - 127)[..., None]


def slots(table, page, pages, b, positions):
    """``(page, slot)`` of sequence b's positions, page -1 where there is none."""
    positions = np.asarray(positions)
    p = np.asarray(table)[b][positions // page]
    return np.where((p >= 0) & (p < pages), p, -1), positions % page


def append(pool, new, table, before, count):
    """``pool [pages, page, ...]`` with ``new[b, :count[b]]`` behind ``before[b]`` keys of
    every sequence, and the lengths then."""
    pool = pool.copy()
    pages, page = pool.shape[:2]
    room = np.asarray(table).shape[1] * page
    lengths = []
    for b in range(len(new)):
        first, n = max(int(before[b]), 0), min(max(int(count[b]), 0), new.shape[1])
        lengths.append(min(first + n, room))
        for t in range(n):
            if first + t < room:
                p, s = slots(table, page, pages, b, first + t)
                if p >= 0:
                    pool[p, s] = new[b, t]
    return pool, np.array(lengths, np.int32)


def gather(pool, table, lengths, length):
    """``(rows [B, length, ...], there [B, length])``: zeros where there is none."""
    pages, page = pool.shape[:2]
    B, N = np.asarray(table).shape
    out = np.zeros((B, length) + pool.shape[2:], pool.dtype)
    there = np.zeros((B, length), bool)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), N * page, length)
        p, s = slots(table, page, pages, b, np.arange(n))
        there[b, :n] = p >= 0
        out[b, :n][p >= 0] = pool[p[p >= 0], s[p >= 0]]
    return out, there


def paged_decode(q, k, v, there, lengths, scale):
    """``q [B, T, Hq, D]`` over gathered ``k, v [B, S, Hkv, D]``: token t sees the first
    ``lengths[b] - (T - 1 - t)`` keys that are there."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    B, T, Hq, _ = q.shape
    S, Hkv = k.shape[1:3]
    res = {"out": np.zeros(q.shape), "spread": np.zeros(q.shape), "lse": np.zeros((B, Hq, T)),
           "reach": np.zeros((B, Hq, T))}
    for b in range(B):
        n = min(max(int(lengths[b]), 0), S)
        keep = (np.arange(S) < n - (T - 1 - np.arange(T))[:, None]) & there[b]
        for h in range(Hq):
            g = h // (Hq // Hkv)
            o, lse, _, spread, reach = attend(q[b, :, h], k[b, :, g], v[b, :, g], keep, scale)
            res["out"][b, :, h], res["spread"][b, :, h] = o, spread
            res["lse"][b, h], res["reach"][b, h] = lse, reach
    return res
