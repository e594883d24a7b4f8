"""The operators over a KV cache, restated in float64 (oracle).

Tree attention, attention that adds up the weight its keys were given, eviction
by that weight, and rotation by positions of several axes, each from its
definition.  ``inv_freq = base^(-2i/d)`` and the interleaved pair rotation are
the reference's (``probjax/nn/layers/encoding.py:171-211``); the rest has no
counterpart there.  Pinned in ``tests/test_oracle_cache_ops.py``.
"""

import numpy as np


def tree_sees(parents):
    """``(sees [T, T], token [T])`` of one tree: row t holds t and what its chain
    of parents names; a parent that is no earlier token ends the chain, one below
    -1 marks a slot without a token."""
    T = len(parents)
    sees = np.zeros((T, T), bool)
    for t in range(T):
        j = t
        while j >= 0:
            sees[t, j] = True
            j = int(parents[j]) if parents[j] < j else -1
    return sees, np.asarray(parents) >= -1


def attend(q, k, v, keep, scale):
    """One head's attention in float64: ``q [T, D]``, ``k, v [n, D]``, ``keep
    [T, n]`` -> ``(out, lse, p, spread, reach)`` with ``spread = sum p |v|`` and
    ``reach = max scale sum |q| |k|`` per row, what rounding errors scale with.
    What a row does not keep does not reach it."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    T, n = keep.shape
    out, spread = np.zeros((T, v.shape[1])), np.zeros((T, v.shape[1]))
    lse, reach, p = np.full(T, np.inf), np.zeros(T), np.zeros((T, n))
    for t in range(T):
        at = np.flatnonzero(keep[t])
        if not at.size:
            continue
        s = scale * (k[at] @ q[t])
        m = s.max()
        e = np.exp(s - m)
        p[t, at] = e / e.sum()
        lse[t] = m + np.log(e.sum())
        out[t] = p[t, at] @ v[at]
        spread[t] = p[t, at] @ np.abs(v[at])
        reach[t] = scale * (np.abs(k[at]) @ np.abs(q[t])).max()
    return out, lse, p, spread, reach


def _heads(q, k, v, keep_of, scale):
    """``attend`` over ``q [B, T, Hq, D]`` and ``k, v [B, S, Hkv, D]``; ``keep_of(b)``
    gives ``[T, S]``."""
    B, T, Hq, D = q.shape
    S, Hkv = k.shape[1:3]
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    lse, reach = np.zeros((B, Hq, T)), np.zeros((B, Hq, T))
    weights = np.zeros((B, Hkv, S))
    for b in range(B):
        keep = keep_of(b)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            o, l, p, sp, re = attend(q[b, :, h], k[b, :, g], v[b, :, g], keep, scale)
            out[b, :, h], lse[b, h], spread[b, :, h], reach[b, h] = o, l, sp, re
            weights[b, g] += p.sum(0)
    return dict(out=out, lse=lse, weights=weights, spread=spread, reach=reach)


def tree_attention(q, k, v, lengths, sees, token, scale):
    """``sees [B, T, T]``, ``token [B, T]``; the drafted keys are slots
    ``lengths[b] ..`` as far as the cache reaches."""
    T, S = q.shape[1], k.shape[1]

    def keep_of(b):
        P = int(np.clip(lengths[b], 0, S))
        n = min(T, S - P)
        keep = np.zeros((T, S), bool)
        keep[:, :P] = True
        keep[:, P:P + n] = sees[b][:, :n]
        keep[~np.asarray(token[b], bool)] = False
        return keep

    return _heads(q, k, v, keep_of, scale)


def key_weight_attention(q, k, v, weights, keep, scale):
    """Attention and ``weights [B, Hkv, S]`` plus the softmax weight of every key,
    summed over the rows and heads that look at it; ``keep [B, T, S]``."""
    r = _heads(q, k, v, lambda b: keep[b], scale)
    r["weights"] = np.asarray(weights, np.float64) + r["weights"]
    return r


def evict(weights, length, keep, sinks=0, recent=0):
    """Slots that one head keeps, ascending: every one of a sequence of at most
    ``keep`` keys; else the first ``sinks``, the last ``recent`` and the largest
    weights (NaN first, ties to the lowest slot)."""
    length = int(np.clip(length, 0, len(weights)))
    if length <= keep:
        return list(range(length))

    def rank(j):
        w = float(weights[j])
        middle = sinks <= j < length - recent
        return (middle, w == w, -w if w == w else 0.0, j)

    return sorted(sorted(range(length), key=rank)[:keep])


def rotary(x, positions, sections, base=10000.0, interleaved=True, shared_spectrum=False, sign=1):
    """``x [B, T, H, D]`` turned by ``positions [B, T, A]`` (``sign`` -1: back)."""
    x = np.asarray(x, np.float64)
    out = x.copy()
    width, at = sum(sections), 0
    for a, d in enumerate(sections):
        for i in range(d // 2):
            power = (at + 2 * i) / width if shared_spectrum else 2 * i / d
            lo, n = (0, width) if shared_spectrum else (at, d)
            p = (at // 2 if shared_spectrum else 0) + i
            f, s = (lo + 2 * p, lo + 2 * p + 1) if interleaved else (lo + p, lo + p + n // 2)
            t = sign * np.asarray(positions, np.float64)[..., a] * float(base) ** -power
            c, n_ = np.cos(t)[..., None], np.sin(t)[..., None]
            out[..., f] = x[..., f] * c - x[..., s] * n_
            out[..., s] = x[..., s] * c + x[..., f] * n_
        at += d
    return out
