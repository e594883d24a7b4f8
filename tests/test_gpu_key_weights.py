"""Attention that adds up the softmax weight of its keys against its definition
in float64.

Tolerances.  The output's are those of tests/test_gpu_tree_attention.py.  A
weight exp(s - lse) is float32: its score and its row's LSE are off by at most
(2 D reach + n + 24) 2^-24 together (sums of D products, of n weights, exp2),
and a score, its LSE and their difference, rounded in units of their size, by
8 |lse| 2^-24 more; a key's sum over m rows and the sum before it by m + 2 steps
of 2^-24.
"""

import math

import numpy as np
import pytest

from oracle import cache_ops as ref
from tests._helpers import to_np
from tests.test_gpu_tree_attention import _inputs, _types, check

pytestmark = pytest.mark.gpu


def check_weights(got, want, base, D, n, rows):
    lse = np.where(np.isfinite(want["lse"]), np.abs(want["lse"]), 0.0)
    rel = (2 * D * want["reach"] + n + 24 + 8 * lse).max() * 2.0 ** -24
    tol = rel * (want["weights"] - base) + (rows + 2) * 2.0 ** -24 * np.abs(want["weights"])
    err = np.abs(to_np(got) - want["weights"])
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])


CASES = [
    # dtype, B, T, S, Hq, Hkv, D, lengths (None: all), causal (None, "top", "bottom")
    ("bf16", 2, 1, 600, 8, 2, 128, [600, 77], None),      # decode steps: scores kept
    ("bf16", 3, 1, 129, 4, 4, 64, [129, 0, 1], None),
    ("bf16", 2, 2, 1500, 16, 2, 64, [1500, 1025], None),
    ("bf16", 1, 8, 2100, 8, 1, 128, None, None),          # 64 rows
    ("f16", 2, 5, 333, 6, 2, 80, [333, 10], None),
    ("f16", 2, 3, 131, 4, 2, 256, [131, 130], None),
    ("bf16", 2, 1, 97, 4, 2, 100, [97, 50], None),        # zero-padded rows
    ("f32", 2, 1, 515, 8, 2, 64, [515, 3], None),
    ("f32", 1, 12, 300, 8, 2, 128, [299], None),          # 48 rows
    ("f32", 2, 2, 150, 2, 2, 256, [150, 20], None),
    ("bf16", 1, 65, 200, 2, 2, 64, None, None),           # more rows: scores formed again
    ("bf16", 2, 300, 300, 4, 2, 128, None, "top"),
    ("bf16", 1, 257, 513, 4, 1, 64, None, "bottom"),
    ("bf16", 2, 400, 400, 4, 2, 64, [400, 130], "top"),
    ("f16", 1, 200, 200, 4, 2, 96, None, "top"),
    ("f16", 1, 130, 130, 2, 1, 256, [99], "top"),
    ("bf16", 1, 130, 90, 2, 1, 64, None, "bottom"),       # rows that see nothing
    ("bf16", 1, 70, 50, 2, 1, 200, None, "top"),
    ("f32", 1, 260, 260, 4, 2, 64, None, "top"),
    ("f32", 2, 100, 180, 2, 1, 128, [180, 33], None),
    ("f32", 1, 90, 90, 2, 2, 256, None, "top"),
    ("f32", 1, 70, 70, 2, 1, 48, None, "top"),
    ("bf16", 1, 1, 70, 2, 1, 64, None, "bottom"),         # one row under a causal mask
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_matches_definition(device, case):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights

    name, B, T, S, Hq, Hkv, D, lengths, causal = case
    dtype = _types()[name]
    (q, k, v), host = _inputs(15, dtype, B, T, S, Hq, Hkv, D, device)
    rng = np.random.default_rng(S)
    base = rng.random((B, Hkv, S)).astype(np.float32)
    scale = 1.0 / math.sqrt(D)
    L = np.array([S] * B if lengths is None else lengths)
    j, i = np.arange(S)[None, :], np.arange(T)[:, None]
    shift = {None: S, "top": 0, "bottom": S - T}[causal]
    keep = np.stack([(j < L[b]) & (j <= i + shift) for b in range(B)])
    mask = None
    if lengths is not None:
        mask = masks.KVLenMask(torch.tensor(lengths, dtype=torch.int32, device=device))
    if causal is not None:
        c = masks.CausalMask() if causal == "top" else masks.CausalFromBottomRightMask(T, S)
        mask = c if mask is None else c & mask
    want = ref.key_weight_attention(*host, base, keep, scale)
    print(f"key weights {case}", flush=True)
    out, w, lse = attention_with_key_weights(q, k, v, torch.from_numpy(base).to(device), mask=mask, sm_scale=scale,
                                             return_lse=True)
    torch.cuda.synchronize()
    check(out, lse, want, dtype, D, S)
    check_weights(w, want, base, D, S, T * Hq // Hkv)
    w0 = attention_with_key_weights(q, k, v, mask=mask, sm_scale=scale)[1]
    want["weights"] = want["weights"] - base
    check_weights(w0, want, 0.0, D, S, T * Hq // Hkv)


def test_both_ways_agree(device):
    """A step's kept scores and the scores formed again from its LSE give one sum,
    each within its tolerance."""
    import torch
    from probjax_amd import hip_attention as hip

    B, T, S, Hq, Hkv, D = 2, 4, 700, 8, 2, 128
    (q, k, v), host = _inputs(16, torch.bfloat16, B, T, S, Hq, Hkv, D, device)
    L = torch.tensor([700, 301], dtype=torch.int32, device=device)
    o, w, lse = hip.weighted_decode(q, k, v, sm_scale=0.09, kv_lengths=L, return_lse=True)
    w2 = hip.key_weights(q, k, lse, sm_scale=0.09, kv_lengths=L)
    keep = np.stack([np.broadcast_to(np.arange(S) < int(n), (T, S)) for n in L])
    want = ref.key_weight_attention(*host, np.zeros((B, Hkv, S)), keep, 0.09)
    for x in (w, w2):
        check_weights(x, want, 0.0, D, S, T * Hq // Hkv)
        assert (to_np(x)[1, :, 301:] == 0).all()
    # every row's weights add up to one
    assert abs(float(w.double().sum()) - B * T * Hq) <= 1e-4 * B * T * Hq


def test_what_a_mask_hides_does_not_reach_the_weights(device):
    """K and V past the lengths, and K past the diagonal's end, hold NaN."""
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights

    for T, mask_of in ((1, lambda L: masks.KVLenMask(L)), (90, lambda L: masks.CausalMask() & masks.KVLenMask(L))):
        (q, k, v), _ = _inputs(17, torch.bfloat16, 2, T, 300, 8, 2, 128, device)
        L = torch.tensor([211, 64], dtype=torch.int32, device=device)
        want = attention_with_key_weights(q, k, v, mask=mask_of(L))
        for b in range(2):
            k[b, int(L[b]):] = float("nan")
            v[b, int(L[b]):] = float("inf")
        got = attention_with_key_weights(q, k, v, mask=mask_of(L))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_caches_in_any_order_of_axes(device):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights

    for T in (1, 100):
        (q, k, v), _ = _inputs(18, torch.float16, 2, T, 260, 4, 2, 64, device)
        mask = masks.KVLenMask(torch.tensor([260, 99], device=device))
        w = torch.rand((2, 2, 260), device=device)
        want = attention_with_key_weights(q, k, v, w, mask=mask)
        kt, vt = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
        wt = w.permute(2, 0, 1).contiguous().permute(1, 2, 0)
        got = attention_with_key_weights(q, kt, vt, wt, mask=mask)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_replayed_graph(device):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights

    (q, k, v), _ = _inputs(19, torch.bfloat16, 2, 1, 900, 8, 2, 128, device)
    (p, kp, vp), _ = _inputs(20, torch.bfloat16, 1, 200, 200, 4, 2, 64, device)
    L = torch.tensor([900, 450], dtype=torch.int32, device=device)
    w = torch.zeros((2, 2, 900), device=device)

    def step():
        return (*attention_with_key_weights(q, k, v, w, mask=masks.KVLenMask(L)),
                *attention_with_key_weights(p, kp, vp, mask=masks.CausalMask()))

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        torch.manual_seed(i)
        for x in (q, k, v, p, kp, vp, w):
            x.copy_(torch.rand(x.shape, device=device))
        L.copy_(torch.tensor([900 - i, 3 + 100 * i], device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step())), i


def test_rejects(device):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights as f

    q = torch.zeros((2, 4, 4, 64), dtype=torch.bfloat16, device=device)
    k = torch.zeros((2, 50, 2, 64), dtype=torch.bfloat16, device=device)
    w = torch.zeros((2, 2, 50), device=device)
    f(q, k, k, w)
    bad = [
        (lambda: f(q, k, k, w[:, :1]), "shape"),
        (lambda: f(q, k, k, w.half()), "float32"),
        (lambda: f(q, k, k, w.cpu()), "float32 tensor on"),
        (lambda: f(q, k, k, w, mask=masks.LocalWindowMask(3, 3)), "takes no mask"),
        (lambda: f(q, k, k, w, mask=masks.KVLenMask([1, 2, 3])), "kv_lengths"),
        (lambda: f(q[:, :, :3], k, k, w), "multiple"),
        (lambda: f(q, k, k.float(), w), "one dtype"),
        (lambda: f(q, k[:1], k[:1], w), "incompatible"),
        (lambda: f(q.requires_grad_(), k, k, w), "no gradient"),
        (lambda: f(q.detach(), k, k, w, sm_scale=-1.0), "sm_scale"),
        (lambda: f(q.detach()[0], k, k, w), "must be"),
    ]
    for call, msg in bad:
        with pytest.raises(ValueError, match=msg):
            call()
    q = q.detach()
    o, w2 = f(q, k[:, :0], k[:, :0], w[:, :, :0])
    assert torch.equal(o, torch.zeros_like(q)) and w2.shape == (2, 2, 0)
    o, w2 = f(q[:, :0], k, k, w + 1)
    assert o.shape == (2, 0, 4, 64) and torch.equal(w2, w + 1)
