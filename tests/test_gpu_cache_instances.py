"""Kernel instances of the operators over a KV cache that only large calls, or a
switch, reach: trees of 128 rows a workgroup, and decode steps with weights whose
cache is streamed.  Each test asserts which instance ran; results are compared with
the definition in float64, tolerances those of the operators' own tests."""

import math

import numpy as np
import pytest

from oracle import cache_ops as ref
from tests.test_gpu_key_weights import check_weights
from tests.test_gpu_tree_attention import _inputs, _types, check, random_parents

pytestmark = pytest.mark.gpu

FORMAT = {"bf16": "Bf16Fmt", "f16": "F16Fmt"}


def _ran(kernel):
    from probjax_amd import native

    assert kernel in native.last_launches(), native.last_launches()


def _prefixes(rng, B, S, T):
    """Lengths of every kind: none, one, up to the cache's end, past it."""
    L = rng.integers(0, S - T + 1, B)
    L[:6] = [0, 1, S - T, S - 1, S, S + 9]
    return L


# 512 workgroups of 128 rows and more than 64 rows a KV head: eight waves each
WIDE = [
    # dtype, B, T, S, Hq, Hkv, D, chunk
    ("bf16", 64, 33, 150, 16, 8, 128, 0),     # 66 rows
    ("f16", 64, 65, 300, 8, 8, 64, 128),      # 65 rows, three chunks
    ("bf16", 64, 17, 140, 32, 8, 72, 0),      # 68 rows of 72 features
    ("f16", 64, 20, 130, 32, 8, 40, 128),     # 80 rows of 40
    ("bf16", 32, 36, 520, 32, 8, 128, 512),   # 144 rows: two row groups
]


@pytest.mark.parametrize("form", ["parents", "mask"])
@pytest.mark.parametrize("case", WIDE, ids=lambda c: "-".join(map(str, c)))
def test_trees_of_128_rows_a_workgroup(device, case, form):
    import torch
    from probjax_amd.hip_attention import tree_decode

    name, B, T, S, Hq, Hkv, D, chunk = case
    dtype, scale = _types()[name], 1.0 / math.sqrt(D)
    (q, k, v), host = _inputs(41, dtype, B, T, S, Hq, Hkv, D, device)
    rng = np.random.default_rng(T)
    L = _prefixes(rng, B, S, T)
    if form == "mask":
        sees = rng.random((B, T, T)) < 0.3
        sees[:, 0] = False
        token = np.ones((B, T), bool)
        kw = dict(tree_mask=torch.from_numpy(sees).to(device))
    else:
        parents = random_parents(rng, B, T, absent=True)
        sees, token = zip(*(ref.tree_sees(p) for p in parents))
        kw = dict(parents=torch.from_numpy(parents).to(device))
    print(f"wide tree {case} {form}", flush=True)
    got, lse = tree_decode(q, k, v, sm_scale=scale, kv_lengths=torch.from_numpy(L).to(device), chunk=chunk,
                           return_lse=True, **kw)
    torch.cuda.synchronize()
    _ran(f"tree_wide_kernel<{FORMAT[name]}, {64 if D <= 64 else 128}, 4, 2>")
    check(got, lse, ref.tree_attention(*host, L, sees, token, scale), dtype, D, S)


@pytest.mark.parametrize("name,D", [("bf16", 128), ("f16", 64)])
def test_unseen_infinities_in_trees_of_128_rows_a_workgroup(device, name, D):
    import torch
    from probjax_amd.attention import tree_attention

    B, T, S, Hq, Hkv = 64, 33, 200, 16, 8
    (q, k, v), _ = _inputs(42, _types()[name], B, T, S, Hq, Hkv, D, device)
    rng = np.random.default_rng(8)
    tree = random_parents(rng, 1, T)[0]
    sees, _ = ref.tree_sees(tree)
    bad_v = next(t for t in range(4, T) if sees[:, t].sum() > 1)  # a token that others descend from
    bad_k = next(t for t in range(bad_v + 1, T) if not sees[t, bad_v])
    L = torch.from_numpy(rng.integers(0, S - T + 1, B)).to(device)
    kw = dict(parents=tree.tolist(), kv_lengths=L)
    clean = tree_attention(q, k, v, **kw)
    for b in range(B):
        P = int(L[b])
        v[b, P + bad_v, :, 3], v[b, P + bad_v, :, 50] = float("inf"), float("nan")
        k[b, P + bad_k] = float("nan")
        k[b, P + T:], v[b, P + T:] = float("nan"), float("nan")  # behind the draft: never read
    got = tree_attention(q, k, v, **kw)
    torch.cuda.synchronize()
    _ran(f"tree_wide_kernel<{FORMAT[name]}, {D}, 4, 2>")
    rest = [d for d in range(D) if d not in (3, 50)]
    for t in range(T):
        if sees[t, bad_k]:
            assert torch.isnan(got[:, t]).all(), t
        elif sees[t, bad_v]:
            assert torch.isposinf(got[:, t, :, 3]).all() and torch.isnan(got[:, t, :, 50]).all(), t
            assert torch.equal(got[:, t][..., rest], clean[:, t][..., rest]), t
        else:
            assert torch.equal(got[:, t], clean[:, t]), t
    assert (~sees[:, bad_v] & ~sees[:, bad_k]).any()


STREAMED = [
    # dtype, B, T, S, Hq, Hkv, D, lengths, 16-row blocks
    ("bf16", 4, 1, 700, 8, 2, 128, [700, 129, 1, 0], 1),
    ("bf16", 3, 5, 1301, 8, 2, 128, [1301, 640, 33], 2),   # 20 rows, a cache of an odd length
    ("f16", 3, 3, 515, 8, 2, 64, [515, 128, 31], 1),
    ("f16", 2, 8, 300, 8, 2, 64, [299, 40], 2),
    ("bf16", 2, 1, 257, 2, 2, 64, None, 1),                # without lengths
    ("bf16", 300, 1, 150, 2, 1, 128, "any", 1),            # more sequences than the schedule sorts
]


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("case", STREAMED, ids=lambda c: "-".join(map(str, c)))
def test_decode_steps_with_weights_of_a_streamed_cache(device, monkeypatch, case, strided):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights

    monkeypatch.setenv("PJX_DECODE_STREAM", "1")
    name, B, T, S, Hq, Hkv, D, lengths, blocks = case
    dtype, scale = _types()[name], 1.0 / math.sqrt(D)
    (q, k, v), host = _inputs(43, dtype, B, T, S, Hq, Hkv, D, device)
    rng = np.random.default_rng(S)
    L = rng.integers(0, S + 1, B) if lengths == "any" else np.array([S] * B if lengths is None else lengths)
    base = rng.random((B, Hkv, S)).astype(np.float32)
    mask = None if lengths is None else masks.KVLenMask(torch.from_numpy(L).to(device))
    for b in range(B):  # behind the lengths: never read
        k[b, L[b]:], v[b, L[b]:] = float("nan"), float("inf")
    if strided:
        k, v = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    print(f"streamed {case} {strided}", flush=True)
    out, w, lse = attention_with_key_weights(q, k, v, torch.from_numpy(base).to(device), mask=mask, return_lse=True)
    torch.cuda.synchronize()
    _ran(f"scored_decode_kernel<{FORMAT[name]}, {D}, {blocks}, true, false>")
    keep = np.stack([np.broadcast_to(np.arange(S) < n, (T, S)) for n in L])
    want = ref.key_weight_attention(*host, base, keep, scale)
    check(out, lse, want, dtype, D, S)
    check_weights(w, want, base, D, S, T * Hq // Hkv)
