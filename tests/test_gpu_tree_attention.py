"""Tree attention (drafted tokens over a KV cache) against its definition in
float64.

Tolerances.  With u half a step of the type (relative), a 16-bit kernel rounds
every weight once (u sum p|v|) and the output once (u |o|).  In every type the
scores are float32 sums of D products, off by at most D 2^-24 reach (reach =
scale sum |q||k|), which moves a weight by that much relative and its norm by as
much again, and so do exp2 and the sums over n keys (2^-24 each, at most n + 16
of them): rel = 2 D 2^-24 reach + (n + 16) 2^-24, times spread = sum p|v|.
"""

import math

import numpy as np
import pytest

from oracle import cache_ops as ref
from tests._helpers import rng_normal, to_np

pytestmark = pytest.mark.gpu


def _types():
    import torch

    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _half_step(dtype):
    import torch

    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def check(got, lse, want, dtype, D, n):
    u = _half_step(dtype)
    rel = (2 * D * want["reach"] + n + 16) * 2.0 ** -24  # [B, Hq, T]
    rel = np.moveaxis(rel, 1, 2)[..., None]
    tol = u * (1 + rel) * (want["spread"] + np.abs(want["out"])) + rel * want["spread"] + 2.0 ** -24 * np.abs(want["out"])
    err = np.abs(to_np(got) - want["out"])
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])
    if lse is not None:
        lse, fin = to_np(lse), np.isfinite(want["lse"])
        np.testing.assert_array_equal(np.isposinf(lse), ~fin)
        off = np.abs(lse[fin] - want["lse"][fin])
        lim = (D * want["reach"][fin] + n + 16 + 4 * np.abs(want["lse"][fin])) * 2.0 ** -24
        assert (off <= lim).all(), (off.max(), lim.min())


def _inputs(seed, dtype, B, T, S, Hq, Hkv, D, device):
    import torch

    q, k, v = rng_normal(seed, (B, T, Hq, D), (B, S, Hkv, D), (B, S, Hkv, D))
    dev = [torch.from_numpy(x).to(device, dtype) for x in (q, k, v)]
    return dev, [to_np(x).astype(np.float64) for x in dev]


def random_parents(rng, B, T, absent=False):
    p = np.stack([[t - 1 - int(rng.integers(0, min(t + 1, 5))) for t in range(T)] for _ in range(B)])
    if absent:
        for b in range(B):
            p[b, T - (b % T):] = -2
    return p.astype(np.int32)


CASES = [
    # dtype, B, T, S, Hq, Hkv, D, prefix lengths, chunk
    ("bf16", 2, 5, 300, 4, 4, 64, [295, 17], 0),
    ("bf16", 1, 1, 130, 8, 2, 128, [129], 0),          # one token: a decode step
    ("bf16", 3, 8, 200, 8, 2, 128, [0, 1, 192], 128),  # no prefix: the root sees itself alone
    ("bf16", 2, 16, 700, 8, 2, 128, [684, 120], 128),  # the draft straddles two chunks
    ("bf16", 2, 33, 400, 4, 1, 64, [300, 127], 128),   # 132 rows, sets of two words
    ("bf16", 1, 64, 1200, 8, 2, 128, [1136], 256),     # 256 rows
    ("f16", 3, 16, 900, 8, 2, 64, [0, 884, 401], 256),  # 64 rows
    ("bf16", 5, 61, 400, 8, 2, 120, [300, 10, 339, 0, 77], 0),
    ("bf16", 1, 100, 300, 4, 2, 256, [200], 0),
    ("bf16", 1, 256, 600, 2, 1, 64, [300], 128),       # the widest draft
    ("f16", 2, 7, 333, 6, 3, 80, [320, 55], 128),      # rows of 80 features
    ("f16", 2, 26, 260, 8, 4, 96, [234, 100], 128),
    ("f16", 2, 12, 150, 4, 2, 128, [149, 145], 0),     # the cache ends inside the draft
    ("bf16", 2, 6, 140, 4, 2, 72, [150, -3], 0),       # lengths past the cache and negative
    ("bf16", 2, 6, 140, 4, 2, 100, [100, 30], 0),      # zero-padded rows
    ("bf16", 2, 6, 140, 4, 2, 200, [100, 30], 0),
    ("f32", 2, 5, 512, 4, 4, 64, [507, 200], 0),
    ("f32", 1, 17, 300, 8, 2, 128, [250], 128),
    ("f32", 2, 9, 140, 2, 1, 256, [131, 60], 0),
    ("f32", 2, 3, 140, 4, 2, 40, [100, 30], 0),
]


@pytest.mark.parametrize("form", ["parents", "shared", "mask"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:7])))
def test_matches_definition(device, case, form):
    import torch
    from probjax_amd.hip_attention import tree_decode

    name, B, T, S, Hq, Hkv, D, lengths, chunk = case
    dtype = _types()[name]
    (q, k, v), host = _inputs(5, dtype, B, T, S, Hq, Hkv, D, device)
    rng = np.random.default_rng(T)
    scale = 1.0 / math.sqrt(D)
    L = torch.tensor(lengths, dtype=torch.int32, device=device)
    kw = {}
    if form == "mask":
        sees = rng.random((B, T, T)) < 0.4
        sees[:, 0] = False  # a row that sees the prefix alone, and nothing without one
        token = np.ones((B, T), bool)
        kw["tree_mask"] = torch.from_numpy(sees).to(device)
    else:
        parents = random_parents(rng, 1 if form == "shared" else B, T, absent=form == "parents")
        trees = [ref.tree_sees(p) for p in parents] * (B if form == "shared" else 1)
        sees, token = [t[0] for t in trees], [t[1] for t in trees]
        kw["parents"] = torch.from_numpy(parents[0] if form == "shared" else parents).to(device)
    want = ref.tree_attention(*host, lengths, sees, token, scale)
    print(f"tree {case} {form}", flush=True)
    got, lse = tree_decode(q, k, v, sm_scale=scale, kv_lengths=L, chunk=chunk, return_lse=True, **kw)
    torch.cuda.synchronize()
    check(got[..., :D], lse, want, dtype, D, S)


@pytest.mark.parametrize("hq", [2, 8])  # 20 or 80 rows per KV head
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_unseen_infinities_do_not_reach_a_row(device, dtype, hq):
    """K and V of the drafted keys hold infinities and NaN; rows that do not see
    such a key are what they are with ordinary numbers there, rows that see it
    follow the sum."""
    import torch
    from probjax_amd.attention import tree_attention

    dt = _types()[dtype]
    B, T, S, Hq, Hkv, D = 2, 20, 400, hq, 2, 128
    (q, k, v), _ = _inputs(6, dt, B, T, S, Hq, Hkv, D, device)
    parents = torch.from_numpy(random_parents(np.random.default_rng(2), 1, T)[0]).to(device)
    L = torch.tensor([370, 100], dtype=torch.int32, device=device)
    scale = 0.09
    clean = tree_attention(q, k, v, parents=parents, kv_lengths=L, sm_scale=scale)
    sees, _ = ref.tree_sees(parents.tolist())
    bad_v, bad_k = 7, 11
    k2, v2 = k.clone(), v.clone()
    for b in range(B):
        P = int(L[b])
        v2[b, P + bad_v, :, 3] = float("inf")
        v2[b, P + bad_v, :, 70] = float("nan")
        k2[b, P + bad_k] = float("nan")
        k2[b, P + T:] = float("nan")  # behind the draft: never read
        v2[b, P + T:] = float("nan")
    got = tree_attention(q, k2, v2, parents=parents, kv_lengths=L, sm_scale=scale)
    torch.cuda.synchronize()
    for t in range(T):
        if sees[t, bad_k]:
            assert torch.isnan(got[:, t]).all(), t
        elif sees[t, bad_v]:
            assert torch.isposinf(got[:, t, :, 3]).all() and torch.isnan(got[:, t, :, 70]).all(), t
            rest = [d for d in range(D) if d not in (3, 70)]
            assert torch.equal(got[:, t][..., rest], clean[:, t][..., rest]), t
        else:
            assert torch.equal(got[:, t], clean[:, t]), t
    assert sees[:, bad_k].any() and (sees[:, bad_v] & ~sees[:, bad_k]).any() and (~sees[:, bad_v] & ~sees[:, bad_k]).any()


def test_caches_in_any_order_of_axes(device):
    """Caches that lie as [B, H, S, D], a slice of longer ones and a shared one
    give what contiguous copies give, and are read in place."""
    import torch
    from probjax_amd.attention import tree_attention

    B, T, S, Hq, Hkv, D = 2, 9, 300, 8, 2, 128
    (q, k, v), _ = _inputs(7, torch.bfloat16, B, T, S, Hq, Hkv, D, device)
    parents = torch.from_numpy(random_parents(np.random.default_rng(3), 1, T)[0]).to(device)
    L = torch.tensor([280, 31], dtype=torch.int32, device=device)
    want = tree_attention(q, k, v, parents=parents, kv_lengths=L)
    kt, vt = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    long_k = torch.full((B, 2 * S, Hkv, D), float("nan"), dtype=torch.bfloat16, device=device)
    long_k[:, :S] = k
    odd = torch.empty((B, S, Hkv, D + 3), dtype=torch.bfloat16, device=device)[..., :D].copy_(v)  # rows off 16 bytes
    for kk, vv in ((kt, vt), (long_k[:, :S], v), (k, odd), (kt, v)):
        got = tree_attention(q, kk, vv, parents=parents.long(), kv_lengths=L.long())
        assert torch.equal(got, want)
    shared_k, shared_v = k[:1].expand(B, S, Hkv, D), v[:1].expand(B, S, Hkv, D)
    got = tree_attention(q, shared_k, shared_v, parents=parents, kv_lengths=L)
    assert torch.equal(got, tree_attention(q, shared_k.contiguous(), shared_v.contiguous(), parents=parents, kv_lengths=L))
    qt = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    assert torch.equal(tree_attention(qt, k, v, parents=parents, kv_lengths=L), want)


def test_slots_far_apart_in_memory(device):
    """A cache whose slots lie 2^24 + 8 elements apart (a slice of a much longer
    row), with more rows per KV head than one 16-row block twice: offsets of a tile
    of keys pass 32 bits."""
    import torch

    B, T, S, Hq, Hkv, D, step = 1, 12, 150, 4, 1, 64, 2 ** 24 + 8
    (q, k, v), (qn, kn, vn) = _inputs(31, torch.bfloat16, B, T, S, Hq, Hkv, D, device)
    far = torch.empty((S * step,), dtype=torch.bfloat16, device=device).as_strided((B, S, Hkv, D), (0, step, D, 1))
    far.copy_(k)
    parents = random_parents(np.random.default_rng(31), B, T)
    from probjax_amd.hip_attention import tree_decode

    sees, token = ref.tree_sees(parents[0])
    want = ref.tree_attention(qn, kn, vn, [S - T], [sees], [token], D ** -0.5)
    out, lse = tree_decode(q, far, v, parents=torch.from_numpy(parents).to(device), sm_scale=D ** -0.5, return_lse=True)
    check(out, lse, want, torch.bfloat16, D, S)


def test_without_lengths_the_draft_is_the_cache_end(device):
    import torch
    from probjax_amd.attention import tree_attention

    B, T, S = 2, 5, 150
    (q, k, v), _ = _inputs(8, torch.float16, B, T, S, 4, 2, 64, device)
    parents = [-1, 0, 0, 1, 2]
    L = torch.full((B,), S - T, dtype=torch.int32, device=device)
    assert torch.equal(tree_attention(q, k, v, parents=parents), tree_attention(q, k, v, parents=parents, kv_lengths=L))


def test_a_chain_is_causal_attention(device):
    """A draft that is one chain gives what causal attention gives its last rows."""
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import mha, tree_attention

    B, T, S, D = 1, 11, 200, 64
    (q, k, v), _ = _inputs(9, torch.float32, B, T, S, 4, 4, D, device)
    got = tree_attention(q, k, v, parents=list(range(-1, T - 1)), sm_scale=0.125)
    want = mha(q, k, v, mask=masks.CausalFromBottomRightMask(T, S), sm_scale=0.125)
    # two float32 orders of the same sums: each within (2 D reach + S + 16) 2^-24 of the exact output
    assert float((got - want).abs().max()) <= 2 * (2 * D * 10 + S + 16) * 2.0 ** -24 * float(v.abs().max())


def test_replayed_graph_and_other_streams(device):
    """A captured call replayed on new inputs, and calls on two streams at once."""
    import torch
    from probjax_amd.attention import tree_attention

    B, T, S = 3, 16, 900
    (q, k, v), _ = _inputs(10, torch.bfloat16, B, T, S, 8, 2, 128, device)
    parents = torch.from_numpy(random_parents(np.random.default_rng(4), B, T)).to(device)
    L = torch.tensor([800, 3, 450], dtype=torch.int32, device=device)

    def step():
        return tree_attention(q, k, v, parents=parents, kv_lengths=L)

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        torch.manual_seed(i)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, device=device))
        L.copy_(torch.tensor([800 - 100 * i, 3 + i, 450 + i], device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step()), i
    want = step()
    outs = []
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_rejects(device):
    import torch
    from probjax_amd.attention import tree_attention

    q = torch.zeros((2, 4, 4, 64), dtype=torch.bfloat16, device=device)
    k = torch.zeros((2, 50, 2, 64), dtype=torch.bfloat16, device=device)
    parents = torch.tensor([-1, 0, 1, 1], dtype=torch.int32, device=device)
    ok = dict(parents=parents)
    tree_attention(q, k, k, **ok)
    bad = [
        (lambda: tree_attention(q, k, k), "parents or tree_mask"),
        (lambda: tree_attention(q, k, k, parents=parents, tree_mask=torch.ones((4, 4), dtype=torch.bool)), "not both"),
        (lambda: tree_attention(q, k, k, parents=parents[:3]), "shape"),
        (lambda: tree_attention(q, k, k, parents=parents.float()), "integers"),
        (lambda: tree_attention(q, k, k, tree_mask=torch.ones((4, 5), dtype=torch.bool)), "shape"),
        (lambda: tree_attention(q, k, k, tree_mask=torch.ones((4, 4))), "boolean"),
        (lambda: tree_attention(q, k, k, kv_lengths=[1, 2, 3], **ok), "kv_lengths"),
        (lambda: tree_attention(q, k[:, :3], k[:, :3], **ok), "does not hold"),
        (lambda: tree_attention(q, k.float(), k, **ok), "one dtype"),
        (lambda: tree_attention(q, k, k[:, :49], **ok), "incompatible"),
        (lambda: tree_attention(q, k[:1], k[:1], **ok), "incompatible"),
        (lambda: tree_attention(q[:, :, :3], k, k, **ok), "incompatible"),
        (lambda: tree_attention(q[0], k, k, **ok), "must be"),
        (lambda: tree_attention(q.cpu(), k, k, **ok), "ROCm device"),
        (lambda: tree_attention(q, k, k, sm_scale=0.0, **ok), "sm_scale"),
        (lambda: tree_attention(q.clone().requires_grad_(), k, k, **ok), "no gradient"),
        (lambda: tree_attention(q.new_zeros((2, 300, 4, 64)), k, k, parents=[-1] * 300), "256"),
        (lambda: tree_attention(q.new_zeros((2, 4, 4, 300)), k.new_zeros((2, 9, 2, 300)), k.new_zeros((2, 9, 2, 300)),
                                **ok), "head dims"),
    ]
    for call, msg in bad:
        with pytest.raises(ValueError, match=msg):
            call()
    with torch.no_grad():
        tree_attention(q.clone().requires_grad_(), k, k, **ok)
    assert tree_attention(q[:0], k[:0], k[:0], **ok).shape == (0, 4, 4, 64)
    empty = tree_attention(q, k[:, :0], k[:, :0], kv_lengths=[0, 0], return_lse=True, **ok)
    assert torch.equal(empty[0], torch.zeros_like(q)) and torch.isposinf(empty[1]).all()
