"""Eviction from a KV cache: whole numbers and copies, so everything is equal to
the definition's (oracle/cache_ops.py) bit for bit."""

import numpy as np
import pytest

from oracle import cache_ops as ref
from tests.test_gpu_tree_attention import _types

pytestmark = pytest.mark.gpu


def _weights(rng, kind, shape):
    w = rng.standard_normal(shape).astype(np.float32)
    if kind == "sums":  # a few keys carry most, many equal zeros
        w = np.where(rng.random(shape) < 0.3, 0.0, np.exp(3 * w)).astype(np.float32)
    elif kind == "equal":
        w[:] = 0.25
    elif kind == "few":
        w = np.round(w).astype(np.float32)  # ties across the threshold, -0 among them
    elif kind == "odd":
        w[rng.random(shape) < 0.05] = np.nan
        w[rng.random(shape) < 0.05] = -np.nan
        w[rng.random(shape) < 0.05] = np.inf
        w[rng.random(shape) < 0.05] = -np.inf
        w[rng.random(shape) < 0.05] = -0.0
    elif kind == "near":  # neighbours of one value: the last bits decide
        w = (np.float32(1.0).view(np.uint32) + rng.integers(0, 40, shape).astype(np.uint32)).view(np.float32)
    return w


CASES = [
    # dtype, B, S, H, D, keep, sinks, recent, lengths, weights
    ("bf16", 3, 300, 2, 128, 100, 4, 16, [300, 100, 101], "sums"),
    ("bf16", 4, 70, 3, 64, 1, 0, 0, [0, 1, 2, 70], "normal"),
    ("f16", 2, 1500, 2, 80, 700, 0, 0, [1500, 1024], "few"),
    ("f32", 2, 1030, 1, 64, 1029, 1, 33, [1030, 1029], "equal"),
    ("bf16", 2, 2049, 2, 96, 512, 256, 256, [2049, 513], "normal"),  # nothing to choose between
    ("bf16", 2, 5000, 2, 64, 999, 0, 100, [5000, 4097], "odd"),
    ("bf16", 1, 8192, 1, 128, 4096, 4, 32, None, "near"),
    ("f32", 2, 9000, 1, 20, 3000, 3, 0, [9000, 8999], "sums"),       # more registers
    ("f16", 1, 33000, 1, 8, 16000, 4, 5, None, "few"),               # read again each round
    ("bf16", 2, 40000, 1, 64, 39000, 0, 1, [40000, 39500], "odd"),
    ("bf16", 2, 90, 2, 3, 30, 1, 1, [90, 60], "normal"),             # rows of 6 bytes
    ("f32", 2, 90, 2, 3, 30, 1, 1, [-5, 200], "normal"),             # lengths off the cache's ends
    ("bf16", 2, 50, 2, 64, 60, 2, 2, [50, 20], "normal"),            # room for all
]


def _check(got, k, v, w, case, filled=True):
    name, B, S, H, D, keep, sinks, recent, lengths, _ = case
    lengths = [S] * B if lengths is None else lengths
    index = got[4].cpu().numpy()
    at = np.full((B, H, keep), -1)
    for b in range(B):
        n = min(max(min(lengths[b], S), 0), keep)
        assert int(got[3][b]) == n
        for h in range(H):
            at[b, h, :n] = ref.evict(w[b, h], lengths[b], keep, sinks, recent)
            np.testing.assert_array_equal(index[b, h], at[b, h], err_msg=f"{case} {b} {h}")
            i = at[b, h, :n]
            for x, y in ((k, got[0]), (v, got[1])):
                assert np.array_equal(_bits(y[b, :n, h]), _bits(x[b, i, h])), (case, b, h)
                if filled:
                    assert not _bits(y[b, n:keep, h]).any()
            assert np.array_equal(_bits(got[2][b, h, :n]), w[b, h, i].view(np.int32))
            if filled:
                assert not _bits(got[2][b, h, n:keep]).any()


def _bits(x):
    import torch

    return x.contiguous().view(torch.int32 if x.element_size() == 4 else torch.int16).cpu().numpy()


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:8])) + "-" + c[-1])
def test_matches_definition(device, case):
    import torch
    from probjax_amd.attention import evict_keys

    name, B, S, H, D, keep, sinks, recent, lengths, kind = case
    rng = np.random.default_rng(S + keep)
    w = _weights(rng, kind, (B, H, S))
    g = torch.Generator(device=device).manual_seed(S)
    k, v = (torch.randn((B, S, H, D), generator=g, device=device).to(_types()[name]) for _ in range(2))
    k[0, S // 2:S // 2 + 1] = float("nan")  # copied as it is
    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    print(f"evict {case}", flush=True)
    got = evict_keys(k, v, torch.from_numpy(w).to(device), keep, kv_lengths=L, sinks=sinks, recent=recent)
    torch.cuda.synchronize()
    _check(got, k, v, w, case)


def test_into_given_buffers(device):
    """Rows behind the kept keys stay, and caches in any order of axes are read
    and written in place."""
    import torch
    from probjax_amd.attention import evict_keys

    case = ("bf16", 2, 300, 2, 64, 100, 4, 16, [300, 60], "sums")
    _, B, S, H, D, keep, sinks, recent, lengths, kind = case
    w = _weights(np.random.default_rng(0), kind, (B, H, S))
    g = torch.Generator(device=device).manual_seed(0)
    k, v = (torch.randn((B, S, H, D), generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    kt, vt = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    wd, L = torch.from_numpy(w).to(device), torch.tensor(lengths, device=device)
    C = 130
    for kk, vv, off in ((k, v, 0), (kt, vt, 0), (kt, v, 3)):
        # `off`: rows of 67 features, not whole 16-byte chunks
        ko = torch.full((B, H, C, D + off), 7.0, dtype=torch.bfloat16, device=device).permute(0, 2, 1, 3)[..., :D]
        vo = torch.full((B, C, H, D + off), 7.0, dtype=torch.bfloat16, device=device)[..., :D]
        wo = torch.full((B, H, C), 7.0, device=device)
        got = evict_keys(kk, vv, wd, keep, kv_lengths=L, sinks=sinks, recent=recent, out=(ko, vo, wo))
        assert got.k is ko and got.v is vo and got.key_weights is wo
        _check(got, k, v, w, case, filled=False)
        for b, n in enumerate((100, 60)):
            assert (ko[b, n:] == 7).all() and (vo[b, n:] == 7).all() and (wo[b, :, n:] == 7).all()


def test_replayed_graph(device):
    import torch
    from probjax_amd.attention import evict_keys

    k, v = (torch.randn((2, 500, 2, 64), device=device) for _ in range(2))
    w, L = torch.rand((2, 2, 500), device=device), torch.tensor([500, 300], dtype=torch.int32, device=device)

    def step():
        return evict_keys(k, v, w, 200, kv_lengths=L, sinks=2, recent=10)

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
        for x in (k, v, w):
            x.copy_(torch.rand(x.shape, device=device))
        L.copy_(torch.tensor([500 - 80 * i, 190 + i], device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step())), i


def test_rejects(device):
    import torch
    from probjax_amd.attention import evict_keys as f

    k = torch.zeros((2, 50, 2, 64), dtype=torch.bfloat16, device=device)
    w = torch.zeros((2, 2, 50), device=device)
    room = [torch.zeros((2, 20, 2, 64), dtype=torch.bfloat16, device=device) for _ in range(2)]
    room.append(torch.zeros((2, 2, 20), device=device))
    f(k, k, w, 10, out=tuple(room))
    bad = [
        (lambda: f(k, k, w, 0), "keep"),
        (lambda: f(k, k, w, 10, sinks=6, recent=5), "sinks"),
        (lambda: f(k, k, w, 10, sinks=-1), "sinks"),
        (lambda: f(k, k[:, :49], w, 10), "one shape"),
        (lambda: f(k, k.float(), w, 10), "dtype"),
        (lambda: f(k.int(), k.int(), w, 10), "dtype"),
        (lambda: f(k, k, w[:1], 10), "shape"),
        (lambda: f(k, k, w.double(), 10), "float32"),
        (lambda: f(k, k, w, 10, kv_lengths=[1, 2, 3]), "kv_lengths"),
        (lambda: f(k, k, w, 10, kv_lengths=torch.ones(2, device=device)), "integers"),
        (lambda: f(k, k, w, 21, out=tuple(room)), "out must"),
        (lambda: f(k, k, w, 10, out=(room[0], room[0], room[2])), "share memory"),
        (lambda: f(k, k, w, 10, out=(k, room[1], room[2])), "out must|share memory"),
        (lambda: f(room[0], room[1], w[:, :, :20].contiguous(), 10, out=(k[:, :20], room[1], room[2])), "share memory"),
        (lambda: f(k.clone().requires_grad_(), k, w, 10), "no gradient"),
        (lambda: f(k.cpu(), k, w, 10), "ROCm device"),
    ]
    for call, msg in bad:
        with pytest.raises(ValueError, match=msg):
            call()
    got = f(k[:, :0], k[:, :0], w[:, :, :0], 5)
    assert (got.index == -1).all() and (got.kv_lengths == 0).all() and not got.k.any()
    assert f(k[:0], k[:0], w[:0], 5).k.shape == (0, 5, 2, 64)
