"""A serving loop that evicts into two spare caches by turns.  Eviction leaves what
a given buffer holds behind the kept keys, so the spares hold the keys and weights
of earlier turns there; keys appended to them start from a weight of zero because
the loop zeroes those weights, as ``evict_keys`` documents."""

import math

import numpy as np
import pytest

from oracle import cache_ops as ref
from tests._helpers import to_np
from tests.test_gpu_key_weights import check_weights
from tests.test_gpu_tree_attention import _types

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_spares_by_turns(device, name):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights, evict_keys

    B, Hq, Hkv, D, keep, steps, room = 2, 4, 2, 64, 24, 5, 40
    dtype, scale = _types()[name], 1.0 / math.sqrt(D)
    g = torch.Generator(device=device).manual_seed(1)

    def new(T, H):
        return torch.randn((B, T, H, D), generator=g, device=device).to(dtype)

    spares = []
    for _ in range(2):
        k, v = (torch.full((B, room, Hkv, D), 3.0, dtype=dtype, device=device) for _ in range(2))
        spares.append((k, v, torch.full((B, Hkv, room), 100.0, device=device)))
    slots = torch.arange(room, device=device)
    k, v = new(room, Hkv), new(room, Hkv)
    w = torch.rand((B, Hkv, room), generator=g, device=device)
    L = torch.tensor([room, 20], dtype=torch.int32, device=device)
    at = torch.arange(B, device=device)
    for turn in range(4):
        kept = evict_keys(k, v, w, keep, kv_lengths=L, sinks=2, recent=4, out=spares[turn % 2])
        kept.key_weights.masked_fill_(slots >= kept.kv_lengths[:, None, None], 0)
        k, v, w, L = kept[:4]
        # what the keys appended in this turn were given, and the steps' errors (check_weights) added up
        start, sums, tol = L.clone(), np.zeros((B, Hkv, room)), np.zeros((B, Hkv, room))
        for _ in range(steps):
            k[at, L.long()], v[at, L.long()] = new(1, Hkv)[:, 0], new(1, Hkv)[:, 0]
            L = L + 1
            q = new(1, Hq)
            base = to_np(w).astype(np.float64)
            _, w = attention_with_key_weights(q, k, v, w, mask=masks.KVLenMask(L))
            see = np.arange(room)[None, None, :] < to_np(L)[:, None, None]
            want = ref.key_weight_attention(*(to_np(x).astype(np.float64) for x in (q, k, v)), base, see, scale)
            check_weights(w, want, base, D, room, Hq // Hkv)
            sums += want["weights"] - base
            lse = np.where(np.isfinite(want["lse"]), np.abs(want["lse"]), 0.0)
            tol += (2 * D * want["reach"] + room + 24 + 8 * lse).max() * 2.0 ** -24 * (want["weights"] - base)
            tol += (Hq // Hkv + 2) * 2.0 ** -24 * np.abs(want["weights"])
        for b in range(B):
            fresh = slice(int(start[b]), int(L[b]))
            # the sums of the steps alone, whatever lay there before
            assert (np.abs(to_np(w)[b, :, fresh] - sums[b, :, fresh]) <= tol[b, :, fresh]).all(), (turn, b)


@pytest.mark.parametrize("axis", [0, 2, 3])
def test_buffers_and_inputs_of_one_allocation(device, axis):
    """K and V of one tensor, whose spare slots take what is kept of the others."""
    import torch
    from probjax_amd.attention import evict_keys

    B, S, H, D, keep, room = 2, 300, 2, 64, 50, 70
    shape = [B, S + room, H, D]
    pool = torch.randn((*shape[:axis], 2, *shape[axis:]), generator=torch.Generator(device=device).manual_seed(2),
                       device=device).to(torch.bfloat16)
    k, v = pool.select(axis, 0), pool.select(axis, 1)
    w = torch.rand((B, H, S), device=device)
    L = torch.tensor([300, 45], dtype=torch.int32, device=device)
    want = evict_keys(k[:, :S].clone(), v[:, :S].clone(), w, keep, kv_lengths=L, recent=3)
    before = pool.clone()
    out = (k[:, S:], v[:, S:], torch.zeros((B, H, room), device=device))
    got = evict_keys(k[:, :S], v[:, :S], w, keep, kv_lengths=L, recent=3, out=out)
    torch.cuda.synchronize()
    assert torch.equal(got.index, want.index) and torch.equal(got.kv_lengths, want.kv_lengths)
    for x, y, z in ((k, got.k, want.k), (v, got.v, want.v)):
        assert y.data_ptr() == x[:, S:].data_ptr()
        for b, n in enumerate((50, 45)):
            assert torch.equal(y[b, :n], z[b, :n])
            y[b, :n] = before.select(axis, 0 if x is k else 1)[b, S:S + n]
    assert torch.equal(pool, before)  # nothing else was written
