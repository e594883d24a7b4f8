"""Pinning of the oracle of the operators over a KV cache (oracle/cache_ops.py)
against torch's attention and sort on the CPU, closed forms, and the oracle's
own rotary encoding and attention."""

import numpy as np
import pytest

import oracle
from oracle import cache_ops as ref


def test_tree_sees():
    sees, token = ref.tree_sees([-1, 0, 0, 1, -1, 4, 9, -2])
    want = np.array([
        [1, 0, 0, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0, 0, 0], [1, 0, 1, 0, 0, 0, 0, 0], [1, 1, 0, 1, 0, 0, 0, 0],
        [0, 0, 0, 0, 1, 0, 0, 0], [0, 0, 0, 0, 1, 1, 0, 0], [0, 0, 0, 0, 0, 0, 1, 0], [0, 0, 0, 0, 0, 0, 0, 1]], bool)
    np.testing.assert_array_equal(sees, want)
    np.testing.assert_array_equal(token, [True] * 7 + [False])


@pytest.mark.parametrize("lengths", [[40, 13], [0, 60], [-3, 43]])
def test_tree_attention_against_torch(lengths):
    import torch

    rng = np.random.default_rng(0)
    B, T, S, Hq, Hkv, D = 2, 6, 43, 4, 2, 8
    q, k, v = (rng.standard_normal(s) for s in ((B, T, Hq, D), (B, S, Hkv, D), (B, S, Hkv, D)))
    sees, token = ref.tree_sees([-1, 0, 0, 1, -1, -2])
    r = ref.tree_attention(q, k, v, lengths, [sees] * B, [token] * B, 0.3)
    for b in range(B):
        P = min(max(lengths[b], 0), S)
        keep = torch.zeros((T, S), dtype=torch.bool)
        keep[:, :P] = True
        n = min(T, S - P)
        keep[:, P:P + n] = torch.from_numpy(sees[:, :n])
        keep[5] = False
        x, y, z = (torch.from_numpy(a[b]).transpose(0, 1) for a in (q, k, v))
        want = torch.nn.functional.scaled_dot_product_attention(x, y, z, attn_mask=keep, scale=0.3, enable_gqa=True)
        want = torch.nan_to_num(want).transpose(0, 1).numpy()
        np.testing.assert_allclose(r["out"][b], want, atol=1e-12)
        np.testing.assert_array_equal(np.isinf(r["lse"][b]), np.broadcast_to(~keep.any(1).numpy(), (Hq, T)))
    assert not r["out"][:, 5].any()


def test_key_weights_are_column_sums_of_the_softmax():
    rng = np.random.default_rng(1)
    B, T, S, Hq, Hkv, D = 2, 5, 9, 4, 2, 8
    q, k, v = (rng.standard_normal(s) for s in ((B, T, Hq, D), (B, S, Hkv, D), (B, S, Hkv, D)))
    keep = np.broadcast_to(np.tril(np.ones((T, S), bool), 2), (B, T, S))
    r = ref.key_weight_attention(q, k, v, np.ones((B, Hkv, S)), keep, 0.4)
    s = 0.4 * np.einsum("bthd,bshd->bhts", q, np.repeat(k, Hq // Hkv, 2))
    p = np.exp(np.where(keep[:, None], s, -np.inf))
    p /= p.sum(-1, keepdims=True)
    np.testing.assert_allclose(r["weights"], 1 + p.reshape(B, Hkv, 2, T, S).sum((2, 3)), rtol=1e-12)
    np.testing.assert_allclose((r["weights"] - 1).sum(-1), np.full((B, Hkv), 2 * T), rtol=1e-12)
    want, lse = oracle.xla_attention(*(a.astype(np.float32) for a in (q, k, v)), sm_scale=0.4, return_lse=True)
    full = ref.key_weight_attention(q, k, v, np.zeros((B, Hkv, S)), np.ones((B, T, S), bool), 0.4)
    np.testing.assert_allclose(full["out"], want, atol=1e-5)
    np.testing.assert_allclose(full["lse"], lse, atol=1e-5)


def test_evict():
    w = np.array([5, 1, 1, 3, 0, 1, 2, 9], np.float32)
    assert ref.evict(w, 8, 8) == list(range(8)) and ref.evict(w, 3, 5) == [0, 1, 2]
    assert ref.evict(w, 8, 3) == [0, 3, 7]
    assert ref.evict(w, 8, 5) == [0, 1, 3, 6, 7]  # of equal ones the first
    assert ref.evict(w, 8, 4, sinks=2, recent=1) == [0, 1, 3, 7]
    assert ref.evict(w, 6, 3, recent=2) == [0, 4, 5]
    assert ref.evict(np.array([1, np.nan, -0.0, 0.0, np.inf], np.float32), 5, 2) == [1, 4]
    assert ref.evict(np.array([-1, -0.0, 0.0], np.float32), 3, 1) == [1]
    import torch

    x = np.random.default_rng(0).integers(0, 6, 200).astype(np.float32)
    order = torch.sort(torch.from_numpy(x), descending=True, stable=True).indices[:70]
    assert ref.evict(x, 200, 70) == sorted(order.tolist())


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("shared", [True, False])
def test_rotary(interleaved, shared):
    rng = np.random.default_rng(2)
    x, y = rng.standard_normal((2, 1, 5, 2, 24))
    pos = rng.integers(0, 50, (1, 5, 3))
    rule = dict(interleaved=interleaved, shared_spectrum=shared)
    r = ref.rotary(x, pos, (8, 4, 10), **rule)
    np.testing.assert_allclose(np.linalg.norm(r, axis=-1), np.linalg.norm(x, axis=-1))  # norms stay
    np.testing.assert_array_equal(r[..., 22:], x[..., 22:])  # the rest passes
    np.testing.assert_allclose(ref.rotary(r, pos, (8, 4, 10), sign=-1, **rule), x, atol=1e-12)  # and back
    # only the difference of two positions counts
    a = ref.rotary(x, pos + 7, (8, 4, 10), **rule), ref.rotary(y, pos[:, ::-1] + 7, (8, 4, 10), **rule)
    b = ref.rotary(x, pos, (8, 4, 10), **rule), ref.rotary(y, pos[:, ::-1], (8, 4, 10), **rule)
    np.testing.assert_allclose((a[0] * a[1]).sum(-1), (b[0] * b[1]).sum(-1), atol=1e-10)
    # one axis: the reference's own; the spectrum is shared with itself
    one = ref.rotary(x, pos[..., :1], (24,), **rule)
    if interleaved:
        np.testing.assert_allclose(one, oracle.apply_rotary(x[0], pos[0, :, 0])[None], atol=1e-4)
    else:  # the same pairs, in another order of features
        order = np.arange(24).reshape(2, 12).T.reshape(-1)
        np.testing.assert_allclose(one[..., order], ref.rotary(x[..., order], pos[..., :1], (24,)), atol=1e-12)
