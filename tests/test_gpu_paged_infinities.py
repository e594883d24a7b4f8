"""Infinities that a row sees, in a paged cache of floats: an infinite value makes its
feature infinite (both signs of it: NaN) in every row that sees it and in no other, a key
whose score is -inf has no weight.  In steps that every row sees whole and in the last,
ragged one; in sequences of one workgroup and in those that are cut into shares.

The features beside the infinite ones are held to the definition by the bound of
``test_gpu_paged_decode``: their sums may be taken in another order, not less exactly."""

import math

import numpy as np
import pytest

from oracle import paged as ref
from tests._helpers import to_np
from tests.test_gpu_paged_cache import make_cache, make_table, types
from tests.test_gpu_paged_decode import check, gathered

pytestmark = pytest.mark.gpu

CASES = [
    # type, T, Hq, Hkv, D, page, keys
    ("bf16", 1, 4, 2, 64, 16, 300),
    ("f16", 1, 4, 2, 64, 16, 300),
    ("f32", 1, 4, 2, 64, 16, 300),
    ("bf16", 1, 4, 2, 128, 16, 2500),
    ("f16", 1, 4, 2, 128, 16, 2500),
    ("f32", 1, 4, 2, 128, 16, 2500),
    ("bf16", 4, 4, 2, 64, 5, 2500),
    ("f16", 4, 4, 2, 80, 7, 300),
    ("f16", 5, 8, 2, 64, 16, 2500),   # two blocks of rows
    ("bf16", 20, 2, 1, 128, 16, 700),
    ("f16", 1, 4, 2, 256, 16, 100),
    ("bf16", 1, 4, 2, 192, 16, 2500),
]


def make(device, name, T, Hq, Hkv, D, page, keys, seed):
    import torch

    B, N, dtype = 2, -(-keys // page), types()[name]
    rng = np.random.default_rng(seed)
    lengths = [keys, keys // 2 + 5]
    table = make_table(rng, B, N, B * N, lengths, page)
    cache = make_cache(device, rng, name, B * N, page, Hkv, D, table)
    q = torch.from_numpy(rng.standard_normal((B, T, Hq, D), dtype=np.float32)).to(device, dtype)
    return cache, table, lengths, q, dtype


def attend(device, q, cache, lengths):
    import torch
    from probjax_amd.attention import paged_decode

    out, lse = paged_decode(q, cache, kv_lengths=torch.tensor(lengths, dtype=torch.int32, device=device), return_lse=True)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_values(device, case):
    import torch

    name, T, Hq, Hkv, D, page, keys = case
    cache, table, lengths, q, dtype = make(device, *case, seed=keys + D)
    clean, clean_lse = attend(device, q, cache, lengths)
    k, v, there = gathered(cache, table, lengths)
    want = ref.paged_decode(to_np(q), k, v, there, lengths, 1.0 / math.sqrt(D))
    check(clean, clean_lse, want, dtype, D, k.shape[1])
    # (sequence, key, feature, sign): a whole step, the last key of all, both signs of one feature
    places = [(0, 40, 3, 1), (0, 41, D - 1, -1), (0, keys - 1, 1, -1), (1, 37, 5, 1), (1, lengths[1] - 1, 5, -1),
              (1, 29, 2, -1)]
    for b, key, d, sign in places:
        p, s = ref.slots(table, page, len(cache.k), b, key)
        cache.v[int(p), int(s), :, d] = sign * math.inf
    out, lse = attend(device, q, cache, lengths)
    assert torch.equal(lse, clean_lse)
    out = to_np(out)
    spoilt = np.zeros(out.shape, bool)
    for t in range(T):
        seen = {}
        for b, key, d, sign in places:
            if key < lengths[b] - (T - 1 - t):
                seen.setdefault((b, d), []).append(sign)
        for (b, d), signs in seen.items():
            spoilt[b, t, :, d] = True
            got = out[b, t, :, d]
            assert (np.isnan(got) if len(signs) > 1 else got == signs[0] * np.inf).all(), (b, t, d, got)
    rest = {n: x if n in ("lse", "reach") else np.where(spoilt, 0.0, x) for n, x in want.items()}
    check(torch.from_numpy(np.where(spoilt, 0.0, out)), lse, rest, dtype, D, k.shape[1])


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_keys_of_no_weight(device, case):
    """A key with a score of -inf: as if it were not there, its infinite value aside
    (0 * inf is NaN by the definition, so its value stays finite here)."""
    name, T, Hq, Hkv, D, page, keys = case
    cache, table, lengths, q, dtype = make(device, *case, seed=keys + D + 1)
    q[..., 3] = q[..., 3].abs() + 0.5
    k, v, there = gathered(cache, table, lengths)
    there = there.copy()
    for b, key in ((0, 0), (0, 45), (0, keys - 1), (1, 33), (1, lengths[1] - 1)):
        p, s = ref.slots(table, page, len(cache.k), b, key)
        cache.k[int(p), int(s), :, 3] = -math.inf
        there[b, key] = False
    out, lse = attend(device, q, cache, lengths)
    want = ref.paged_decode(to_np(q), k, v, there, lengths, 1.0 / math.sqrt(D))
    check(out, lse, want, dtype, D, k.shape[1])
