"""Attention sinks over a paged cache: one key takes nearly all of the weight and has a
value of 0, so that the output is made of weights far below the largest.

Held to the definition by the bound of ``test_gpu_paged_decode``, which is relative to
``sum p |v|`` of the small weights themselves: a weight may be rounded, not lost.  (What a
weight loses where the type's numbers end must stay below half a step of the output's
smallest ones, 2^-25 in fp16, which that bound allows for.)"""

import math

import numpy as np
import pytest

from oracle import paged as ref
from tests._helpers import to_np
from tests.test_gpu_paged_cache import make_cache, make_table, types
from tests.test_gpu_paged_decode import check, gathered

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nats,size", [(8, 1.0), (14, 1.0), (16, 1.0), (17.5, 1.0), (17.5, 300.0), (21, 1000.0), (27, 30000.0)])
@pytest.mark.parametrize("name,held,T,Hq,Hkv,D,page,keys", [
    ("f16", "f16", 1, 4, 2, 64, 16, 300),
    ("f16", "f16", 1, 4, 2, 128, 16, 9000),
    ("f16", "f16", 1, 6, 3, 80, 20, 2500),
    ("f16", "f16", 5, 8, 2, 128, 16, 2500),  # two blocks of rows
    ("f16", "f16", 1, 4, 2, 256, 16, 2500),
    ("f16", "e4m3", 1, 4, 2, 128, 16, 2500),
    ("bf16", "bf16", 1, 4, 2, 128, 16, 2500),
    ("f32", "f32", 1, 4, 2, 64, 16, 2500),
])
def test_small_weights_are_kept(device, name, held, T, Hq, Hkv, D, page, keys, nats, size):
    """The sink at the first key, in the midst, and as the last key all tokens see; the
    other keys' scores within about a nat of each other, their values of one sign."""
    import torch
    from probjax_amd.attention import PagedCache, paged_decode, write_pages

    B, N, dtype = 3, -(-keys // page), types()[name]
    rng = np.random.default_rng(int(10 * nats) + D)
    lengths = [keys, keys - 3, keys - page]
    table = make_table(rng, B, N, B * N, lengths, page)
    scale = 1.0 / math.sqrt(D)
    q = rng.standard_normal((B, T, Hq, D), dtype=np.float32)
    q[..., 0] = 4.0
    k = (0.25 * rng.standard_normal((B, keys, Hkv, D))).astype(np.float32)
    k[..., 0] = 0.0
    v = (size * (1.0 + rng.random((B, keys, Hkv, D)))).astype(np.float32)
    for b, key in enumerate((0, keys // 2, lengths[2] - T)):
        k[b, key] = 0.0
        k[b, key, :, 0] = nats / (4.0 * scale)
        v[b, key] = 0.0
    q, k, v = (torch.from_numpy(x).to(device, dtype) for x in (q, k, v))
    pools = make_cache(device, rng, held, B * N, page, Hkv, D, table)
    cache = PagedCache(pools.k, pools.v, pools.page_table, pools.k_exponents, pools.v_exponents)
    L = write_pages(cache, k, v, new_lengths=torch.tensor(lengths, dtype=torch.int32, device=device))
    out, lse = paged_decode(q, cache, kv_lengths=L, sm_scale=scale, return_lse=True)
    torch.cuda.synchronize()
    keys_held, values, there = gathered(cache, table, lengths)
    want = ref.paged_decode(to_np(q), keys_held, values, there, lengths, scale)
    check(out, lse, want, dtype, D, keys_held.shape[1])
