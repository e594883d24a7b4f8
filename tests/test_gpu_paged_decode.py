"""Attention over a paged cache against its definition in float64.

Tolerances are those of ``test_gpu_tree_attention``: a rounding of every weight and of
the output to the type (u, half a step), float32 sums.  Over 8 bits the oracle gets the
values that the codes stand for, so the bounds are the same.  An output below the type's
smallest normal number has even steps there, so its rounding is off by up to half of one
(fp16: 2^-25, more than u |o| below 2^-14), which is added."""

import math

import numpy as np
import pytest

from oracle import paged as ref
from tests._helpers import to_np
from tests.test_gpu_paged_cache import host_rows, make_cache, make_table, types

pytestmark = pytest.mark.gpu


def check(got, lse, want, dtype, D, n):
    import torch

    info = torch.finfo(dtype)
    u = 0.0 if dtype == torch.float32 else info.eps / 2
    rel = (2 * D * want["reach"] + n + 16) * 2.0 ** -24  # [B, Hq, T]
    rel = np.moveaxis(rel, 1, 2)[..., None]
    tol = u * (1 + rel) * (want["spread"] + np.abs(want["out"])) + rel * want["spread"] + 2.0 ** -24 * np.abs(want["out"])
    tol = tol + info.smallest_normal * info.eps / 2
    err = np.abs(to_np(got) - want["out"])
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])
    lse, fin = to_np(lse), np.isfinite(want["lse"])
    np.testing.assert_array_equal(np.isposinf(lse), ~fin)
    off = np.abs(lse[fin] - want["lse"][fin])
    lim = (D * want["reach"][fin] + n + 16 + 4 * np.abs(want["lse"][fin])) * 2.0 ** -24
    assert (off <= lim).all(), (off.max(), lim.min())


def gathered(cache, table, lengths):
    B, N = table.shape
    S = N * cache.page_size
    k, there = ref.gather(host_rows(cache, 0), table, [S] * B, S)
    v, _ = ref.gather(host_rows(cache, 1), table, [S] * B, S)
    return k, v, there


def run(device, cache, table, lengths, q, dtype, what=""):
    import torch
    from probjax_amd.attention import paged_decode

    L = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    print(what, flush=True)
    got, lse = paged_decode(q, cache, kv_lengths=L, return_lse=True)
    torch.cuda.synchronize()
    k, v, there = gathered(cache, table, lengths)
    S, D = k.shape[1], q.shape[-1]
    want = ref.paged_decode(to_np(q), k, v, there, [S] * len(k) if lengths is None else lengths, 1.0 / math.sqrt(D))
    check(got, lse, want, dtype, D, S)
    return got, lse


CASES = [
    # type, cache, B, T, Hq, Hkv, D, page, room (pages), layout
    ("bf16", "bf16", 2, 1, 8, 2, 128, 16, 20, "tokens"),
    ("bf16", "e4m3", 2, 1, 8, 2, 128, 16, 20, "tokens"),
    ("bf16", "bf16", 3, 1, 4, 4, 64, 32, 9, "heads"),
    ("bf16", "e4m3", 3, 1, 4, 4, 64, 32, 9, "heads"),
    ("f16", "f16", 2, 1, 32, 2, 128, 64, 5, "tokens"),
    ("f16", "e4m3", 2, 1, 32, 2, 128, 64, 5, "heads"),
    ("f16", "f16", 2, 1, 6, 3, 80, 20, 17, "tokens"),
    ("f16", "e4m3", 2, 1, 6, 3, 80, 20, 17, "tokens"),
    ("bf16", "bf16", 1, 1, 7, 1, 96, 100, 3, "tokens"),
    ("bf16", "e4m3", 1, 1, 7, 1, 112, 1, 150, "heads"),
    ("bf16", "bf16", 2, 1, 4, 2, 256, 16, 10, "tokens"),
    ("bf16", "e4m3", 2, 1, 4, 2, 256, 8, 20, "tokens"),
    ("bf16", "bf16", 2, 1, 4, 2, 192, 48, 4, "heads"),
    ("bf16", "e4m3", 2, 1, 4, 2, 192, 256, 2, "tokens"),
    ("bf16", "bf16", 2, 1, 3, 1, 8, 3, 50, "tokens"),
    ("bf16", "e4m3", 2, 1, 3, 1, 16, 5, 30, "tokens"),
    ("f32", "f32", 2, 1, 4, 4, 64, 16, 12, "tokens"),
    ("f32", "e4m3", 2, 1, 4, 4, 64, 16, 12, "tokens"),
    ("f32", "f32", 2, 1, 8, 2, 128, 32, 6, "heads"),
    ("f32", "e4m3", 2, 1, 8, 2, 128, 10, 20, "heads"),
    ("f32", "f32", 1, 1, 2, 1, 256, 64, 3, "tokens"),
    ("f32", "e4m3", 1, 1, 2, 1, 256, 64, 3, "tokens"),
    ("f32", "f32", 2, 1, 3, 3, 20, 7, 20, "tokens"),
    ("bf16", "bf16", 2, 5, 8, 2, 128, 16, 20, "tokens"),
    ("f16", "e4m3", 2, 5, 8, 2, 128, 16, 20, "tokens"),
    ("bf16", "e4m3", 2, 8, 16, 2, 64, 32, 10, "tokens"),   # 64 rows
    ("bf16", "bf16", 2, 17, 16, 2, 128, 32, 10, "heads"),  # 136 rows
    ("f32", "f32", 2, 9, 8, 2, 64, 16, 20, "tokens"),      # 36 rows
    ("f32", "e4m3", 2, 3, 4, 2, 256, 16, 9, "tokens"),
    ("bf16", "bf16", 2, 40, 4, 2, 80, 20, 15, "tokens"),
    ("bf16", "e4m3", 1, 1, 128, 1, 64, 64, 4, "tokens"),   # 128 rows of one head
]


@pytest.mark.parametrize("times", [1, 12])  # sequences short enough for a workgroup each, and cut into shares
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_matches_definition(device, case, times):
    import torch
    from probjax_amd import native

    name, held, B, T, Hq, Hkv, D, page, N, layout = case
    N *= times
    rng = np.random.default_rng(D + page + T)
    S, dtype = N * page, types()[name]
    pages = B * N + 1
    lengths = [S] + [int(x) for x in rng.integers(0, S + 1, B - 1)]
    table = make_table(rng, B, N, pages, lengths, page)
    cache = make_cache(device, rng, held, pages, page, Hkv, D, table, layout, spread=3)
    q = torch.from_numpy(rng.standard_normal((B, T, Hq, D), dtype=np.float32)).to(device, dtype)
    run(device, cache, table, lengths, q, dtype, "full and random lengths")
    width = 64 if D <= 64 else 128 if D <= 128 else 256
    whole = S * 2 * width * cache.k.element_size() <= 128 << 10
    assert len(native.last_launches()) == (1 if whole else 2), native.last_launches()
    run(device, cache, table, [max(S - 1, 0)] + [min(T, S)] * (B - 1), q, dtype, "as many keys as tokens")
    run(device, cache, table, [1] + [0] * (B - 1), q, dtype, "one key, none")
    run(device, cache, table, [S + 100] + [-5] * (B - 1), q, dtype, "past the capacity, negative")
    run(device, cache, table, None, q, dtype, "without lengths")


@pytest.mark.parametrize("name,held", [("bf16", "bf16"), ("f16", "e4m3"), ("f32", "f32"), ("bf16", "e4m3"), ("f32", "e4m3")])
@pytest.mark.parametrize("B,S", [(1, 5000), (5, 1100), (300, 40), (70, 300), (64, 2100), (65, 2100), (130, 2500), (300, 2100)])
def test_lengths_of_every_kind(device, name, held, B, S):
    """One long sequence, ragged batches, more sequences than a wave has lanes (shares
    that run through several short ones among them)."""
    import torch

    Hq, Hkv, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(B)
    N, dtype = -(-S // page), types()[name]
    lengths = [S] + [int(x) for x in rng.integers(0, S + 1, B - 1)]
    if B >= 64:  # long runs of short ones
        lengths = [n if b % 9 == 0 else n % 40 for b, n in enumerate(lengths)]
        lengths[3:7] = [0] * 4
        lengths[-2:] = [0, 0]
    table = make_table(rng, B, N, B * N, lengths, page)
    cache = make_cache(device, rng, held, B * N, page, Hkv, D, table)
    q = torch.from_numpy(rng.standard_normal((B, 1, Hq, D), dtype=np.float32)).to(device, dtype)
    run(device, cache, table, lengths, q, dtype)
    run(device, cache, table, [0] * B, q, dtype, "no keys")


@pytest.mark.parametrize("name,held,H,T,D,S", [("bf16", "e4m3", 16, 1040, 256, 300), ("f32", "f32", 32, 1100, 64, 600),
                                               ("f16", "f16", 6, 333, 128, 900)])
def test_prompts_of_many_rows(device, name, held, H, T, D, S):
    """So many groups of rows that a wave has all sequences' keys to itself (the first
    two), or a few have; tokens with no key, more tokens than keys."""
    import torch

    B, page, dtype = 3, 20, types()[name]
    rng = np.random.default_rng(T)
    N = -(-S // page)
    lengths = [S, 0, S // 2]
    table = make_table(rng, B, N, B * N, lengths, page)
    cache = make_cache(device, rng, held, B * N, page, H, D, table)
    q = torch.from_numpy(rng.standard_normal((B, T, H, D), dtype=np.float32)).to(device, dtype)
    run(device, cache, table, lengths, q, dtype)


@pytest.mark.parametrize("held,S", [("bf16", 200), ("bf16", 3000), ("e4m3", 3000)])
def test_the_same_call_gives_the_same_bits(device, held, S):
    import torch
    from probjax_amd.attention import paged_decode

    B, H, D, page = 9, 4, 128, 16
    rng = np.random.default_rng(S)
    N = -(-S // page)
    lengths = [S] + [int(x) for x in rng.integers(0, S + 1, B - 1)]
    table = make_table(rng, B, N, B * N, lengths, page)
    cache = make_cache(device, rng, held, B * N, page, H, D, table)
    q = torch.from_numpy(rng.standard_normal((B, 2, 4 * H, D), dtype=np.float32)).to(device, torch.bfloat16)
    L = torch.tensor(lengths, dtype=torch.int32, device=device)
    first = paged_decode(q, cache, kv_lengths=L, return_lse=True)
    for _ in range(20):
        again = paged_decode(q, cache, kv_lengths=L, return_lse=True)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(first, again))


def _spoil(pool, at, value):
    """Sets one feature of every head in slot ``at = (page, slot)``."""
    import torch

    if pool.dtype is torch.float8_e4m3fn:
        pool.view(torch.uint8)[at[0], at[1], :, 3] = 0x7F
    else:
        pool[at[0], at[1], :, 3] = value


@pytest.mark.parametrize("name,held", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "e4m3"), ("f32", "e4m3")])
@pytest.mark.parametrize("T,page,keys", [(1, 16, 300), (4, 16, 300), (4, 5, 300), (1, 64, 300), (1, 16, 2500), (5, 16, 2500), (20, 7, 2500)])
def test_what_is_not_seen_does_not_reach_the_output(device, name, held, T, page, keys):
    """NaN and infinities behind the lengths, in pages of no sequence, in keys that the
    earlier tokens do not see; missing pages among the others."""
    import torch
    from probjax_amd.attention import paged_decode

    B, Hq, Hkv, D, dtype = 3, 4, 2, 64, types()[name]
    N = -(-keys // page)
    rng = np.random.default_rng(7)
    pages = B * N + 2
    table = rng.permutation(pages)[:B * N].reshape(B, N).astype(np.int32)
    lengths = [N * page - 7, keys // 2 - 19, T + 1]
    table[0, 3], table[0, N // 2], table[1, 0], table[2, 0] = -1, pages + 3, -2 ** 31, -1
    cache = make_cache(device, rng, held, pages, page, Hkv, D, table)
    clean_k, clean_v, there = gathered(cache, table, lengths)
    used = np.zeros((pages, page), bool)
    for b in range(B):
        n = np.arange(lengths[b])
        p, s = ref.slots(table, page, pages, b, n)
        used[p[p >= 0], s[p >= 0]] = True
    for i, at in enumerate(np.argwhere(~used)):
        _spoil(cache.k, at, [np.nan, np.inf, -np.inf][i % 3])
        _spoil(cache.v, at, [np.inf, np.nan, -np.inf][i % 3])
    q = torch.from_numpy(rng.standard_normal((B, T, Hq, D), dtype=np.float32)).to(device, dtype)
    L = torch.tensor(lengths, dtype=torch.int32, device=device)
    scale = 1.0 / math.sqrt(D)
    print("unused slots", flush=True)
    got, lse = paged_decode(q, cache, kv_lengths=L, return_lse=True)
    torch.cuda.synchronize()
    want = ref.paged_decode(to_np(q), clean_k, clean_v, there, lengths, scale)
    check(got, lse, want, dtype, D, N * page)
    if page > T:  # the third sequence's only keys are in a missing page
        assert not got[2].any() and torch.isposinf(lse[2]).all()
    if T > 1:
        print("keys that the last tokens alone see", flush=True)
        for b in range(2):
            p, s = ref.slots(table, page, pages, b, [lengths[b] - 1, lengths[b] - 2])
            for at in zip(p, s):
                _spoil(cache.k, at, np.nan)
                _spoil(cache.v, at, np.inf if b else np.nan)
        got, lse = paged_decode(q, cache, kv_lengths=L, return_lse=True)
        torch.cuda.synchronize()
        early = {n: x[:, :T - 2] if n in ("out", "spread") else x[..., :T - 2] for n, x in want.items()}
        check(got[:, :T - 2], lse[..., :T - 2], early, dtype, D, N * page)
        assert torch.isnan(got[:2, T - 2:]).any(-1).all()


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,D,page,keys", [(1, 64, 16, 300), (4, 64, 5, 300), (5, 128, 16, 2500), (1, 256, 16, 200)])
def test_exponents_of_unwritten_slots(device, name, T, D, page, keys):
    """Any byte may stand where nothing was written, 255 (a power of two that is
    infinite) too: behind the lengths, in page 0 (where missing pages are read from)
    and, for the keys that the last token alone sees, for the earlier ones."""
    import torch
    from probjax_amd.attention import paged_decode

    B, Hq, Hkv, dtype = 2, 4, 2, types()[name]
    N = -(-keys // page)
    rng = np.random.default_rng(8)
    pages = B * N + 1
    table = (1 + rng.permutation(B * N)).reshape(B, N).astype(np.int32)  # page 0: no one's
    lengths = [N * page - 3, keys // 2 - 19]
    table[0, 2], table[1, 1] = -1, pages
    cache = make_cache(device, rng, "e4m3", pages, page, Hkv, D, table)
    k, v, there = gathered(cache, table, lengths)
    used = np.zeros((pages, page), bool)
    for b in range(B):
        p, s = ref.slots(table, page, pages, b, np.arange(lengths[b]))
        used[p[p >= 0], s[p >= 0]] = True
    spoil = torch.from_numpy(~used).to(device)[:, None].expand(pages, Hkv, page)
    cache.k_exponents[spoil] = 255
    cache.v_exponents[spoil] = 255
    q = torch.from_numpy(rng.standard_normal((B, T, Hq, D), dtype=np.float32)).to(device, dtype)
    L = torch.tensor(lengths, dtype=torch.int32, device=device)
    want = ref.paged_decode(to_np(q), k, v, there, lengths, 1.0 / math.sqrt(D))
    got, lse = paged_decode(q, cache, kv_lengths=L, return_lse=True)
    torch.cuda.synchronize()
    check(got, lse, want, dtype, D, N * page)
    if T > 1:
        for b in range(B):
            p, s = ref.slots(table, page, pages, b, [lengths[b] - 1])
            cache.v_exponents[p[0], :, s[0]] = 255
        got, lse = paged_decode(q, cache, kv_lengths=L, return_lse=True)
        torch.cuda.synchronize()
        early = {n: x[:, :T - 1] if n in ("out", "spread") else x[..., :T - 1] for n, x in want.items()}
        check(got[:, :T - 1], lse[..., :T - 1], early, dtype, D, N * page)


@pytest.mark.parametrize("name,held", [("bf16", "bf16"), ("f16", "e4m3"), ("f32", "f32")])
def test_nan_and_infinities_that_are_seen(device, name, held):
    """As the definition has them: NaN in a seen value spoils its feature, in a seen key
    the row."""
    import torch
    from probjax_amd.attention import paged_decode

    B, Hq, Hkv, D, page, dtype = 2, 4, 2, 64, 16, types()[name]
    rng = np.random.default_rng(3)
    for S in (48, 1600):
        N = S // page
        table = rng.permutation(B * N).reshape(B, N).astype(np.int32)
        cache = make_cache(device, rng, held, B * N, page, Hkv, D, table)
        q = torch.from_numpy(rng.standard_normal((B, 1, Hq, D), dtype=np.float32)).to(device, dtype)
        clean = paged_decode(q, cache)
        _spoil(cache.v, (table[0, 1], 5), np.nan)
        got, lse = paged_decode(q, cache, return_lse=True)
        torch.cuda.synchronize()
        assert torch.isnan(got[0, ..., 3]).all() and not torch.isnan(lse).any()
        rest = torch.arange(D, device=device) != 3
        assert torch.equal(got[0][..., rest], clean[0][..., rest]) and torch.equal(got[1], clean[1])
        _spoil(cache.k, (table[1, 2], 0), np.nan)
        got, lse = paged_decode(q, cache, return_lse=True)
        torch.cuda.synchronize()
        assert torch.isnan(got[1]).all() and torch.isnan(lse[1]).all() and not torch.isnan(lse[0]).any()


@pytest.mark.parametrize("name,held", [("bf16", "bf16"), ("f16", "e4m3"), ("f32", "f32")])
def test_caches_without_a_page(device, name, held):
    """No pool, no page of a sequence, no sequence: zeros, LSE +inf, lengths of 0."""
    import torch
    from probjax_amd.attention import PagedCache, paged_decode, read_pages, write_pages

    dtype, pool = types()[name], types().get(held, torch.float8_e4m3fn)
    for pages, shape in ((0, (2, 3)), (4, (2, 0)), (0, (2, 0)), (4, (0, 3)), (0, (0, 0))):
        print(pages, shape, flush=True)
        table = torch.zeros(shape, dtype=torch.int32, device=device)
        cache = PagedCache.allocate(pages, 16, 2, 64, page_table=table, dtype=pool)
        B = shape[0]
        q = torch.full((B, 3, 4, 64), float("nan"), dtype=dtype, device=device)
        out, lse = paged_decode(q, cache, return_lse=True)
        k, v = read_pages(cache, length=20, dtype=dtype)
        lengths = write_pages(cache, q[:, :, :2], q[:, :, 2:])
        torch.cuda.synchronize()
        assert out.shape == q.shape and not out.any() and torch.isposinf(lse).all() and lse.shape == (B, 4, 3)
        assert k.shape == v.shape == (B, 20, 2, 64) and not k.any() and not v.any()
        assert lengths.tolist() == [min(3, cache.capacity)] * B


def test_contiguous_caches_and_views(device):
    """Without a table: page b is sequence b's; one sequence shared by the batch; the
    table a slice of a wider one; equal to the split-KV decode's result within both's
    roundings."""
    import torch
    from probjax_amd.attention import PagedCache, paged_decode, splitkv_forward

    B, S, Hq, Hkv, D = 3, 700, 8, 2, 128
    gen = torch.Generator(device=device).manual_seed(1)
    q, k, v = (torch.randn(s, generator=gen, device=device).to(torch.bfloat16)
               for s in ((B, 1, Hq, D), (B, S, Hkv, D), (B, S, Hkv, D)))
    L = torch.tensor([700, 33, 0], dtype=torch.int32, device=device)
    one = np.arange(B, dtype=np.int32)[:, None]
    cache = PagedCache(k, v)
    assert cache.capacity == S and cache.batch == B
    a, lse = run(device, cache, one, [700, 33, 0], q, torch.bfloat16)
    b = splitkv_forward(q, k, v, sm_scale=1.0 / math.sqrt(D), kv_lengths=L)
    torch.cuda.synchronize()
    # (each within 2^-8 of itself and of sum p|v| <= max|v| < 8)
    assert (a.float() - b.float()).abs().max() <= 4 * 2 ** -8 * 8
    shared = PagedCache(k[:1].expand(B, S, Hkv, D), v[:1].expand(B, S, Hkv, D))
    c = paged_decode(q, shared)
    d = paged_decode(q, PagedCache(k[:1].repeat(B, 1, 1, 1), v[:1].repeat(B, 1, 1, 1)))
    wide = torch.full((B, 9), -1, dtype=torch.int32, device=device)
    wide[:, 4] = torch.arange(B)
    torch.cuda.synchronize()
    assert torch.equal(c, d)
    # (room for twice the keys: sums in another order, so held to the definition, not to a)
    table = np.concatenate([one, np.full((B, 1), -1, np.int32)], 1)
    run(device, PagedCache(k, v, wide[:, 4:6]), table, [700, 33, 0], q, torch.bfloat16)


def test_scales_far_apart(device):
    """8-bit rows whose exponents lie 2^60 apart: the weights follow the true values."""
    import torch

    name, held, B, Hq, Hkv, D, page, N = "f32", "e4m3", 2, 4, 2, 64, 16, 4
    rng = np.random.default_rng(2)
    table = rng.permutation(B * N).reshape(B, N).astype(np.int32)
    for dtype in ("f32", "bf16"):
        cache = make_cache(device, rng, held, B * N, page, Hkv, D, table)
        cache.v_exponents.copy_(torch.from_numpy(rng.integers(60, 180, cache.v_exponents.shape).astype(np.uint8)))
        cache.k_exponents.copy_(torch.from_numpy(rng.integers(60, 119, cache.k_exponents.shape).astype(np.uint8)))
        q = torch.from_numpy(rng.standard_normal((B, 1, Hq, D), dtype=np.float32)).to(device, types()[dtype])
        run(device, cache, table, [N * page, 20], q, types()[dtype])


def test_many_heads(device):
    """More KV heads than the device holds waves, and numbers that no workgroup divides."""
    import torch

    rng = np.random.default_rng(4)
    for H, D, N, held in ((2053, 16, 33, "e4m3"), (37, 64, 40, "bf16"), (6, 128, 70, "bf16")):
        B, page, G = 2, 64, 2
        lengths = [N * page - 3, 70]
        table = make_table(rng, B, N, B * N, lengths, page)
        cache = make_cache(device, rng, held, B * N, page, H, D, table)
        q = torch.from_numpy(rng.standard_normal((B, 1, H * G, D), dtype=np.float32)).to(device, torch.bfloat16)
        run(device, cache, table, lengths, q, torch.bfloat16)


def test_a_share_of_keys_in_missing_pages(device):
    """Nothing but missing pages in whole parts of a sequence, and in all of it."""
    import torch

    rng = np.random.default_rng(5)
    B, Hq, Hkv, D, page, N = 3, 4, 2, 64, 16, 300
    lengths = [N * page, 4000, 700]
    for dtype, held in (("bf16", "bf16"), ("f16", "e4m3"), ("f32", "f32")):
        table = make_table(rng, B, N, B * N, lengths, page)
        table[0, 20:250], table[1, :200], table[2] = -1, -1, -1
        cache = make_cache(device, rng, held, B * N, page, Hkv, D, table)
        q = torch.from_numpy(rng.standard_normal((B, 2, Hq, D), dtype=np.float32)).to(device, types()[dtype])
        got, lse = run(device, cache, table, lengths, q, types()[dtype])
        assert not got[2].any() and torch.isposinf(lse[2]).all()
