"""Writing to and reading from a paged cache, against the oracle.  Copies, codes and
exponents are the oracle's bit for bit; what is read of 8 bits is its float64 value
rounded once to the type.  Everything that a call does not name stays as it was."""

import dataclasses

import numpy as np
import pytest

from oracle import paged as ref
from tests._helpers import to_np

pytestmark = pytest.mark.gpu


def types():
    import torch

    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}


def raw(t):
    """The bits of a tensor, as integers on the host."""
    import torch

    as_int = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]
    return t.detach().contiguous().view(as_int).cpu().numpy()


def make_table(rng, B, N, pages, lengths, page):
    """Random pages of one pool for every sequence, none behind its keys."""
    table = rng.permutation(pages)[:B * N].reshape(B, N).astype(np.int32)
    table[np.arange(N) * page >= np.asarray(lengths)[:, None]] = -1
    return table


def make_cache(device, rng, name, pages, page, H, D, table, layout="tokens", spread=0):
    """A cache whose pools hold random rows (8-bit ones: any code but NaN, exponents
    around 1 over ``2 * spread`` octaves)."""
    import torch
    from probjax_amd.attention import PagedCache

    dtype, pools, exps = types()[name], [], [None, None]
    for i in range(2):
        if name == "e4m3":
            codes = rng.integers(0, 255, (pages, page, H, D), dtype=np.uint8)
            codes[codes & 127 == 127] = 0
            x = torch.from_numpy(codes).to(device)
            exps[i] = torch.from_numpy(rng.integers(118 - spread, 121 + spread, (pages, H, page)).astype(np.uint8)).to(device)
        else:
            x = torch.from_numpy(rng.standard_normal((pages, page, H, D), dtype=np.float32)).to(device, dtype)
        if layout == "heads":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        pools.append(x.view(dtype))
    t = None if table is None else torch.from_numpy(np.ascontiguousarray(table)).to(device)
    return PagedCache(*pools, t, *exps)


def host_rows(cache, kv):
    """A pool's rows as float64 ``[pages, page, H, D]``."""
    pool, e = (cache.k, cache.k_exponents) if kv == 0 else (cache.v, cache.v_exponents)
    if e is None:
        return to_np(pool).astype(np.float64)
    return ref.decode(raw(pool), np.moveaxis(e.cpu().numpy(), 1, 2))


WRITES = [
    # type, cache, B, T, H, D, page, room (pages), layout
    ("bf16", "e4m3", 3, 1, 8, 128, 16, 3, "tokens"),
    ("bf16", "e4m3", 2, 70, 2, 64, 16, 6, "heads"),
    ("f16", "e4m3", 2, 33, 3, 80, 20, 4, "tokens"),
    ("f32", "e4m3", 2, 9, 1, 256, 8, 3, "tokens"),
    ("f32", "e4m3", 1, 300, 4, 112, 1, 320, "heads"),
    ("bf16", "e4m3", 2, 5, 2, 16, 7, 2, "tokens"),
    ("bf16", "bf16", 2, 40, 2, 128, 32, 3, "tokens"),
    ("f16", "f16", 2, 17, 2, 72, 5, 6, "heads"),
    ("f16", "f16", 1, 3, 1, 8, 3, 2, "tokens"),
    ("f32", "f32", 2, 21, 2, 256, 48, 1, "tokens"),
    ("f32", "f32", 3, 2, 5, 20, 4, 2, "heads"),
    ("bf16", "bf16", 1, 1000, 1, 256, 100, 12, "tokens"),
]


@pytest.mark.parametrize("case", WRITES, ids=lambda c: "-".join(map(str, c)))
def test_write(device, case):
    import torch
    from probjax_amd.attention import write_pages

    name, held, B, T, H, D, page, N, layout = case
    rng = np.random.default_rng(T + D)
    pages = B * N + 2
    before = rng.integers(0, max(N * page - T, 0) + 3, B)
    count = rng.integers(0, T + 1, B)
    before[0], count[0] = N * page - T + 1, T  # one more than there is room for
    count[-1] = T if B > 1 else count[-1]
    table = make_table(rng, B, N, pages, before + count, page)
    cache = make_cache(device, rng, held, pages, page, H, D, table, layout)
    x = [(rng.standard_normal((B, T, H, D)) * np.exp2(rng.integers(-9, 9, (B, T, H, 1)))).astype(np.float32) for _ in range(2)]
    new = [torch.from_numpy(y).to(device, types()[name]) for y in x]
    L, n = (torch.from_numpy(y.astype(np.int32)).to(device) for y in (before, count))
    old = [raw(cache.k), raw(cache.v)]
    old_e = [e.cpu().numpy() for e in (cache.k_exponents, cache.v_exponents)] if held == "e4m3" else None
    lengths = write_pages(cache, *new, kv_lengths=L, new_lengths=n)
    torch.cuda.synchronize()
    for i, pool in enumerate((cache.k, cache.v)):
        rows = raw(new[i])
        if held == "e4m3":
            rows, e = ref.encode(to_np(new[i]), name)
            got = (cache.k_exponents, cache.v_exponents)[i].cpu().numpy()
            want, _ = ref.append(np.moveaxis(old_e[i], 1, 2), e, table, before, count)
            np.testing.assert_array_equal(np.moveaxis(got, 1, 2), want)
        want, want_lengths = ref.append(old[i], rows, table, before, count)
        np.testing.assert_array_equal(raw(pool), want)
    np.testing.assert_array_equal(lengths.cpu().numpy(), want_lengths)


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_extremes_in_8_bits(device, name):
    """Zeros, infinities, NaN, the type's ends, ties and subnormals, row by row."""
    import torch
    from probjax_amd.attention import PagedCache, read_pages, write_pages

    dtype, D = types()[name], 64
    info = torch.finfo(dtype)
    rng = np.random.default_rng(1)
    rows = [np.zeros(D), np.full(D, info.max), np.full(D, -info.max), np.full(D, info.tiny), np.full(D, info.smallest_normal),
            np.full(D, np.inf), np.full(D, np.nan), np.r_[np.full(D - 1, -np.inf), 3.0], np.r_[np.nan, np.arange(D - 1)],
            448.0 - np.arange(D) / 2, np.r_[448.0, 449.0, np.arange(D - 2)], np.arange(D) * info.tiny,
            np.r_[1.0, np.exp2(-np.arange(D - 1, dtype=float))], np.r_[448.0, (2 * np.arange(D - 1) + 1) * 2.0 ** -10],
            np.full(D, info.tiny * info.eps), np.r_[info.max, -np.ones(D - 1)], -np.zeros(D)]
    rows += [rng.standard_normal(D) * 2.0 ** int(e) for e in range(-12, 12)]
    x = torch.tensor(np.array(rows), dtype=torch.float64).to(dtype).to(device)[None, :, None]
    T = x.shape[1]
    cache = PagedCache.allocate(1, T, 1, D, dtype=torch.float8_e4m3fn, device=device)
    y = x.flip(1).contiguous()
    lengths = write_pages(cache, x, y)
    torch.cuda.synchronize()
    assert lengths.tolist() == [T]
    for t, pool, exps in ((x, cache.k, cache.k_exponents), (y, cache.v, cache.v_exponents)):
        codes, e = ref.encode(to_np(t), name)
        np.testing.assert_array_equal(exps.cpu().numpy(), np.moveaxis(e, 1, 2))
        got = raw(pool)
        nan = codes & 127 == 127
        np.testing.assert_array_equal(got[~nan], codes[~nan])
        assert (got[nan] & 127 == 127).all()
    k, v = read_pages(cache, dtype=dtype)
    torch.cuda.synchronize()
    back = ref.decode(*ref.encode(to_np(x), name))
    want = torch.from_numpy(back).to(dtype)
    got = k.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and not torch.isinf(got).any()
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert torch.equal(torch.nan_to_num(v.cpu().flip(1)), torch.nan_to_num(want))


READS = [
    # cache, type read, B, H, D, page, room (pages), layout, length
    ("e4m3", "bf16", 3, 8, 128, 16, 4, "tokens", None),
    ("e4m3", "f16", 2, 2, 80, 20, 3, "heads", 50),
    ("e4m3", "f32", 2, 3, 64, 1, 40, "tokens", 41),
    ("e4m3", "bf16", 1, 1, 256, 7, 5, "tokens", 1),
    ("bf16", "bf16", 2, 2, 128, 32, 3, "heads", None),
    ("f16", "f16", 2, 3, 72, 5, 6, "tokens", 31),
    ("f16", "f16", 70, 1, 8, 2, 2, "tokens", 3),
    ("f32", "f32", 2, 2, 256, 48, 2, "tokens", 100),
    ("f32", "f32", 2, 5, 20, 4, 2, "heads", 9),
]


@pytest.mark.parametrize("case", READS, ids=lambda c: "-".join(map(str, c)))
def test_read(device, case):
    import torch
    from probjax_amd.attention import read_pages

    held, name, B, H, D, page, N, layout, length = case
    rng = np.random.default_rng(D + page)
    pages, dtype = B * N + 1, types()[name]
    lengths = rng.integers(0, N * page + 1, B)
    lengths[0] = N * page + 5
    table = make_table(rng, B, N, pages, lengths, page)
    table[0, N // 2] = -7  # pages that are missing among others
    if B > 1:
        table[1, 0] = pages
    cache = make_cache(device, rng, held, pages, page, H, D, table, layout, spread=6)
    L = torch.from_numpy(lengths).to(device)
    for given in (L, None):
        got = read_pages(cache, kv_lengths=given, length=length, dtype=dtype)
        torch.cuda.synchronize()
        for kv in range(2):
            want, _ = ref.gather(host_rows(cache, kv), table, lengths if given is not None else [N * page] * B,
                                 N * page if length is None else length)
            assert got[kv].dtype == dtype and got[kv].is_contiguous()
            assert torch.equal(got[kv].cpu(), torch.from_numpy(want).to(dtype))


def test_strided_rows_are_read_in_place_and_others_copied(device):
    """Slices of a fused projection, transposed heads, rows that start off 16 bytes."""
    import torch
    from probjax_amd import hip_attention as hip
    from probjax_amd.attention import PagedCache, write_pages

    B, T, H, D = 2, 11, 2, 64
    gen = torch.Generator(device=device).manual_seed(0)
    fused = torch.randn((B, T, 4 * H, D), generator=gen, device=device).to(torch.bfloat16)
    odd = torch.randn((B * T * H * D + 1,), generator=gen, device=device).to(torch.bfloat16)[1:].view(B, T, H, D)
    turned = torch.randn((B, H, T, D), generator=gen, device=device).to(torch.bfloat16).transpose(1, 2)
    apart = torch.randn((B, T, H, D + 1), generator=gen, device=device).to(torch.bfloat16)[..., :D]
    one = torch.randn((1, 1, H, D), generator=gen, device=device).to(torch.bfloat16).expand(B, T, H, D)
    assert hip._new_rows(fused[:, :, H:2 * H], fused[:, :, 3 * H:])[0].data_ptr() == fused[:, :, H:].data_ptr()
    for x, y in ((fused[:, :, H:2 * H], fused[:, :, 3 * H:]), (odd, turned), (apart, one), (turned, odd)):
        caches = [PagedCache.allocate(B, T, H, D, dtype=torch.float8_e4m3fn, device=device) for _ in range(2)]
        write_pages(caches[0], x, y)
        write_pages(caches[1], x.clone(memory_format=torch.contiguous_format), y.clone(memory_format=torch.contiguous_format))
        torch.cuda.synchronize()
        for name in ("k", "v", "k_exponents", "v_exponents"):
            assert np.array_equal(raw(getattr(caches[0], name)), raw(getattr(caches[1], name)))


def test_a_layer_of_many_and_pools_of_one_allocation(device):
    """K and V beside each other in one tensor, one layer of several: the rest stays."""
    import torch
    from probjax_amd.attention import PagedCache, read_pages, write_pages

    pages, page, H, D, layers = 5, 8, 2, 64, 3
    store = torch.full((layers, pages, 2, H, page, D), 7.0, dtype=torch.bfloat16, device=device)
    k, v = store[1, :, 0].transpose(1, 2), store[1, :, 1].transpose(1, 2)
    table = torch.tensor([[4, 0], [2, -1]], dtype=torch.int32, device=device)
    cache = PagedCache(k, v, table)
    new = torch.randn((2, 12, H, D), device=device).to(torch.bfloat16)
    lengths = write_pages(cache, new, -new)
    got = read_pages(cache, kv_lengths=lengths, length=13)
    torch.cuda.synchronize()
    assert lengths.tolist() == [12, 12]
    assert torch.equal(got[0][0, :12], new[0]) and torch.equal(got[1][0, :12], -new[0])
    assert torch.equal(got[0][1, :8], new[1, :8]) and not got[0][1, 8:].any() and not got[0][:, 12:].any()
    touched = torch.zeros((layers, pages, 2, H, page), dtype=torch.bool, device=device)
    touched[1, 4], touched[1, 0, :, :, :4], touched[1, 2] = True, True, True
    assert (store[~touched] == 7.0).all() and (store[touched] != 7.0).any()
    # the same pools for one sequence of them
    part = dataclasses.replace(cache, page_table=table[1:])
    assert part.batch == 1
    one = read_pages(part, kv_lengths=[8], length=8)
    torch.cuda.synchronize()
    assert torch.equal(one[0][0], new[1, :8])


@pytest.mark.parametrize("name,held", [("bf16", "e4m3"), ("bf16", "bf16"), ("f32", "f32")])
def test_nothing_to_do(device, name, held):
    import torch
    from probjax_amd.attention import PagedCache, read_pages, write_pages

    dtype, H, D = types()[name], 2, 64
    for B, T, pages, N in ((0, 3, 4, 2), (2, 0, 4, 2), (2, 3, 0, 2), (2, 3, 4, 0)):
        table = torch.full((B, N), -1, dtype=torch.int32, device=device)
        cache = PagedCache.allocate(pages, 4, H, D, page_table=table, dtype=types()[held])
        new = torch.ones((B, T, H, D), dtype=dtype, device=device)
        lengths = write_pages(cache, new, new, kv_lengths=torch.full((B,), 1, device=device))
        k, v = read_pages(cache, kv_lengths=lengths, length=5, dtype=dtype)
        none, _ = read_pages(cache, length=0, dtype=dtype)
        torch.cuda.synchronize()
        assert lengths.tolist() == [min(1 + T, 4 * N)] * B
        assert k.shape == v.shape == (B, 5, H, D) and not k.any() and not v.any() and none.shape == (B, 0, H, D)
