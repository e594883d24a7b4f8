"""What the paged cache and its operators take and refuse, and where they launch (host
logic: devices, streams and launches are stubs, no GPU needed)."""

import copy
import dataclasses

import pytest
import torch
import torch.autograd.forward_ad as fwd

from probjax_amd import attention as A
from probjax_amd import hip_attention as hip
from probjax_amd import native
from tests.test_current_device import CURRENT, THEIRS, calls  # noqa: F401  (a fixture)

PAGES, PAGE, H, D, B, N = 6, 4, 2, 64, 2, 3


@pytest.fixture(autouse=True)
def anywhere(monkeypatch):
    monkeypatch.setattr(hip, "_gpu", lambda *ts: 0)


def table(*shape, dtype=torch.int32):
    return torch.zeros(shape or (B, N), dtype=dtype)


def pools(dtype=torch.bfloat16, shape=(PAGES, PAGE, H, D)):
    return torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)


def exponents():
    return [torch.zeros((PAGES, H, PAGE), dtype=torch.uint8) for _ in range(2)]


def cache(dtype=torch.bfloat16):
    x = exponents() if dtype is torch.float8_e4m3fn else ()
    return A.PagedCache(*pools(dtype), table(), *x)


def test_what_a_cache_knows():
    c = cache()
    assert (c.batch, c.page_size, c.capacity, c.kv_heads, c.head_dim) == (B, PAGE, N * PAGE, H, D)
    alone = A.PagedCache(*pools())
    assert (alone.batch, alone.capacity) == (PAGES, PAGE)
    one = dataclasses.replace(c, page_table=table(1, 7))
    assert (one.batch, one.capacity) == (1, 7 * PAGE) and one.k is c.k
    st = cache(torch.float8_e4m3fn).pages()
    assert st.k_exponents and st.table_len == N and st.pages == PAGES and st.k_token == H * D
    with pytest.raises(dataclasses.FrozenInstanceError):
        c.k = c.v


def test_allocate():
    c = A.PagedCache.allocate(PAGES, PAGE, H, D, page_table=table(), dtype=torch.float8_e4m3fn)
    assert c.k.dtype is torch.float8_e4m3fn and c.k_exponents.shape == (PAGES, H, PAGE) and c.unwritable is None
    assert A.PagedCache.allocate(B, 100, H, D, device="cpu").capacity == 100


def test_copies(tmp_path):
    """A cache is copied, and saved, as its tensors are."""
    c = cache(torch.float8_e4m3fn)
    same, other = copy.copy(c), copy.deepcopy(c)
    assert same.k is c.k and other.k is not c.k
    st = other.pages()
    assert (st.k, st.v_exponents, st.table) == (other.k.data_ptr(), other.v_exponents.data_ptr(), other.page_table.data_ptr())
    pair = torch.zeros((2, PAGES, PAGE, H, D), dtype=torch.bfloat16)
    both = copy.deepcopy(A.PagedCache(*pair, table()))
    assert both.unwritable is None and both.v.data_ptr() - both.k.data_ptr() == 2 * both.k.numel()
    torch.save(c, tmp_path / "cache")
    back = torch.load(tmp_path / "cache", weights_only=False)
    assert back.capacity == c.capacity and back.k.dtype is c.k.dtype and torch.equal(back.page_table, c.page_table)


def _offset(t):
    return torch.zeros((t.numel() + 1,), dtype=t.dtype)[1:].view(t.shape)


@pytest.mark.parametrize("make,msg", [
    (lambda: (torch.zeros(2, 3, 4), torch.zeros(2, 3, 4)), r"\[pages, page_size"),
    (lambda: (pools()[0], pools(shape=(PAGES, PAGE, H, 2 * D))[0]), "one shape"),
    (lambda: (pools()[0], pools(torch.float16)[0]), "one shape and dtype"),
    (lambda: pools(torch.float64), "unsupported cache dtype"),
    (lambda: pools(torch.int8), "unsupported cache dtype"),
    (lambda: pools(shape=(PAGES, 0, H, D)), "needs slots and heads"),
    (lambda: pools(shape=(PAGES, PAGE, H, 60)), "multiples of 8"),
    (lambda: (*pools(torch.float8_e4m3fn, (PAGES, PAGE, H, 72)), None, *exponents()), "multiples of 16"),
    (lambda: pools(torch.float32, (PAGES, PAGE, H, 6)), "multiples of 4"),
    (lambda: pools(shape=(PAGES, PAGE, H, 264)), "up to 256"),
    (lambda: pools(torch.float8_e4m3fn), "needs k_exponents"),
    (lambda: (*pools(), None, *exponents()), "take none"),
    (lambda: (*pools(torch.float8_e4m3fn), None, exponents()[0], None), "needs k_exponents"),
    (lambda: (*pools(torch.float8_e4m3fn), None, exponents()[0], exponents()[1].int()), "contiguous uint8"),
    (lambda: (*pools(torch.float8_e4m3fn), None, exponents()[0], exponents()[1].transpose(0, 1)), "contiguous uint8"),
    (lambda: tuple(t.transpose(2, 3) for t in pools(shape=(PAGES, PAGE, D, 8))), "contiguous features"),
    (lambda: tuple(_offset(t) for t in pools()), "start on 16 bytes"),
    (lambda: tuple(t[..., :56] for t in pools(shape=(PAGES, PAGE, H, 60))), "start on 16 bytes"),
    (lambda: (*pools(), table(dtype=torch.int64)), "int32"),
    (lambda: (*pools(), table(6)), "int32"),
    (lambda: (*pools(), table(N, B).t()), "contiguous rows"),
    (lambda: (*pools(shape=(1, 1 << 16, 1, 8)), table(1, (1 << 14) + 1)), r"2\^30"),
    (lambda: (pools()[0].requires_grad_(), pools()[1]), "no gradient"),
])
def test_caches_that_are_refused(make, msg):
    with pytest.raises(ValueError, match=msg):
        A.PagedCache(*make())


def test_caches_that_can_only_be_read():
    k, v = pools()
    x = torch.zeros((B, 3, H, D), dtype=torch.bfloat16)
    for args, why in (((k, k), "share memory"), ((k[:1].expand(B, PAGE, H, D), v[:B]), "expanded"),
                      ((k[:4], k[2:]), "share memory"),
                      ((torch.as_strided(k, (B, PAGE, H, D), (H * D, H * D, D, 1)), v[:B]), "overlap")):
        c = A.PagedCache(*args, table())
        assert why in c.unwritable
        with pytest.raises(ValueError, match=why):
            A.write_pages(c, x, x)
    beside = torch.zeros((PAGES, 2, PAGE, H, D), dtype=torch.bfloat16)
    assert A.PagedCache(beside[:, 0], beside[:, 1], table()).unwritable is None
    assert A.PagedCache(k[:3], k[3:], table()).unwritable is None


def new(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape or (B, 3, H, D), dtype=dtype)


@pytest.mark.parametrize("call,msg", [
    (lambda c: A.write_pages(c, new(B, 3, H), new(B, 3, H)), r"\[B, T, Hkv, D\]"),
    (lambda c: A.write_pages(c, new(), new(B, 4, H, D)), "one shape"),
    (lambda c: A.write_pages(c, new(), new(dtype=torch.float16)), "one shape and dtype"),
    (lambda c: A.write_pages(c, new(3, 3, H, D), new(3, 3, H, D)), "does not fit"),
    (lambda c: A.write_pages(c, new(B, 3, 1, D), new(B, 3, 1, D)), "does not fit"),
    (lambda c: A.write_pages(c, new(dtype=torch.float16), new(dtype=torch.float16)), "that dtype"),
    (lambda c: A.write_pages(c, new(dtype=torch.float64), new(dtype=torch.float64)), "unsupported dtype"),
    (lambda c: A.write_pages(c, new(), new(), kv_lengths=torch.zeros(3, dtype=torch.int32)), "kv_lengths must have shape"),
    (lambda c: A.write_pages(c, new(), new(), new_lengths=torch.zeros(B)), "new_lengths must hold integers"),
    (lambda c: A.write_pages(c, new().requires_grad_(), new()), "no gradient"),
    (lambda c: A.read_pages(c, dtype=torch.float16), "what it holds"),
    (lambda c: A.read_pages(c, length=-1), "length"),
    (lambda c: A.read_pages(c, kv_lengths=[1, 2, 3]), "kv_lengths"),
    (lambda c: A.paged_decode(new(B, H, D), c), r"\[B, T, Hq, D\]"),
    (lambda c: A.paged_decode(new(B, 1, 3, D), c), "does not fit"),
    (lambda c: A.paged_decode(new(B, 0, H, D), c), "does not fit"),
    (lambda c: A.paged_decode(new(B, 1, H, 80), c), "does not fit"),
    (lambda c: A.paged_decode(new(3, 1, H, D), c), "does not fit"),
    (lambda c: A.paged_decode(new(B, 1, H, D, dtype=torch.float32), c), "of that dtype"),
    (lambda c: A.paged_decode(new(B, 1, H, D).requires_grad_(), c), "no gradient"),
    (lambda c: A.paged_decode(new(B, 1, H, D), c, kv_lengths=torch.zeros(B, dtype=torch.bool)), "integers"),
])
def test_calls_that_are_refused(call, msg):
    with pytest.raises(ValueError, match=msg):
        call(cache())


def test_new_rows_in_the_pools_are_refused(monkeypatch):
    """What a launch would read and write in an open order; pools beside them are not."""
    both = torch.zeros((PAGES, 3, PAGE, H, D), dtype=torch.bfloat16)
    c = A.PagedCache(both[:, 0], both[:, 1], table())
    flat = both.view(-1, H, D)
    launched = []
    monkeypatch.setattr(hip, "_call", lambda *args: launched.append(args))
    for x in (both[:B, 0, :3], both[:B, 1, 1:4], flat[:10].view(B, 5, H, D)):
        for k, v in ((x, torch.zeros_like(x)), (torch.zeros_like(x), x)):
            with pytest.raises(ValueError, match="share memory"):
                A.write_pages(c, k, v)
    assert not launched
    A.write_pages(c, both[:B, 2, :3], both[2:2 + B, 2, :3])
    assert len(launched) == 1


def test_reads_of_8_bits_name_a_float_type():
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        A.read_pages(cache(torch.float8_e4m3fn), dtype=torch.float8_e4m3fn)


def test_tangents_are_refused():
    x = new()
    with fwd.dual_level(), torch.no_grad():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: A.write_pages(cache(), d, x), lambda: A.write_pages(cache(), x, d),
                     lambda: A.paged_decode(d, cache())):
            with pytest.raises(ValueError, match="no gradient"):
                call()
        k, v = pools()
        with pytest.raises(ValueError, match="no gradient"):
            A.PagedCache(fwd.make_dual(k, torch.ones_like(k)), v)


def test_tensors_of_two_devices_are_refused(monkeypatch):
    monkeypatch.undo()
    with pytest.raises(ValueError, match="ROCm device"):
        A.PagedCache(*pools(), table())


def test_launches_on_the_tensors_device(calls):  # noqa: F811
    c, q = cache(torch.float8_e4m3fn), cache()
    object.__setattr__(c, "index", THEIRS)
    for call in (lambda: A.write_pages(c, new(), new()), lambda: A.read_pages(c), lambda: A.paged_decode(new(B, 1, 4, D), q)):
        before = len(calls)
        call()
        assert len(calls) > before
    assert {(device, stream) for _, device, stream in calls} == {(THEIRS, 1000 + THEIRS)} and CURRENT != THEIRS
    assert {name for name, *_ in calls} == {"pjx_write_pages", "pjx_read_pages", "pjx_paged_decode"}


def test_addresses_are_taken_on_every_call(monkeypatch):
    """A tensor whose storage is replaced is read where it is then."""
    seen = []
    monkeypatch.setattr(hip, "_call", lambda index, entry, *args: seen.append([a.k for a in args if isinstance(a, native.Pages)]))
    monkeypatch.setattr(native, "load", lambda: type("L", (), {"pjx_read_pages": None})())
    c = cache()
    A.read_pages(c)
    c.k.set_(torch.zeros_like(c.k))
    A.read_pages(c)
    assert seen[0] != seen[1] and seen[1] == [c.k.data_ptr()]
