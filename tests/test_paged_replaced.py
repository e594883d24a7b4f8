"""A paged cache whose tensors are given other memory, another order or another size after
it was made: the next call takes them as they are then, or refuses them (host logic:
launches are stubs, no GPU needed)."""

import pytest
import torch

from probjax_amd import attention as A
from probjax_amd import hip_attention as hip
from probjax_amd import native
from tests.test_paged_host import B, D, H, N, PAGE, PAGES, anywhere, cache, new, table  # noqa: F401  (a fixture)


@pytest.fixture
def launched(monkeypatch):
    """The ``pjx_pages`` of every launch, as field values."""
    seen = []

    def call(index, entry, *args):
        seen.extend({n: getattr(a, n) for n, _ in a._fields_} for a in args if isinstance(a, native.Pages))

    monkeypatch.setattr(hip, "_call", call)
    return seen


def operators(c):
    x = new(c.batch, 3, c.kv_heads, c.head_dim)
    return (lambda: A.write_pages(c, x, x), lambda: A.read_pages(c), lambda: A.paged_decode(x, c))


def test_rows_of_the_new_pools_are_refused(launched):
    c = cache()
    store = torch.zeros((3, PAGES, PAGE, H, D), dtype=torch.bfloat16)
    c.k.set_(store[0])
    c.v.set_(store[1])
    for x in (store[0, :B, :3], store[1, :B, :3]):
        with pytest.raises(ValueError, match="share memory"):
            A.write_pages(c, x, torch.zeros_like(x))
        with pytest.raises(ValueError, match="share memory"):
            A.write_pages(c, torch.zeros_like(x), x)
    assert not launched
    A.write_pages(c, store[2, :B, :3], store[2, :B, :3])
    assert launched[-1]["k"] == store[0].data_ptr() and launched[-1]["v"] == store[1].data_ptr()


def test_pools_that_come_to_share_memory_are_not_written(launched):
    c = cache()
    c.v.set_(c.k)
    with pytest.raises(ValueError, match="share memory"):
        A.write_pages(c, new(), new())
    assert not launched
    A.read_pages(c)
    assert launched[-1]["k"] == launched[-1]["v"]
    c.v.set_(torch.zeros_like(c.k))
    A.write_pages(c, new(), new())


@pytest.mark.parametrize("i", range(3))
def test_new_strides_are_taken(launched, i):
    c = cache()
    for x in (c.k, c.v):
        x.set_(torch.zeros((PAGES, H, PAGE, D), dtype=torch.bfloat16).transpose(1, 2))
    operators(c)[i]()
    assert launched[-1]["k_token"] == launched[-1]["v_token"] == D
    assert launched[-1]["k_head"] == launched[-1]["v_head"] == PAGE * D
    # the same memory in another order
    before = launched[-1]["k"]
    c.k.as_strided_((PAGES, PAGE, H, D), (PAGE * H * D, H * D, D, 1))
    operators(c)[i]()
    assert launched[-1]["k"] == before and launched[-1]["k_token"] == H * D and launched[-1]["v_token"] == D


@pytest.mark.parametrize("i", range(3))
def test_new_sizes_are_taken(launched, i):
    """Fewer pages (what lies behind them is not the cache's any more), another table."""
    c = cache(torch.float8_e4m3fn)
    pools = [torch.zeros((2, PAGE, H, D), dtype=torch.float8_e4m3fn) for _ in range(2)]
    for x, y in zip((c.k, c.v), pools):
        x.set_(y)
    with pytest.raises(ValueError, match="exponents"):
        operators(c)[i]()
    for x in (c.k_exponents, c.v_exponents):
        x.set_(torch.zeros((2, H, PAGE), dtype=torch.uint8))
    c.page_table.set_(table(3, 7))
    if i != 1:
        with pytest.raises(ValueError, match="does not fit"):
            x = new(B, 3, H, D)
            A.write_pages(c, x, x) if i == 0 else A.paged_decode(x, c)
    A.read_pages(c)
    operators(c)[i]()
    assert launched[-1]["pages"] == 2 and launched[-1]["table_len"] == 7
    assert launched[-1]["k_exponents"] == c.k_exponents.data_ptr()
    assert (c.batch, c.capacity) == (3, 7 * PAGE)


@pytest.mark.parametrize("i", range(3))
def test_what_a_cache_cannot_be_is_refused(launched, i):
    for replace, msg in (
        (lambda c: c.k.set_(torch.zeros((PAGES, PAGE, H, 2 * D), dtype=torch.bfloat16)), "one shape"),
        (lambda c: c.page_table.set_(table(N, B).t()), "contiguous rows"),
        (lambda c: c.v.set_(torch.zeros(PAGES * PAGE * H * D + 1, dtype=torch.bfloat16)[1:].view(c.k.shape)), "16 bytes"),
        (lambda c: setattr(c.v, "data", c.v.data.to(torch.float16)), "one shape and dtype"),
    ):
        c = cache()
        calls = operators(c)
        replace(c)
        with pytest.raises(ValueError, match=msg):
            calls[i]()
    assert not launched


def test_a_cache_that_stays_is_checked_once(monkeypatch, launched):
    c, checks = cache(), []
    whole = hip.pages_struct
    monkeypatch.setattr(hip, "pages_struct", lambda *ts: checks.append(1) or whole(*ts))
    for call in operators(c) * 2:
        call()
    c.page_table.fill_(1), c.k.zero_()  # contents are the caller's
    for call in operators(c):
        call()
    assert not checks
    c.k.set_(torch.zeros_like(c.k))
    for call in operators(c):
        call()
    assert len(checks) == 1
