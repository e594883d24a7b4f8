"""Refusals of the paged cache's entry points: every argument is checked before any HIP
call, so this runs without a GPU (the pointers are never followed)."""

import ctypes

import pytest

from probjax_amd import native
from tests.test_native_cache_ops import refused

P = ctypes.c_void_p
F32, BF16, F16, E4M3 = (getattr(native, "PJX_DTYPE_" + n) for n in ("F32", "BF16", "F16", "E4M3"))


@pytest.fixture(scope="module")
def lib():
    return native.load()


def pages(**over):
    a = dict(k=16, v=16, k_exponents=16, v_exponents=16, table=16, table_stride=5, table_len=5, pages=12, page_size=16,
             k_page=16 * 128, k_token=128, k_head=64, v_page=16 * 128, v_token=128, v_head=64)
    return native.Pages(**{**a, **over})


def _write(cache=None, **over):
    a = dict(dtype=BF16, held=E4M3, k=P(16), v=P(16), cache=cache or pages(), lengths=None, fresh=None, out=P(16), B=2,
             T=3, H=2, D=64, strides=None, stream=None)
    return {**a, **over}


def _read(cache=None, **over):
    a = dict(dtype=BF16, held=E4M3, cache=cache or pages(), lengths=None, k=P(16), v=P(16), B=2, L=10, H=2, D=64,
             stream=None)
    return {**a, **over}


def _decode(cache=None, **over):
    a = dict(dtype=BF16, held=E4M3, q=P(16), cache=cache or pages(), lengths=None, o=P(16), lse=None, ws=P(16),
             ws_bytes=1 << 30, B=2, T=1, Hq=4, H=2, D=64, scale=0.1, stream=None)
    return {**a, **over}


CACHES = [
    (pages(pages=-1), "bad sizes"),
    (pages(page_size=0), "bad sizes"),
    (pages(table_len=-1), "bad sizes"),
    (pages(page_size=1 << 20, table_len=1 << 11), "2^30"),
    (pages(pages=1 << 31), "out of range"),
    (pages(table=None), "without a table"),
    (pages(table=None, table_len=1, pages=1), "without a table"),
    (pages(table_stride=-1), "table stride"),
    (pages(k_page=-16), "strides out of range"),
    (pages(k_token=100), "16-byte"),
    (pages(v_head=8), "16-byte"),
    (pages(k=None), "null"),
    (pages(k_exponents=None), "null"),
    (pages(v=24), "16 bytes"),
]


@pytest.mark.parametrize("entry,make", [("pjx_write_pages", _write), ("pjx_read_pages", _read), ("pjx_paged_decode", _decode)])
@pytest.mark.parametrize("cache,msg", CACHES, ids=lambda x: x if isinstance(x, str) else "")
def test_caches(lib, entry, make, cache, msg):
    refused(lib, entry, make(cache), msg)


@pytest.mark.parametrize("entry,make", [("pjx_write_pages", _write), ("pjx_read_pages", _read), ("pjx_paged_decode", _decode)])
@pytest.mark.parametrize("over,msg", [
    (dict(held=9), "cache_dtype"),
    (dict(dtype=E4M3), "dtype"),
    (dict(held=F16), "another dtype"),
    (dict(D=272), "head_dim"),
    (dict(D=72), "head_dim"),  # whole chunks in 16 bits, not in 8
    (dict(D=0), "head_dim"),
    (dict(H=0), "bad sizes"),
    (dict(B=-1), "bad sizes"),
    (dict(B=1 << 25), "out of range"),
])
def test_what_the_calls_share(lib, entry, make, over, msg):
    refused(lib, entry, make(**over), msg)


@pytest.mark.parametrize("over,msg", [
    (dict(T=-1), "out of range"),
    (dict(k=None), "null"),
    (dict(out=None), "null"),
    (dict(v=P(8)), "16 bytes"),
    (dict(strides=native.CacheStrides(128, 128, 68, 128, 128, 64)), "16-byte"),
    (dict(strides=native.CacheStrides(128, -128, 64, 128, 128, 64)), "out of range"),
])
def test_write_pages(lib, over, msg):
    refused(lib, "pjx_write_pages", _write(**over), msg)


def test_more_than_a_launch_counts(lib):
    wide = dict(H=256, T=1 << 30, strides=native.CacheStrides(0, 0, 64, 0, 0, 64))
    refused(lib, "pjx_write_pages", _write(**wide), "too many new tokens")
    refused(lib, "pjx_write_pages", _write(held=BF16, cache=pages(k_exponents=None), **wide), "too many new tokens")
    refused(lib, "pjx_read_pages", _read(H=256, L=1 << 30), "too long")


@pytest.mark.parametrize("over,msg", [(dict(L=-1), "out of range"), (dict(k=None), "null"), (dict(v=P(4)), "16 bytes")])
def test_read_pages(lib, over, msg):
    refused(lib, "pjx_read_pages", _read(**over), msg)


@pytest.mark.parametrize("over,msg,code", [
    (dict(T=0), "bad sizes", 1),
    (dict(Hq=3), "bad sizes", 1),
    (dict(Hq=0), "bad sizes", 1),
    (dict(Hq=1 << 21), "out of range", 1),
    (dict(Hq=1 << 20, T=2), "out of range", 1),
    (dict(scale=0.0), "sm_scale", 1),
    (dict(scale=float("nan")), "sm_scale", 1),
    (dict(q=None), "null", 1),
    (dict(o=P(8)), "16 bytes", 1),
    (dict(ws=P(8)), "16 bytes", 1),
    (dict(ws=None), "workspace", 3),
    (dict(ws_bytes=1000), "workspace", 3),
])
def test_paged_decode(lib, over, msg, code):
    refused(lib, "pjx_paged_decode", _decode(**over), msg, code)


def test_room_for_too_many_keys(lib):
    cache = pages(page_size=1 << 15, table_len=1 << 15, table_stride=1 << 15)
    refused(lib, "pjx_paged_decode", _decode(cache, B=17), "2^34")


def test_nothing_to_do(lib):
    for entry, args in (("pjx_write_pages", _write(B=0, k=None, v=None, out=None)), ("pjx_read_pages", _read(L=0, k=None)),
                        ("pjx_read_pages", _read(B=0)), ("pjx_paged_decode", _decode(B=0, q=None, o=None))):
        assert getattr(lib, entry)(*args.values()) == 0, lib.pjx_last_error()
        assert native.last_launches() == []


def test_workspace_size_grows_with_what_is_joined(lib):
    size = lib.pjx_paged_decode_workspace_size
    assert size(2, 8, 4, 4096, 128) < size(2, 8, 8, 4096, 128) and size(2, 8, 4, 4096, 64) < size(2, 8, 4, 4096, 128)
    # a partial result of every share (2048 over the heads at most) and sequence, and 16 bytes
    assert size(32, 8, 4, 8192, 128) == (2048 // 8 + 32) * 8 * 4 * (128 + 2) * 4 + 16
