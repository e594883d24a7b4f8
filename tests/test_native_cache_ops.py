"""Refusals of the cache and position operators' entry points: every argument is
checked before any HIP call, so this runs without a GPU (the pointers are never
followed)."""

import ctypes

import pytest

from probjax_amd import native

P = ctypes.c_void_p
BF16, F32 = native.PJX_DTYPE_BF16, native.PJX_DTYPE_F32


@pytest.fixture(scope="module")
def lib():
    return native.load()


def refused(lib, entry, args, msg, code=1):
    rc = getattr(lib, entry)(*args.values())
    assert rc == code, (rc, lib.pjx_last_error())
    assert msg in lib.pjx_last_error().decode(), lib.pjx_last_error()


def _tree(**over):
    a = dict(dtype=BF16, q=P(16), k=P(16), v=P(16), lengths=None, parents=P(16), mask=None, trees=1, o=P(16), lse=None,
             ws=P(16), ws_bytes=1 << 30, B=2, T=4, S=100, Hq=4, Hkv=2, D=64, row=64, strides=None, scale=0.1, chunk=0,
             stream=None)
    return {**a, **over}


@pytest.mark.parametrize("over,msg,code", [
    (dict(dtype=9), "dtype", 1),
    (dict(q=None), "null", 1),
    (dict(k=P(8)), "16 bytes", 1),
    (dict(T=257), "256", 1),
    (dict(T=0), "bad sizes", 1),
    (dict(Hq=3), "bad sizes", 1),
    (dict(D=96), "head_dim", 1),
    (dict(row=60), "row_dim", 1),
    (dict(D=256, row=128), "row_dim", 1),
    (dict(dtype=F32, row=40), "row_dim", 1),
    (dict(scale=0.0), "sm_scale", 1),
    (dict(chunk=100), "chunk", 1),
    (dict(parents=None), "parents or tree_mask", 1),
    (dict(mask=P(16)), "not both", 1),
    (dict(trees=3), "one tree", 1),
    (dict(S=3), "hold the drafted", 1),
    (dict(S=1 << 31), "out of range", 1),
    (dict(strides=native.CacheStrides(100, 64, 4, 100, 64, 64)), "16-byte", 1),
    (dict(strides=native.CacheStrides(-64, 64, 64, 64, 64, 64)), "out of range", 1),
    (dict(ws=None), "workspace", 3),
    (dict(ws_bytes=100), "workspace", 3),
])
def test_tree_decode(lib, over, msg, code):
    refused(lib, "pjx_tree_decode", _tree(**over), msg, code)


def test_tree_decode_of_nothing(lib):
    assert lib.pjx_tree_decode(*_tree(B=0, q=None, k=None, v=None, o=None).values()) == 0
    assert native.last_launches() == []


def _weighted(**over):
    a = dict(dtype=BF16, q=P(16), k=P(16), v=P(16), lengths=None, w=None, w_out=P(16), o=P(16), lse=None, ws=P(16),
             ws_bytes=1 << 30, B=2, T=4, S=100, Hq=4, Hkv=2, D=64, row=64, strides=None, scale=0.1, chunk=0,
             stream=None)
    return {**a, **over}


@pytest.mark.parametrize("over,msg,code", [
    (dict(w_out=None), "null", 1),
    (dict(T=33), "64 rows", 1),
    (dict(D=80), "head_dim", 1),
    (dict(ws=P(8)), "16 bytes", 1),
    (dict(ws_bytes=1000), "workspace", 3),
])
def test_weighted_decode(lib, over, msg, code):
    refused(lib, "pjx_weighted_decode", _weighted(**over), msg, code)


def test_weighted_decode_workspace(lib):
    part = lib.pjx_decode_workspace_size(2, 3, 5, 101, 64, 128)
    assert lib.pjx_weighted_decode_workspace_size(2, 3, 5, 101, 64, 128) == (part + 255) // 256 * 256 + 2 * 3 * 5 * 104 * 4


def _weights(**over):
    a = dict(dtype=BF16, q=P(16), k=P(16), lse=P(16), lengths=None, w=None, w_out=P(16), ws=P(16), ws_bytes=1 << 30,
             B=2, T=4, S=100, Hq=4, Hkv=2, D=64, row=64, causal=1, shift=0, scale=0.1, stream=None)
    return {**a, **over}


@pytest.mark.parametrize("over,msg,code", [
    (dict(lse=None), "null", 1),
    (dict(dtype=5), "dtype", 1),
    (dict(dtype=F32, row=32), "row_dim", 1),
    (dict(row=65), "row_dim", 1),
    (dict(D=72), "head_dim", 1),
    (dict(Hkv=3), "bad sizes", 1),
    (dict(shift=1 << 30), "out of range", 1),
    (dict(q=P(2)), "16 bytes", 1),
    (dict(ws_bytes=8), "workspace", 3),
])
def test_key_weights(lib, over, msg, code):
    refused(lib, "pjx_key_weights", _weights(**over), msg, code)


def _rotary(sections=(32, 32), **over):
    a = dict(dtype=BF16, q=P(16), k=P(16), y=P(16), z=P(16), pos=P(16), pos_type=0, pb=0, pt=2, B=2, T=5, Hq=4, Hk=2,
             D=64, strides=None, sections=None if sections is None else (ctypes.c_int32 * len(sections))(*sections),
             axes=len(sections or ()), base=1e4, inter=1, shared=0, inverse=0, stream=None)
    return {**a, **over}


@pytest.mark.parametrize("args,msg", [
    (_rotary(dtype=4), "dtype"),
    (_rotary(pos_type=4), "position type"),
    (_rotary(D=300), "head_dim"),
    (_rotary((2, 2, 2, 2, 2)), "axes"),
    (_rotary(None), "axes"),
    (_rotary((33, 1)), "even"),
    (_rotary((40, 40)), "exceed"),
    (_rotary(base=0.0), "base"),
    (_rotary(base=float("nan")), "base"),
    (_rotary(y=None), "null"),
    (_rotary(z=None), "null"),
    (_rotary(q=P(17)), "aligned"),
    (_rotary(strides=native.CacheStrides(-1, 1, 1, 1, 1, 1)), "strides"),
    (_rotary(pt=-2), "strides"),
])
def test_rotary(lib, args, msg):
    refused(lib, "pjx_rotary", args, msg)


def _evict(**over):
    a = dict(size=2, k=P(16), v=P(16), w=P(16), lengths=None, ko=P(16), vo=P(16), wo=P(16), lo=P(16), index=P(16), B=2,
             S=100, H=2, D=64, C=50, keep=50, sinks=4, recent=8, strides=None, out_strides=None, fill=1, stream=None)
    return {**a, **over}


@pytest.mark.parametrize("over,msg", [
    (dict(size=8), "elem_size"),
    (dict(keep=11), "sinks + recent"),
    (dict(sinks=-1), "sinks + recent"),
    (dict(C=49), "out_len"),
    (dict(H=0), "bad sizes"),
    (dict(B=70000), "out of range"),
    (dict(index=None), "null"),
    (dict(w=None), "null"),
    (dict(k=P(17)), "aligned"),
    (dict(out_strides=native.CacheStrides(1, 1, -1, 1, 1, 1)), "strides"),
])
def test_evict_keys(lib, over, msg):
    refused(lib, "pjx_evict_keys", _evict(**over), msg)
