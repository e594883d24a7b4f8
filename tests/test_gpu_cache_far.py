"""Caches, inputs and buffers whose rows lie 2^24 + 8 elements apart (slices of much
longer rows): offsets pass 32 bits.  Results are those on copies that lie close
together, bit for bit."""

import pytest

pytestmark = pytest.mark.gpu

S, H, D, STEP = 150, 2, 64, 2 ** 24 + 8  # 2.5e9 elements from the first row to the last


def _far(near, step=STEP):
    """``near [1, S, H, D]`` with its rows ``step`` elements apart."""
    import torch

    n = near.shape[1]
    wide = torch.empty(((n - 1) * step + near[0, 0].numel(),), dtype=near.dtype, device=near.device)
    far = wide.as_strided(near.shape, (0, step, near.shape[3], 1))
    return far.copy_(near)


def _new(device, dtype, *shape):
    import torch

    gen = torch.Generator(device=device).manual_seed(sum(shape))
    return torch.randn(shape, generator=gen, device=device).to(dtype)


@pytest.mark.parametrize("name,stream", [("bfloat16", "0"), ("bfloat16", "1"), ("float32", "0")])
def test_decode_steps_with_weights(device, monkeypatch, name, stream):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights

    monkeypatch.setenv("PJX_DECODE_STREAM", stream)
    dtype = getattr(torch, name)
    q, k, v = _new(device, dtype, 1, 1, 8, D), _new(device, dtype, 1, S, H, D), _new(device, dtype, 1, S, H, D) + 1
    w = torch.rand((1, H, S), device=device)
    mask = masks.KVLenMask(torch.tensor([S - 1], device=device))
    want = attention_with_key_weights(q, k, v, w, mask=mask)
    far = _far(k)
    got = attention_with_key_weights(q, far, v, w, mask=mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    far.copy_(v)
    got = attention_with_key_weights(q, k, far, w, mask=mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("hq", [4, 16])  # 18 or 72 rows a KV head
def test_trees(device, hq):
    import torch
    from probjax_amd.attention import tree_attention

    q, k, v = (_new(device, torch.bfloat16, 1, n, h, D) for n, h in ((9, hq), (S, H), (S, H)))
    parents = [-1, 0, 0, 1, 1, 2, -2, 5, 7]
    far = _far(v, 2 ** 24)  # the widest step that the kernel of many rows takes
    for kw in (dict(), dict(kv_lengths=torch.tensor([100], device=device))):
        want = tree_attention(q, k, v, parents=parents, **kw)
        assert torch.equal(tree_attention(q, k, far, parents=parents, **kw), want)


@pytest.mark.parametrize("name", ["bfloat16", "float32"])
def test_eviction_from_and_into_far_rows(device, name):
    import torch
    from probjax_amd.attention import evict_keys

    dtype = getattr(torch, name)
    k, v = _new(device, dtype, 1, S, H, D), _new(device, dtype, 1, S, H, D) + 1
    w, keep = torch.rand((1, H, S), device=device), 140
    want = evict_keys(k, v, w, keep, sinks=1, recent=9)
    far = _far(k)
    got = evict_keys(far, v, w, keep, sinks=1, recent=9)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    far.zero_()
    got = evict_keys(v, k, w, keep, sinks=1, recent=9,
                     out=(torch.empty_like(v), far, torch.empty((1, H, S), device=device)))
    assert torch.equal(got.k[:, :keep], want.v) and torch.equal(far[:, :keep], want.k) and not far[:, keep:].any()


@pytest.mark.parametrize("interleaved,sections", [(True, (64,)), (False, (64,)), (False, (26, 30))])
def test_rotary(device, interleaved, sections):
    import torch
    from probjax_amd.attention import rotary

    x, y = _new(device, torch.bfloat16, 1, S, H, D), _new(device, torch.bfloat16, 1, S, 1, D)
    pos = torch.randint(0, 5000, (S, len(sections)), device=device)
    kw = dict(sections=sections, interleaved=interleaved)
    want = rotary(x, y, pos, **kw)
    assert all(torch.equal(a, b) for a, b in zip(rotary(_far(x), y, pos, **kw), want))
