"""Lengths and parents in every form that the operators over a KV cache take."""

import pytest

pytestmark = pytest.mark.gpu


def test_lengths_as_a_column(device):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights, evict_keys, mha, tree_attention

    g = torch.Generator(device=device).manual_seed(0)
    q, k, v = (torch.randn((2, n, h, 64), generator=g, device=device).to(torch.bfloat16)
               for n, h in ((3, 4), (90, 2), (90, 2)))
    p = torch.randn((2, 90, 4, 64), generator=g, device=device).to(torch.bfloat16)
    w = torch.rand((2, 2, 90), generator=g, device=device)
    L = torch.tensor([80, 7], device=device)

    def calls(L):
        causal = masks.CausalMask() & masks.KVLenMask(L)
        yield tree_attention(q, k, v, parents=[-1, 0, 0], kv_lengths=L)
        yield from attention_with_key_weights(q, k, v, w, mask=masks.KVLenMask(L))
        yield from attention_with_key_weights(p, k, v, w, mask=causal)
        yield mha(p, k, v, mask=causal)
        yield from evict_keys(k, v, w, 20, kv_lengths=L)

    column, flat = list(calls(L[:, None])), list(calls(L))
    assert len(column) == len(flat) == 11
    for a, b in zip(column, flat):
        assert torch.equal(a, b)
