"""Forward-mode derivatives on the device: ``rotary`` is linear in q and k, so a
tangent comes out as the same call gives it, bit for bit."""

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["bfloat16", "float32"])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_turns_the_tangents(device, name, interleaved):
    import torch
    import torch.autograd.forward_ad as fwd
    from probjax_amd.attention import rotary

    g = torch.Generator(device=device).manual_seed(4)
    q, dq, k, dk = (torch.randn((2, 30, h, 64), generator=g, device=device).to(getattr(torch, name)) for h in (4, 4, 2, 2))
    pos = torch.randint(0, 500, (2, 30, 2), generator=g, device=device)
    kw = dict(sections=(24, 32), interleaved=interleaved)
    want = rotary(dq, dk, pos, **kw)
    with fwd.dual_level():
        got = rotary(fwd.make_dual(q, dq), fwd.make_dual(k, dk), pos, **kw)
        got, values = [fwd.unpack_dual(x).tangent for x in got], [fwd.unpack_dual(x).primal for x in got]
        x = dq.clone().requires_grad_()
        both = fwd.unpack_dual(rotary(fwd.make_dual(q, x), k, pos, **kw)[0]).tangent
        (g,) = torch.autograd.grad(both, x, dk.new_ones(both.shape))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(values, rotary(q, k, pos, **kw)))
    assert torch.equal(both, want[0])
    assert torch.equal(g, rotary(torch.ones_like(q), None, -pos, **kw))


def test_what_has_no_forward_rule_raises(device):
    import torch
    import torch.autograd.forward_ad as fwd
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights, evict_keys, mha, tree_attention

    q, k = torch.ones((1, 3, 2, 64), device=device), torch.ones((1, 9, 2, 64), device=device)
    w = torch.zeros((1, 2, 9), device=device)
    with fwd.dual_level():
        d = fwd.make_dual(q, torch.ones_like(q))
        for call in (lambda: tree_attention(d, k, k, parents=[-1, 0, 1]), lambda: attention_with_key_weights(d, k, k, w),
                     lambda: attention_with_key_weights(d, k, k, w, mask=masks.CausalMask()),
                     lambda: evict_keys(fwd.make_dual(k, k), k, w, 4)):
            with pytest.raises(ValueError, match="no gradient"):
                call()
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
            mha(d, k, k)
