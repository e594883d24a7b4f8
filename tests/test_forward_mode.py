"""Forward-mode derivatives on the CPU: the entry points below are given tensors
that carry a tangent but require no gradient, with the kernel launches replaced
by torch operations.  ``rotary`` supplies the tangent, everything else refuses."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from probjax_amd import attention as A
from probjax_amd import hip_attention as hip
from probjax_amd import masks


def _turn(q, k, positions, sections, base, interleaved, shared_spectrum, inverse=False):
    """Rotation of one axis, interleaved, in the place of the launch; counts calls."""
    _turn.calls += 1

    def one(x):
        if x is None:
            return None
        x = x.detach()
        d = x.shape[-1]
        angle = positions.double() * float(base) ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        angle = (-angle if inverse else angle).reshape(-1, 1, d // 2)
        z = torch.polar(torch.ones_like(angle), angle) * torch.view_as_complex(x.double().unflatten(-1, (-1, 2)).contiguous())
        return torch.view_as_real(z).flatten(-2).to(x.dtype)

    return one(q), one(k)


@pytest.fixture
def turn(monkeypatch):
    _turn.calls = 0
    monkeypatch.setattr(hip, "rotary", _turn)
    return _turn


def _rand(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape)), dtype=torch.float64)


def test_rotary_turns_the_tangents(turn):
    q, k, dq, dk = _rand(2, 5, 3, 8), _rand(2, 5, 1, 8), _rand(2, 5, 3, 8) + 1, _rand(2, 5, 1, 8) - 1
    pos = torch.arange(5)
    want_q, want_k = A.rotary(dq, dk, pos)
    turn.calls = 0
    with fwd.dual_level():
        y, z = A.rotary(fwd.make_dual(q, dq), fwd.make_dual(k, dk), pos)
        assert turn.calls == 2  # the values in one launch, the tangents in another
        assert torch.equal(fwd.unpack_dual(y).tangent, want_q) and torch.equal(fwd.unpack_dual(z).tangent, want_k)
        assert torch.equal(fwd.unpack_dual(y).primal, A.rotary(q, None, pos))
        y, z = A.rotary(q, fwd.make_dual(k, dk), pos)  # one of them alone
        assert torch.equal(fwd.unpack_dual(z).tangent, want_k) and not fwd.unpack_dual(y).tangent.any()
        y, z = A.rotary(fwd.make_dual(q, dq), k, pos)
        assert torch.equal(fwd.unpack_dual(y).tangent, want_q) and not fwd.unpack_dual(z).tangent.any()
        with torch.no_grad():  # which ends reverse mode alone
            assert torch.equal(fwd.unpack_dual(A.rotary(fwd.make_dual(q, dq), None, pos)).tangent, want_q)


def test_rotary_forward_over_reverse_and_reverse_over_forward(turn):
    q, dq, pos = _rand(1, 4, 2, 6), _rand(1, 4, 2, 6) + 1, torch.arange(4)
    x = q.clone().requires_grad_()
    with fwd.dual_level():
        y = A.rotary(fwd.make_dual(x, dq), None, pos)
        (g,) = torch.autograd.grad((y ** 2).sum(), x)
        # a rotation keeps norms: the gradient is 2 x, its tangent 2 dq
        assert torch.allclose(fwd.unpack_dual(g).primal, 2 * q) and torch.allclose(fwd.unpack_dual(g).tangent, 2 * dq)
    t = dq.clone().requires_grad_()
    with fwd.dual_level():
        tangent = fwd.unpack_dual(A.rotary(fwd.make_dual(q, t), None, pos)).tangent
        (g,) = torch.autograd.grad((tangent ** 2).sum(), t)
    assert torch.allclose(g, 2 * dq)
    eps = 1e-6  # against differences
    with fwd.dual_level():
        tangent = fwd.unpack_dual(A.rotary(fwd.make_dual(q, dq), None, pos)).tangent
    diff = (A.rotary(q + eps * dq, None, pos) - A.rotary(q - eps * dq, None, pos)) / (2 * eps)
    assert (diff - tangent).abs().max() <= 1e-8


def _on_gpu(monkeypatch):
    monkeypatch.setattr(hip, "_gpu", lambda *ts: 0)


@pytest.mark.parametrize("which", ["q", "k", "v", "weights"])
def test_operators_without_a_gradient_refuse_tangents(monkeypatch, which):
    _on_gpu(monkeypatch)
    x = dict(q=_rand(1, 2, 2, 64).float(), k=_rand(1, 9, 2, 64).float(), v=_rand(1, 9, 2, 64).float(),
             weights=_rand(1, 2, 9).float())
    with fwd.dual_level(), torch.no_grad():
        x[which] = fwd.make_dual(x[which], torch.ones_like(x[which]))
        q, k, v, w = x.values()
        calls = [lambda: A.attention_with_key_weights(q, k, v, w),
                 lambda: A.attention_with_key_weights(q, k, v, w, mask=masks.CausalMask())]
        if which != "weights":
            calls.append(lambda: A.tree_attention(q, k, v, parents=[-1, 0]))
        if which != "q":
            calls.append(lambda: A.evict_keys(k, v, w, 5))
        for call in calls:
            with pytest.raises(ValueError, match="no gradient"):
                call()


def test_rotary_refuses_a_tangent_of_the_positions(turn):
    with fwd.dual_level():
        pos = fwd.make_dual(torch.rand(4), torch.ones(4))
        with pytest.raises(ValueError, match="no gradient in the positions"):
            A.rotary(_rand(1, 4, 2, 6), None, pos)


def test_functions_without_a_forward_rule_raise(monkeypatch):
    """The attention entry points have a gradient but no forward-mode rule: a tangent
    takes their autograd function, which raises, and is not dropped."""
    x = torch.ones(3)
    assert not A._needs_grad(x)
    with fwd.dual_level(), torch.no_grad():
        d = fwd.make_dual(x, x)
        assert A._needs_grad(x, d) and not A._needs_grad(x)
    q = _rand(1, 3, 2, 64).float()
    monkeypatch.setattr(hip, "flash_attention_fwd", lambda q, *a, **kw: (q.detach().clone(), q.new_zeros(1, 2, 3)))
    monkeypatch.setattr(A, "hip_device", lambda t: True)
    with fwd.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
            A.mha(fwd.make_dual(q, torch.ones_like(q)), q, q)
