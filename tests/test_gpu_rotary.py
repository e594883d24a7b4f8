"""Rotary positions against complex rotation in float64.

Tolerances.  An angle is exact to float64; its cosine and sine are off by pi 2^-24
(the turn's rounding to float32) and 2^-23 (theirs), the two products and their
sum by 3 2^-24 more: together below 2^-21 of |a| + |b|.  The result is rounded
once, half a step of the type.
"""

import numpy as np
import pytest

from oracle import cache_ops as ref
from tests._helpers import to_np
from tests.test_gpu_tree_attention import _half_step, _types

pytestmark = pytest.mark.gpu


def _close(got, x, want, dtype, np_, sections, interleaved, shared):
    """|error| <= 2^-21 (|a| + |b|) + half a step; |a| + |b| from the norm of a
    pair, which the rotation keeps: at most sqrt(2) times it."""
    norm = np.hypot(want, _partner(want, sections, interleaved, shared))
    tol = 2.0 ** -21 * 1.5 * norm + (_half_step(dtype) + 2.0 ** -24) * np.abs(want)
    err = np.abs(to_np(got) - want)
    bad = ~(err <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5])
    assert np.array_equal(to_np(got)[..., sum(sections):], to_np(x)[..., sum(sections):])


def _partner(x, sections, interleaved, shared):
    at = np.arange(x.shape[-1])
    lo = 0
    for d in ([sum(sections)] if shared else sections):
        i = np.arange(d)
        at[lo:lo + d] = lo + ((i ^ 1) if interleaved else (i + d // 2) % max(d, 1))
        lo += d
    return x[..., at]


CASES = [
    # dtype, B, T, Hq, Hk, D, sections, far, batch positions
    ("bf16", 2, 7, 4, 2, 64, (64,), 100, True),
    ("bf16", 1, 1, 32, 8, 128, (128,), 1000000, True),        # one token, far away
    ("bf16", 1, 300, 3, 3, 128, (32, 48, 48), 200, False),
    ("f16", 2, 33, 4, 1, 96, (32, 32, 32), 50, True),
    ("f16", 3, 5, 2, 2, 80, (26, 26, 26), 5000, True),        # halves that are no whole chunks
    ("bf16", 1, 40, 5, 0, 128, (42, 42, 42), 300, True),      # no k
    ("bf16", 2, 9, 2, 1, 64, (8, 0, 16, 4), 1000, False),     # four axes, one of no features, a rest that passes
    ("f32", 2, 50, 4, 2, 64, (64,), 100000, True),
    ("f32", 1, 20, 3, 2, 40, (20, 20), 64, True),
    ("f32", 1, 20, 3, 2, 256, (84, 86, 86), 64, True),
    ("bf16", 2, 11, 3, 1, 50, (50,), 64, True),               # rows that are no whole chunks
    ("f32", 2, 11, 3, 1, 7, (2, 4), 64, True),
    ("bf16", 1, 5000, 1, 1, 64, (64,), 5000, False),
]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_forward_and_gradient(device, case, shared, interleaved):
    import torch
    from probjax_amd.attention import rotary

    name, B, T, Hq, Hk, D, sections, far, batched = case
    dtype = _types()[name]
    g = torch.Generator(device=device).manual_seed(T + D)
    q, dq = (torch.randn((B, T, Hq, D), generator=g, device=device).to(dtype) for _ in range(2))
    k, dk = (torch.randn((B, T, Hk, D), generator=g, device=device).to(dtype) if Hk else None for _ in range(2))
    shape = ((B,) if batched else ()) + (T, len(sections))
    pos = torch.randint(0, far + 1, shape, generator=g, device=device)
    kw = dict(sections=sections, interleaved=interleaved, shared_spectrum=shared)
    print(f"rotary {case} {shared} {interleaved}", flush=True)
    q.requires_grad_()
    ins = [q] if k is None else [q, k.requires_grad_()]
    outs = rotary(q, k, pos, **kw)
    outs = [outs] if k is None else list(outs)
    grads = torch.autograd.grad(outs, ins, [dq] if k is None else [dq, dk])
    torch.cuda.synchronize()
    p = np.broadcast_to(pos.cpu().numpy(), (B, T, len(sections)))
    rule = dict(sections=sections, interleaved=interleaved, shared_spectrum=shared)
    for x, y, d, dx in zip(ins, outs, (dq, dk), grads):
        args = (dtype, None, sections, interleaved, shared)
        _close(y, x, ref.rotary(to_np(x), p, **rule), *args)
        _close(dx, d, ref.rotary(to_np(d), p, sign=-1, **rule), *args)
    with torch.no_grad():  # the same without a graph
        again = rotary(q, k, pos, **kw)
        assert all(torch.equal(a, b) for a, b in zip([again] if k is None else again, outs))


def test_gradient_against_differences(device):
    """The rotation is linear: <dy, f(x + d) - f(x)> = <f'(dy), d>."""
    import torch
    from probjax_amd.attention import rotary

    g = torch.Generator(device=device).manual_seed(1)
    x, d, dy = (torch.randn((2, 30, 3, 64), generator=g, device=device) for _ in range(3))
    pos = torch.randint(0, 5000, (2, 30, 2), generator=g, device=device)
    kw = dict(sections=(24, 40), interleaved=False)
    x.requires_grad_()
    y = rotary(x, None, pos, **kw)
    (gx,) = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        diff = (rotary(x + d, None, pos, **kw).double() - y.double())
    left, right = (dy.double() * diff).sum(), (gx.double() * d.double()).sum()
    # each of the n terms is off by at most 2^-21 (|a| + |b|) twice: 2^-19 |dy| (|x| + |d|)
    lim = 2.0 ** -19 * (dy.abs() * (x.abs() + d.abs())).double().sum()
    assert abs(left - right) <= lim < abs(right) / 10  # (the bound tells a wrong gradient from a right one)


def test_second_derivative_and_partial_gradients(device):
    import torch
    from probjax_amd.attention import rotary

    q = torch.randn((1, 6, 2, 32), device=device, requires_grad=True)
    k = torch.randn((1, 6, 1, 32), device=device, requires_grad=True)
    pos = torch.arange(6, device=device)
    y, z = rotary(q, k, pos)
    (gk,) = torch.autograd.grad((z * z).sum(), k, create_graph=True, retain_graph=True)
    assert torch.allclose(gk, 2 * k, rtol=1e-5, atol=1e-5)  # a rotation keeps norms
    (hk,) = torch.autograd.grad(gk.sum(), k, retain_graph=True)
    assert torch.allclose(hk, torch.full_like(k, 2.0), rtol=1e-5, atol=1e-5)
    (gq,) = torch.autograd.grad(y.sum(), q)
    assert torch.equal(gq, torch.autograd.grad(rotary(q, None, pos).sum(), q)[0])
    shared = torch.randn((1, 6, 1, 32), device=device, requires_grad=True)  # one head broadcast to four
    out = rotary(shared.expand(1, 6, 4, 32), None, pos)
    (gs,) = torch.autograd.grad(out.sum(), shared)
    (g1,) = torch.autograd.grad(rotary(shared, None, pos).sum(), shared)
    assert torch.allclose(gs, 4 * g1, rtol=1e-6, atol=1e-5)


def test_strides_positions_and_slices(device):
    """Any order of axes, a slice of the features read in place, every type of
    position; what another call gives on copies, bit for bit."""
    import torch
    from probjax_amd.attention import rotary

    g = torch.Generator(device=device).manual_seed(3)
    q = torch.randn((2, 4, 20, 128), generator=g, device=device).to(torch.bfloat16).transpose(1, 2)
    k = torch.randn((2, 20, 2, 576), generator=g, device=device).to(torch.bfloat16)[..., 512 - 64:512 + 64]
    pos = torch.randint(0, 900, (2, 20, 3), generator=g, device=device)
    kw = dict(sections=(32, 48, 48))
    want = rotary(q.contiguous(), k.contiguous(), pos, **kw)
    odd = torch.empty((2, 20, 2, 131), dtype=torch.bfloat16, device=device)[..., 1:129].copy_(k)
    for qq, kk in ((q, k), (q, odd), (q.contiguous(), k)):
        for p in (pos, pos.int(), pos.float(), pos.double(), pos.permute(2, 0, 1).contiguous().permute(1, 2, 0),
                  pos.short()):
            got = rotary(qq, kk, p, **kw)
            assert all(torch.equal(a, b) and a.is_contiguous() for a, b in zip(got, want))
    one = rotary(q, k, pos[:1].expand(2, 20, 3), **kw)
    assert all(torch.equal(a, b) for a, b in zip(one, rotary(q, k, pos[0], **kw)))
    f = torch.rand((20, 1), device=device) * 300  # positions between patches
    got = rotary(q, None, f)
    _close(got, q, ref.rotary(to_np(q), np.broadcast_to(f.double().cpu().numpy(), (2, 20, 1)), (128,)),
           torch.bfloat16, None, (128,), True, False)


def test_follows_the_pair_convention(device):
    """The reference's own rotation (oracle.apply_rotary) on one axis."""
    import oracle
    import torch
    from probjax_amd.attention import rotary

    x = np.random.default_rng(0).standard_normal((1, 9, 2, 64)).astype(np.float32)
    got = rotary(torch.from_numpy(x).to(device), None, torch.arange(9, device=device))
    want = oracle.apply_rotary(x, np.arange(9))
    # the oracle's float32 angles (below 9) are off by 2 steps: 9 2^-23 of |a| + |b|
    assert np.abs(to_np(got) - want).max() <= 12 * 2.0 ** -23 * 2 * np.abs(x).max()


def test_features_that_pass_may_hold_anything(device):
    import torch
    from probjax_amd.attention import rotary

    for interleaved in (True, False):
        x = torch.randn((1, 4, 2, 64), device=device)
        want = rotary(x, None, torch.arange(4), sections=(32,), interleaved=interleaved)
        x[..., 32:] = float("nan")
        x[..., 40] = float("inf")
        got = rotary(x, None, torch.arange(4), sections=(32,), interleaved=interleaved)
        assert torch.equal(got[..., :32], want[..., :32])
        assert torch.isinf(got[..., 40]).all() and torch.isnan(got[..., 41:]).all()


def test_replayed_graph_with_gradients(device):
    import torch
    from probjax_amd.attention import rotary

    q = torch.randn((2, 50, 4, 64), device=device, requires_grad=True)
    k = torch.randn((2, 50, 2, 64), device=device, requires_grad=True)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    pos = torch.randint(0, 99, (50, 2), device=device)

    def step():
        y, z = rotary(q, k, pos, sections=(24, 40))
        return (y, z, *torch.autograd.grad((y, z), (q, k), (dq, dk)))

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        torch.manual_seed(i)
        with torch.no_grad():
            for x in (q, k, dq, dk):
                x.copy_(torch.randn(x.shape, device=device))
            pos.copy_(torch.randint(0, 99, (50, 2), device=device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step())), i


def test_rejects(device):
    import torch
    from probjax_amd.attention import rotary

    q = torch.zeros((2, 5, 4, 64), device=device)
    pos = torch.arange(5, device=device)
    bad = [
        (lambda: rotary(q[0], None, pos), "must be"),
        (lambda: rotary(q, q[:, :4], pos), "incompatible"),
        (lambda: rotary(q, q.half(), pos), "incompatible"),
        (lambda: rotary(q, None, pos[:4]), "positions"),
        (lambda: rotary(q, None, pos[:, None].expand(5, 5)), "positions"),
        (lambda: rotary(q, None, pos.bool()), "integers or floats"),
        (lambda: rotary(q, None, pos.float().requires_grad_()), "no gradient in the positions"),
        (lambda: rotary(q, None, pos, sections=(32, 32)), "sections"),
        (lambda: rotary(q, None, pos, sections=(33,)), "sections"),
        (lambda: rotary(q, None, pos, sections=(66,)), "sections"),
        (lambda: rotary(q, None, pos[:, None].expand(5, 3)), "give sections"),
        (lambda: rotary(q, None, pos, base=0.0), "base"),
        (lambda: rotary(q.int(), None, pos), "dtype"),
        (lambda: rotary(q.cpu(), None, pos.cpu()), "ROCm device"),
        (lambda: rotary(q.new_zeros((1, 5, 1, 300)), None, pos), "head dims"),
    ]
    for call, msg in bad:
        with pytest.raises(ValueError, match=msg):
            call()
    assert rotary(q[:, :0], None, pos[:0]).shape == (2, 0, 4, 64)
    y, z = rotary(q[:, :, :0], q, pos)
    assert y.shape == (2, 5, 0, 64) and torch.equal(z, q)
