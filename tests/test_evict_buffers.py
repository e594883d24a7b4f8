"""Which buffers ``evict_keys`` may write to (host logic, no GPU needed): memory is
compared as the views reach it, not as it was allocated."""

import random

import pytest
import torch

from probjax_amd import hip_attention as hip

B, S, H, D, KEEP = 2, 30, 2, 8, 10


def _inputs(dtype=torch.bfloat16):
    return torch.zeros((B, S, H, D), dtype=dtype), torch.zeros((B, S, H, D), dtype=dtype), torch.zeros((B, H, S))


def _room(C=KEEP):
    return (torch.zeros((B, C, H, D), dtype=torch.bfloat16), torch.zeros((B, C, H, D), dtype=torch.bfloat16),
            torch.zeros((B, H, C)))


def _halves(axis, shape=(B, 12, H, D), dtype=torch.bfloat16):
    """Two buffers of one allocation that lies with the pair's axis at ``axis``."""
    pool = torch.zeros((*shape[:axis], 2, *shape[axis:]), dtype=dtype)
    return pool.select(axis, 0), pool.select(axis, 1)


@pytest.mark.parametrize("axis", [0, 1, 2, 3])
def test_disjoint_views_of_one_allocation_are_taken(axis):
    k, v = _halves(axis)
    hip._check_evict_out((k, v, torch.zeros((B, H, 12))), _inputs(), KEEP)


def test_a_spare_part_of_the_inputs_allocation_is_taken():
    w = torch.zeros((B, H, 12))
    for pool in (torch.zeros((2, B, S + 12, H, D), dtype=torch.bfloat16),
                 torch.zeros((B, S + 12, 2, H, D), dtype=torch.bfloat16).permute(2, 0, 1, 3, 4),
                 torch.zeros((2, B, H, S + 12, D), dtype=torch.bfloat16).transpose(2, 3)):
        ins, out = pool[:, :, :S], pool[:, :, S:]
        hip._check_evict_out((out[0], out[1], w), (ins[0], ins[1], torch.zeros((B, H, S))), KEEP)
        layers = pool.new_zeros((3, *pool.shape))  # every layer's caches in one tensor
        hip._check_evict_out((layers[1, 0, :, :12], layers[1, 1, :, :12], w),
                             (layers[0, 0, :, :S], layers[0, 1, :, :S], torch.zeros((B, H, S))), KEEP)


def test_views_that_meet_are_refused():
    k, v, w = _inputs()
    ko, vo, wo = _room()
    _, v12, w12 = _room(12)
    pool = torch.zeros((B, 40, H, D), dtype=torch.bfloat16)
    floats = torch.zeros((B * H * (S + 12),))
    cases = [
        ((ko, ko, wo), (k, v, w)),
        ((k[:, :12], v12, w12), (k, v, w)),
        ((ko, v[:, 20:], wo), (k, v, w)),
        ((pool[:, 28:], v12, w12), (pool[:, :S], v, w)),            # two slots in common
        ((pool[:, :10], pool[:, 9:19], wo), (k, v, w)),
        ((ko, vo, floats[B * H * S - 1:][:B * H * KEEP].view(B, H, KEEP)), (k, v, floats[:B * H * S].view(B, H, S))),
        ((floats.view(torch.bfloat16)[:B * KEEP * H * D].view(B, KEEP, H, D), vo, wo),
         (k, v, floats[:B * H * S].view(B, H, S))),                 # another type over the same bytes
    ]
    for out, ins in cases:
        with pytest.raises(ValueError, match="share memory"):
            hip._check_evict_out(out, ins, KEEP)


@pytest.mark.parametrize("stride", [(0, 16, 8, 1), (16, 16, 8, 1), (100, 16, 8, 1), (160, 12, 8, 1), (160, 16, 4, 1)])
def test_buffers_whose_rows_overlap_each_other_are_refused(stride):
    """Two rows would be written to one place, in an order that is not defined."""
    k, v, w = _room()
    wide = torch.as_strided(torch.zeros(1000, dtype=torch.bfloat16), (B, KEEP, H, D), stride)
    for out in ((wide, v, w), (k, wide, w)):
        with pytest.raises(ValueError, match="overlap"):
            hip._check_evict_out(out, _inputs(), KEEP)
    for t in (torch.zeros((KEEP, H, B, D), dtype=torch.bfloat16).permute(2, 0, 1, 3),
              torch.zeros((B, 40, H, 24), dtype=torch.bfloat16)[:, 3:23:2, :, 8:16]):
        hip._check_evict_out((t, v, w), _inputs(), KEEP)


def test_shared_bytes_of_random_views():
    """Against the bytes themselves."""
    rng = random.Random(0)
    pool = torch.zeros(600, dtype=torch.int16)
    seen = set()
    for _ in range(3000):
        views = []
        for _ in range(2):
            shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 4))]
            stride = [rng.choice((0, 1, 2, 3, 5, 8, 16, 40)) for _ in shape]
            views.append(torch.as_strided(pool, shape, stride, rng.randint(0, 99)))
        sets = [_offsets(v) for v in views]
        want = bool(sets[0] & sets[1])
        assert hip._share_bytes(*views) == want, [(v.shape, v.stride(), v.storage_offset()) for v in views]
        seen.add(want)
    assert seen == {True, False}


def _offsets(t):
    offsets = {t.storage_offset()}
    for n, s in zip(t.shape, t.stride()):
        offsets = {o + i * s for o in offsets for i in range(n)}
    return offsets
