"""Lengths and parents as the operators over a KV cache take them (host logic, no
GPU needed)."""

import pytest
import torch

from probjax_amd import hip_attention as hip

LIKE = torch.zeros(1)


@pytest.mark.parametrize("lengths", [
    [3, 8], torch.tensor([3, 8]), torch.tensor([[3], [8]]), [[3], [8]], torch.tensor([[3, 8]], dtype=torch.int16),
    torch.tensor([3, 0, 8, 0], dtype=torch.int32)[::2],
])
def test_lengths_of_a_batch(lengths):
    got = hip._key_lengths(lengths, LIKE, 2)
    assert got.dtype == torch.int32 and got.is_contiguous() and got.shape == (2,) and got.tolist() == [3, 8]


def test_lengths_of_another_batch_are_refused():
    assert hip._key_lengths(None, LIKE, 2) is None
    for bad in ([1, 2, 3], torch.ones((2, 2), dtype=torch.int32), 5):
        with pytest.raises(ValueError, match="kv_lengths must have shape"):
            hip._key_lengths(bad, LIKE, 2)
    for bad in ([1.0, 2.0], torch.tensor([True, False])):
        with pytest.raises(ValueError, match="integers"):
            hip._key_lengths(bad, LIKE, 2)
