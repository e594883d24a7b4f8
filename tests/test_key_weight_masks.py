"""Masks of ``attention_with_key_weights`` before any launch (no GPU needed)."""

import pytest
import torch

from probjax_amd import attention as A
from probjax_amd import hip_attention as hip
from probjax_amd import masks


@pytest.mark.parametrize("lengths", [
    torch.tensor([[3, 4], [1, 2], [1, 1]]),      # rows of three sequences
    torch.tensor([3.0, 4.0]),
    torch.ones((2, 1, 1), dtype=torch.int32),
])
def test_lengths_that_fit_no_sequence_are_refused(lengths):
    q, k = torch.zeros((2, 1, 4, 64)), torch.zeros((2, 9, 2, 64))
    with pytest.raises(ValueError, match="key lengths"):
        A.attention_with_key_weights(q, k, k, mask=masks.KeyPaddingMask(lengths))


@pytest.mark.parametrize("lengths,want", [
    (5, [5, 5]), (torch.tensor([7]), [7, 7]), (torch.tensor([[2], [9]]), [2, 9]),
])
def test_one_row_takes_its_padding_lengths(monkeypatch, lengths, want):
    seen = {}

    def decode(q, k, v, weights, *, kv_lengths, **kw):
        seen["lengths"] = kv_lengths.tolist()
        return q, weights

    monkeypatch.setattr(hip, "weighted_decode", decode)
    q, k = torch.zeros((2, 1, 4, 64)), torch.zeros((2, 9, 2, 64))
    A.attention_with_key_weights(q, k, k, mask=masks.KeyPaddingMask(lengths))
    assert seen["lengths"] == want
