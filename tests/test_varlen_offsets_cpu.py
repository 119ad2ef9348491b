"""Offsets that packed attention refuses instead of dropping them."""
import pytest
import torch

from mist_b200.ops import functional as F


def test_offsets_of_keys_beside_a_packing():
    x = torch.randn(7, 2, 16)
    seqs = F.PackedSequences([0, 3, 7])
    with pytest.raises(ValueError):
        F.attention_varlen(x, x, x, seqs, [0, 5, 7])
    F.attention_varlen(x, x, x, seqs)


def test_offsets_that_32_bits_do_not_hold():
    with pytest.raises(ValueError):
        F.PackedSequences([0, 2 ** 31])
