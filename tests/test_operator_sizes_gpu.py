"""Sizes that 32 bits do not hold are refused before anything is launched (the views here take no memory)."""
import pytest
import torch

from mist_b200.ops import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
BIG = 2 ** 31


@pytest.mark.parametrize("positions", [False, True])
def test_embedding_of_too_many_tokens(positions):
    ids = torch.zeros(1, 1, dtype=torch.long, device=DEV).expand(BIG // 8, 8)
    wte = torch.zeros(4, 8, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="32 bits"):
        F.embedding(ids, wte, wte.clone() if positions else None, position_ids=ids[:1] if positions else None)


def test_vocabulary_loss_of_too_many_rows():
    x = torch.zeros(1, 8, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="32 bits"):
        F.linear_cross_entropy(x.expand(BIG, 8), x, torch.zeros(1, dtype=torch.long, device=DEV).expand(BIG))


def test_packing_of_too_many_rows():
    with pytest.raises(ValueError, match="32 bits"):
        F.PackedSequences(torch.zeros(2, dtype=torch.int32, device=DEV), BIG)
    x = torch.zeros(1, 2, 16, device=DEV, dtype=torch.bfloat16).expand(BIG, 2, 16)
    with pytest.raises(ValueError, match="32 bits"):
        F.attention_varlen(x, x, x, [0, 1])


def test_rows_further_apart_than_32_bits():
    """Such a view is copied: its stride does not reach the kernels cut off."""
    from mist_b200.ops.linear_xent import _rows
    wide = torch.as_strided(torch.zeros(8, device=DEV, dtype=torch.bfloat16), (1, 8), (BIG, 1))
    assert _rows(wide, 8).stride(0) == 8
