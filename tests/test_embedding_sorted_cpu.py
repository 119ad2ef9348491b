"""Scaled lookup with explicit positions on the reference path, and what the embedding refuses."""
import pytest
import torch

from mist_b200.modules.layers import VocabParallelEmbedding
from mist_b200.ops import functional as F


def _tables(v=11, p=7, h=8):
    torch.manual_seed(0)
    return torch.randn(v, h, requires_grad=True), torch.randn(p, h, requires_grad=True)


def test_scale_and_positions():
    wte, wpe = _tables()
    ids = torch.tensor([[1, 3, 3, 10, 2], [0, 1, 1, 1, 9]])
    pos = torch.tensor([[0, 1, 2, 0, 1], [0, 6, 7, -1, 2]])          # 7 and -1 are outside the table
    out = F.embedding(ids, wte, wpe, vocab_start=1, scale=2.5, position_ids=pos)
    loc, known = ids - 1, (pos >= 0) & (pos < 7)
    inside = (loc >= 0) & (loc < 11)
    want = 2.5 * wte[loc.clamp(0, 10)] * inside[..., None] + wpe[pos.clamp(0, 6)] * known[..., None]
    assert torch.allclose(out, want, rtol=1e-6, atol=1e-6)
    g = torch.randn_like(out)
    got, ref = torch.autograd.grad(out, (wte, wpe), g), torch.autograd.grad(want, (wte, wpe), g)
    for a, b in zip(got, ref):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-6)


def test_positions_broadcast_over_the_batch():
    wte, wpe = _tables()
    ids = torch.randint(0, 11, (3, 4))
    assert torch.equal(F.embedding(ids, wte, wpe, position_ids=torch.arange(4)), F.embedding(ids, wte, wpe))


def test_module_takes_positions():
    torch.manual_seed(1)
    m = VocabParallelEmbedding(11, 8, max_position_embeddings=7)
    ids, pos = torch.randint(0, 11, (2, 5)), torch.tensor([[0, 1, 0, 1, 2]])
    want = m.word_embeddings.weight[ids] + m.position_embeddings.weight[pos]
    assert torch.allclose(m(ids, position_ids=pos), want, atol=1e-6)


@pytest.mark.parametrize("case", ["rank", "float", "long", "positions", "shape"])
def test_refusals(case):
    wte, wpe = _tables()
    ids, pos = torch.zeros(2, 4, dtype=torch.long), None
    if case == "rank":
        ids = ids[0]
    elif case == "float":
        ids = ids.float()
    elif case == "long":
        ids = torch.zeros(1, 8, dtype=torch.long)                    # 8 positions, 7 in the table
    elif case == "positions":
        pos = torch.zeros(2, 4)
    else:
        pos = torch.zeros(3, 4, dtype=torch.long)
    with pytest.raises((ValueError, RuntimeError)):
        F.embedding(ids, wte, wpe, position_ids=pos)
