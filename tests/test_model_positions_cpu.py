"""Positions that a model's table does not have are refused, as indexing the table refuses them."""
import pytest
import torch

from mist_b200.modules.layers import VocabParallelEmbedding
from mist_b200.ops import functional as F


def _module():
    torch.manual_seed(1)
    return VocabParallelEmbedding(11, 8, max_position_embeddings=7)


@pytest.mark.parametrize("bad", [7, -8, 2 ** 40])
def test_explicit_positions_outside_the_table(bad):
    m, ids = _module(), torch.zeros(2, 3, dtype=torch.long)
    with pytest.raises(IndexError):
        m(ids, position_ids=torch.tensor([[0, 1, bad]]))
    with pytest.raises(IndexError):
        F.embedding(ids, m.word_embeddings.weight, m.position_embeddings.weight,
                    position_ids=torch.tensor([[0, 1, bad]]), strict_positions=True)


def test_negative_positions_count_from_the_end():
    m, ids = _module(), torch.tensor([[1, 2, 3], [4, 5, 6]])
    pos = torch.tensor([[-1, 0, -7], [6, -2, 3]])
    out, want = m(ids, position_ids=pos), m.word_embeddings.weight[ids] + m.position_embeddings.weight[pos]
    assert torch.allclose(out, want, atol=1e-6)
    g = torch.randn_like(out)
    leaves = (m.word_embeddings.weight, m.position_embeddings.weight)
    for a, b in zip(torch.autograd.grad(out, leaves, g), torch.autograd.grad(want, leaves, g)):
        assert torch.allclose(a, b, atol=1e-6)


def test_no_tokens():
    assert _module()(torch.zeros(2, 0, dtype=torch.long), position_ids=torch.zeros(2, 0, dtype=torch.long)).shape == (2, 0, 8)


def _gpt(**more):
    from tests.test_packed_training_cpu import build
    return build("gpt", **more)


def test_documents_longer_than_the_table():
    """A table of 32 rows: documents of 33 tokens are refused as rows of 33 are; rows behind the last document are not."""
    model, ids = _gpt(), torch.randint(0, 250, (1, 52))
    for offsets in ([0, 52], torch.tensor([0, 10, 43, 52])):
        with pytest.raises(ValueError, match="32"):
            model(ids, attention_mask=F.PackedSequences(offsets))
    assert model(ids, attention_mask=F.PackedSequences([0, 32, 52])).shape[:2] == (1, 52)
    packed, alone = model(ids, attention_mask=F.PackedSequences([0, 10], 52)), model(ids[:, :10])
    assert torch.allclose(packed[:, :10], alone, atol=1e-5)
    with pytest.raises(ValueError):
        model(ids)


def test_documents_of_any_length_without_a_table():
    from tests.test_packed_training_cpu import build
    ids = torch.randint(0, 250, (1, 52))
    assert build("llama")(ids, attention_mask=F.PackedSequences([0, 52])).shape[:2] == (1, 52)


def test_generation_behind_the_table():
    """32 rows: a prompt of 30 leaves room for three tokens (the last one is not fed back); an end before it is no error."""
    from mist_b200.inference import generate
    model, ids = _gpt(), torch.randint(0, 250, (1, 30), generator=torch.Generator().manual_seed(3))
    out = generate(model, ids, 3)
    assert out.shape == (1, 33)
    with pytest.raises(IndexError):
        generate(model, ids, 6)
    with pytest.raises(IndexError):
        generate(model, torch.cat([ids, ids], 1), 1)
    assert generate(model, ids, 6, eos_token_id=int(out[0, 32])).shape[1] <= 33


def test_the_status_of_a_position_has_a_name():
    from mist_b200.ops import native
    assert "position" in native.status_message(6) and "unknown" in native.status_message(7)
    assert "peer flag" in native.status_message(4)


@pytest.mark.parametrize("rank", [0, 1])
def test_every_rank_refuses_what_the_first_one_refuses(rank):
    """Only the first rank adds positions; the others must not wait for it in the sum behind the lookup."""
    from mist_b200.parallel.dist_ops import FakeGroup
    m = VocabParallelEmbedding(12, 8, max_position_embeddings=7, process_group=FakeGroup(2, rank))
    ids = torch.zeros(2, 9, dtype=torch.long)
    with pytest.raises(IndexError):
        m(ids[:, :3], position_ids=torch.tensor([[0, 1, 7]]))
    with pytest.raises(ValueError, match="7"):
        m(ids, position_ids=F.PackedSequences([0, 8, 18]))
