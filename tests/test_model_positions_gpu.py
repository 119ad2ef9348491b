"""Positions that a model's table does not have, on the GPU: reported by a status where the host does not know them."""
import pytest
import torch

from mist_b200.modules.layers import VocabParallelEmbedding
from mist_b200.ops import functional as F
from mist_b200.ops import native

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _module(h=64):
    torch.manual_seed(1)
    return VocabParallelEmbedding(50, h, max_position_embeddings=40, device=DEV, dtype=torch.bfloat16)


@pytest.mark.parametrize("tokens", [90, 3000])
def test_negative_positions_count_from_the_end(tokens):
    """Lookup: one sum in fp32, rounded once (half a step: 2^-8).  Gradients: fp32 sums of at most 3000 values, rounded once."""
    m = _module()
    ids, pos = torch.randint(0, 50, (1, tokens), device=DEV), torch.randint(-40, 40, (1, tokens), device=DEV)
    out = m(ids, position_ids=pos)
    leaves = (m.word_embeddings.weight, m.position_embeddings.weight)
    wide = [x.detach().double().requires_grad_(True) for x in leaves]
    want = wide[0][ids] + wide[1][pos]
    g = torch.randn_like(out)
    assert ((out.double() - want).abs() <= 1.01 * 2 ** -8 * want.abs() + 1e-6).all()
    size = [torch.zeros_like(x).index_add_(0, at.reshape(-1) % x.shape[0], g[0].double().abs()) for x, at in zip(wide, (ids, pos))]
    for a, b, s in zip(torch.autograd.grad(out, leaves, g), torch.autograd.grad(want, wide, g.double()), size):
        assert ((a.double() - b).abs() <= 1.01 * 2 ** -8 * b.abs() + tokens * 2 ** -24 * s).all()
    native.check_status()


@pytest.mark.parametrize("bad", [40, -41, 2 ** 40])
def test_positions_outside_the_table_are_reported(bad):
    m = _module()
    ids, pos = torch.randint(0, 50, (2, 5), device=DEV), torch.zeros(2, 5, dtype=torch.long, device=DEV)
    pos[1, 4] = bad
    native.check_status()
    try:
        out = m(ids, position_ids=pos)
        grads = torch.autograd.grad(out, (m.word_embeddings.weight, m.position_embeddings.weight), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="position"):
            native.check_status()
    finally:
        native.read_and_clear_status()
    assert torch.equal(out[1, 4], m.word_embeddings.weight[ids[1, 4]])                # and nothing is added there
    assert (grads[1][0] == 9).all() and not grads[1][1:].any()
    F.embedding(ids, m.word_embeddings.weight, m.position_embeddings.weight, position_ids=pos)
    native.check_status()                                                             # not strict: they add nothing


def test_positions_on_the_host():
    m = _module()
    ids, pos = torch.randint(0, 50, (2, 5), device=DEV), torch.tensor([[0, 1, 39, 0, -1]])
    assert torch.equal(m(ids, position_ids=pos), m(ids, position_ids=pos.to(DEV)))
    with pytest.raises(IndexError):
        m(ids, position_ids=pos + 1)
    native.check_status()


@pytest.mark.parametrize("lens,most", [([40], 40), ([41], 40), ([1] * 300 + [9], 8), ([8] * 300, 8), ([0, 0], 0), ([], 5)])
def test_packed_documents_longer_than_a_table(lens, most):
    """Offsets on the GPU: a status; rows behind the last sequence do not count."""
    cu = [0] + torch.tensor(lens).cumsum(0).tolist() if lens else [0]
    seqs = F.PackedSequences(torch.tensor(cu, device=DEV), cu[-1] + 100)
    native.check_status()
    seqs.limit_lengths(most)
    assert (native.read_and_clear_status() != 0) == (max(lens, default=0) > most)
    known = F.PackedSequences(cu, cu[-1] + 100, device=DEV)
    if max(lens, default=0) > most:
        with pytest.raises(ValueError):
            known.limit_lengths(most)
    else:
        known.limit_lengths(most)
    native.check_status()


def test_a_module_takes_a_packing_as_positions():
    m = _module()
    ids = torch.randint(0, 50, (2, 60), device=DEV)
    for cu, reported in (([0, 40, 80], False), ([0, 41, 80], True)):
        seqs = F.PackedSequences(torch.tensor(cu, device=DEV), 120)
        out = m(ids, position_ids=seqs)
        assert (native.read_and_clear_status() != 0) == reported
        at = torch.cat([torch.arange(cu[1]), torch.arange(80 - cu[1]), torch.arange(40)]).view(2, 60)
        pos = m.position_embeddings.weight[at.clamp(max=39)].float() * (at < 40).to(DEV)[..., None]
        want = m.word_embeddings.weight[ids].float() + pos
        assert ((out.float() - want).abs() <= 1.01 * 2 ** -8 * want.abs() + 1e-6).all()


def test_generation_behind_the_table():
    from mist_b200.inference import generate
    from tests.test_packed_training_cpu import build
    model = build("gpt", device=DEV, dtype=torch.bfloat16, params_dtype="bfloat16", hidden_size=256, intermediate_size=512)
    ids = torch.randint(0, 250, (1, 30), device=DEV)
    assert generate(model, ids, 3).shape == (1, 33)
    with pytest.raises(IndexError):
        generate(model, ids, 6)
    native.check_status()
