"""BERT with a pooler on packed documents: a row's first token belongs to its first document only, so nothing is pooled."""
import pytest
import torch

from mist_b200.ops import functional as F
from tests.test_packed_training_cpu import CU, batch, build


def test_sentence_order_is_refused():
    model, (ids, labels) = build("bert", add_pooler=True), batch(2)
    assert model.binary_head is not None
    order = torch.tensor([0, 1])
    with pytest.raises(NotImplementedError):
        model(ids, attention_mask=F.PackedSequences(CU, 48), lm_labels=labels, sentence_order=order)
    assert torch.isfinite(model(ids, lm_labels=labels, sentence_order=order))


@pytest.mark.parametrize("fused", [False, True])
def test_the_masked_language_loss_alone_is_served(fused):
    model, plain = build("bert", add_pooler=True, fused_lm_loss=fused), build("bert")
    plain.load_state_dict({n: t for n, t in model.state_dict().items() if n in plain.state_dict()})
    (ids, labels), packed = batch(2), F.PackedSequences(CU, 48)
    loss = model(ids, attention_mask=packed, lm_labels=labels)
    assert abs(loss.item() - plain(ids, attention_mask=packed, lm_labels=labels).item()) < 1e-5
    loss.backward()
    assert model.binary_head.weight.grad is None and model.language_model.pooler.dense.weight.grad is None
    logits, binary = model(ids, attention_mask=packed)
    assert logits.shape[:2] == (2, 24) and binary is None
    assert model(ids)[1].shape == (2, 2)
