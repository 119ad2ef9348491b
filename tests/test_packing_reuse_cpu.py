"""One packing for an evaluation under inference mode and a training step after it."""
import pytest
import torch

from mist_b200.ops import functional as F
from tests.test_packed_training_cpu import CU, batch, build


@pytest.mark.parametrize("family", ["gpt", "llama"])
@pytest.mark.parametrize("made_inside", [True, False])
def test_first_use_under_inference_mode(family, made_inside):
    model, (ids, labels) = build(family), batch(1)
    packed = None if made_inside else F.PackedSequences(CU, 48)
    with torch.inference_mode():
        if made_inside:
            packed = F.PackedSequences(torch.tensor(CU), 48)
        want = model(ids, attention_mask=packed, labels=labels)
    loss = model(ids, attention_mask=packed, labels=labels)
    assert loss.item() == want.item()
    loss.backward()
    fresh = build(family)
    fresh(ids, attention_mask=F.PackedSequences(CU, 48), labels=labels).backward()
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(model.parameters(), fresh.parameters()))
