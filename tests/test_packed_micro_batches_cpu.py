"""A packing is of one micro batch: one for several is refused with a reason."""
import pytest
import torch

from mist_b200.api import TrainingSession
from mist_b200.ops import functional as F


class _Session:
    """What splitting a batch needs of a session."""
    pipeline = None
    G = 2

    def __init__(self):
        self.engine = self

    def _beat(self):
        pass

    def train_step(self, batches):
        return batches


def test_one_packing_for_two_micro_batches():
    ids = torch.zeros(2, 24, dtype=torch.long)
    with pytest.raises(ValueError, match="attention_mask.*micro batches"):
        TrainingSession.step_on_device_batch(_Session(), dict(input_ids=ids, attention_mask=F.PackedSequences([0, 48])))
    packings = [F.PackedSequences([0, 24]), F.PackedSequences([0, 5, 24])]
    batches = TrainingSession.step_on_device_batch(_Session(), dict(input_ids=ids, attention_mask=packings))
    assert [b["attention_mask"] for b in batches] == packings and all(b["input_ids"].shape == (1, 24) for b in batches)
