"""What the vocabulary loss holds between its passes stays within ``Settings.xent_keep_bytes``, all of it counted."""
import gc

import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import linear_xent

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _held(fn):
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    out = fn()
    return torch.cuda.memory_stats()["requested_bytes.all.current"] - before, out


@pytest.mark.parametrize("rows,vocab", [(256, 4096), (77, 1003), (1, 300), (515, 2056)])
def test_the_limit_counts_everything(rows, vocab, monkeypatch):
    torch.manual_seed(0)
    monkeypatch.setattr(linear_xent, "KEEP_FROM", 0)
    x = torch.randn(rows, 64, device=DEV).bfloat16().requires_grad_(True)
    w = torch.randn(vocab, 64, device=DEV).bfloat16().requires_grad_(True)
    labels, codes = torch.randint(0, vocab, (rows,), device=DEV), 2 * rows * vocab
    limit = linear_xent.kept_bytes(rows, vocab)
    for allowed in (limit, limit - 1, codes, 0):
        monkeypatch.setattr(F.Settings, "xent_keep_bytes", allowed)
        held, loss = _held(lambda: F.linear_cross_entropy(x, w, labels))
        assert (codes <= held <= allowed) if allowed == limit else held < codes
        assert held <= max(allowed, 8 * rows)            # at least the loss and the log-sum-exp of each row
        loss.sum().backward()
        x.grad = w.grad = None
        del loss
