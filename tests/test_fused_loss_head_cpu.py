"""The head with projection and loss in one passes no hooked or replaced projection by."""
import pytest
import torch

from mist_b200.ops import functional as F
from tests.test_packed_training_cpu import batch, build


class Halved(torch.nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x) * 0.5


def _models():
    plain, fused = build("gpt"), build("gpt", fused_lm_loss=True)
    fused.load_state_dict(plain.state_dict())
    return plain, fused


@pytest.mark.parametrize("change", ["hook", "pre-hook", "backward hook", "wrapped", "forward", "bias", "global hook"])
def test_a_changed_projection_is_called(change):
    ids, labels = (t[:, :30] for t in batch(1))
    seen, losses, grads, handles = [], [], [], []
    for model in _models():
        head = model.lm_head
        if change == "hook":
            head.proj.register_forward_hook(lambda m, a, out: seen.append(1) or out * 0.5)
        elif change == "pre-hook":
            head.proj.register_forward_pre_hook(lambda m, a: seen.append(1) or (a[0] * 0.5,))
        elif change == "backward hook":
            head.proj.register_full_backward_hook(lambda m, gi, go: seen.append(1))
        elif change == "wrapped":
            head.proj = Halved(head.proj)
        elif change == "forward":
            old = head.proj.forward
            head.proj.forward = lambda x, old=old: old(x) * 0.5
        elif change == "bias":
            head.proj.bias = torch.nn.Parameter(torch.linspace(-3, 3, 250))
        else:
            handles.append(torch.nn.modules.module.register_module_forward_hook(
                lambda m, a, out, p=head.proj: seen.append(1) if m is p else None))
        try:
            losses.append(model(ids, labels=labels))
            losses[-1].backward()
        finally:
            for h in handles:
                h.remove()
            handles.clear()
        grads.append({n: p.grad for n, p in model.named_parameters()})
    assert torch.equal(*losses)
    assert all(torch.equal(grads[0][n], grads[1][n]) for n in grads[0])
    assert len(seen) == (0 if change in ("wrapped", "forward", "bias") else 2)


def test_an_untouched_projection_is_not(monkeypatch):
    _, fused = _models()
    ids, labels = (t[:, :30] for t in batch(1))
    called = []
    real = F.linear_cross_entropy
    monkeypatch.setattr(F, "linear_cross_entropy", lambda *a, **k: called.append(1) or real(*a, **k))
    fused(ids, labels=labels)
    assert called == [1]
