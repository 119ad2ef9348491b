"""Vocabulary loss of hidden sizes above 1024, whose products are summed in segments of K, with several tiles per CTA pair.

A logit is a sum of segments of at most 1024 products each, which the tensor cores add (taken as off by at most 1024 * 2^-23 of
the sum of the magnitudes), joined in fp32 (2^-24 each).  A missing or doubled block of 64 products changes a logit by more than
five times that (64 products of variance 4 / K each: 0.32 at K 2560, 0.25 at 4104, where the bound is 0.025), as each test checks."""
import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native
from tests.test_linear_xent_gpu import _case, _Exact, logits  # noqa: F401  (kept, and computed twice)

pytestmark = pytest.mark.gpu


def _exact(x, w, b, labels, g):
    """With the bound of the loss that the segments allow in the place of one sum over all of K."""
    exact, k = _Exact(x, w, b, labels, g), x.shape[1]
    size = (x.detach().double().abs() @ w.detach().double().abs().t()).amax(-1)
    exact.loss_tol = exact.loss_tol - 2 * (k - 1024 - -(-k // 1024)) * 2.0 ** -23 * size
    return exact


@pytest.mark.parametrize("rows,k,vocab,bias", [(1030, 1032, 20011, True), (1030, 2056, 20011, False), (700, 2560, 20011, True),
                                               (1030, 1088, 9000, True), (77, 4104, 5003, True), (300, 2048, 30001, False)])
def test_segments_of_the_hidden_size(rows, k, vocab, bias, logits):  # noqa: F811
    x, w, b, labels, g = _case(rows, k, vocab, bias, seed=k)
    assert -(-k // 1024) > 1
    exact = _exact(x, w, b, labels, g)
    missing = (x.detach()[:, -64:].double() @ w.detach()[:, -64:].double().t()).std()      # what a block changes a logit by
    assert exact.loss_tol.max() < missing / 5
    loss = F.linear_cross_entropy(x, w, labels, b)
    grads = torch.autograd.grad(loss, (x, w) if b is None else (x, w, b), g)
    native.check_status()
    exact.check(loss, grads)


@pytest.mark.parametrize("k", [1032, 2560])
def test_a_bucket_and_pieces(k, monkeypatch, logits):  # noqa: F811
    """Pieces of 512 columns added into an fp32 bucket that holds something already."""
    rows, vocab = 260, 3001
    monkeypatch.setattr(F.Settings, "xent_piece_bytes", 2 * 512 * rows)
    x, w, _, labels, g = _case(rows, k, vocab, False, seed=k)
    exact = _exact(x, w, None, labels, g)
    start = 2.0 ** -10               # what is added to it keeps 2^-34: nothing beside the bound
    w.grad_bucket, w.grad_accumulate = torch.full((vocab, k), start, device=x.device), True
    loss = F.linear_cross_entropy(x, w, labels)
    loss.backward(g)
    native.check_status()
    assert w.grad is None
    exact.check(loss, (x.grad, w.grad_bucket.double() - start))
