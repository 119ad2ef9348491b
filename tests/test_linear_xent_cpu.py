"""Vocabulary projection with cross entropy on the reference path: values, gradients (against the formula's and against
differences), vocabulary slices on two ranks, refusals."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from mist_b200.ops import functional as F
from mist_b200.ops.linear_xent import piece_columns
from mist_b200.utils.device import free_port


def _case(rows=9, k=16, v=37, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g).requires_grad_(True)
    w = torch.randn(v, k, generator=g).requires_grad_(True)
    b = torch.randn(v, generator=g).requires_grad_(True) if bias else None
    labels = torch.randint(0, v, (rows,), generator=g)
    labels[::4] = -100
    return x, w, b, labels, torch.rand(rows, generator=g)


def _plain(x, w, b, labels):
    return torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w, b), labels, reduction="none")


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("shape", [(9,), (3, 3)])
def test_against_the_two_steps(bias, shape):
    x, w, b, labels, g = _case(bias=bias)
    leaves = [t for t in (x, w, b) if t is not None]
    loss = F.linear_cross_entropy(x.view(*shape, -1), w, labels.view(shape), b)
    assert loss.shape == shape and loss.dtype == torch.float32
    want = _plain(x, w, b, labels)
    assert torch.allclose(loss.reshape(-1), want, atol=1e-5)
    for a, r in zip(torch.autograd.grad(loss, leaves, g.view(shape)), torch.autograd.grad(want, leaves, g)):
        assert torch.allclose(a, r, atol=1e-5)


def test_gradient_against_differences():
    x, w, b, labels, g = _case(rows=5, k=8, v=11)
    loss = F.linear_cross_entropy(x, w, labels, b)
    grads = torch.autograd.grad(loss, (x, w, b), g[:5])
    for t, d in zip((x, w, b), grads):
        step = torch.zeros_like(t)
        for at in range(0, t.numel(), 7):
            step.view(-1)[at] = 1e-2
            args = [(u + s * step if u is t else u).detach().double() for s in (1, -1) for u in (x, w, b)]
            diff = ((_plain(*args[:3], labels) - _plain(*args[3:], labels)) * g[:5].double()).sum() / 2e-2
            assert abs(diff - d.view(-1)[at]) < 1e-3          # third derivatives of a softmax stay below 1: 1e-4 / 6
            step.view(-1)[at] = 0


def test_bucket_and_nothing_kept():
    x, w, b, labels, g = _case(bias=False)
    ref = torch.autograd.grad(_plain(x, w, None, labels), w, g)[0]
    for accumulate in (False, True):
        w.grad_bucket, w.grad_accumulate = torch.ones_like(w), accumulate
        F.linear_cross_entropy(x, w, labels).backward(g)
        assert w.grad is None and w.grad_accumulate
        assert torch.allclose(w.grad_bucket, ref + (1.0 if accumulate else 0.0), atol=1e-5)


def test_no_rows_and_all_ignored():
    x, w, b, labels, g = _case()
    loss = F.linear_cross_entropy(x[:0], w, labels[:0], b)
    assert loss.shape == (0,)
    grads = torch.autograd.grad(loss.sum(), (x, w, b))
    assert all(not t.any() for t in grads)
    loss = F.linear_cross_entropy(x, w, torch.full_like(labels, -100), b)
    assert not loss.any() and all(not t.any() for t in torch.autograd.grad(loss, (x, w, b), g))


def test_pieces_cover_the_vocabulary():
    before = F.Settings.xent_piece_bytes
    try:
        for limit in (1, 1 << 16, 1 << 22, 1 << 40):
            F.Settings.xent_piece_bytes = limit
            for rows in (1, 77, 8192):
                for v in (1, 255, 256, 257, 50304, 1003):
                    n = piece_columns(rows, v)
                    assert 1 <= n <= v and (n == v or n % 256 == 0)
                    assert n <= 256 or 2 * rows * n <= max(limit, 512 * rows)
    finally:
        F.Settings.xent_piece_bytes = before


@pytest.mark.parametrize("case", ["hidden", "labels", "type", "bias", "empty"])
def test_refusals(case):
    x, w, b, labels, _ = _case()
    if case == "hidden":
        w = w[:, :8]
    elif case == "labels":
        labels = labels[:4]
    elif case == "type":
        labels = labels.float()
    elif case == "bias":
        b = b[:5]
    else:
        w, b = w[:0], None
    with pytest.raises(ValueError):
        F.linear_cross_entropy(x, w, labels, b)


def _slice_worker(rank, port, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2")
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        x, w, b, labels, g = _case(v=38)
        half = w.detach()[rank * 19:(rank + 1) * 19].clone().requires_grad_(True)
        hb = b.detach()[rank * 19:(rank + 1) * 19].clone().requires_grad_(True)
        loss = F.linear_cross_entropy(x, half, labels, hb, vocab_start=19 * rank, group=dist.group.WORLD)
        ret[rank] = [t.detach() for t in (loss, *torch.autograd.grad(loss, (x, half, hb), g))]
    finally:
        dist.destroy_process_group()


def test_vocabulary_slices_on_two_ranks():
    ret = mp.Manager().dict()
    mp.spawn(_slice_worker, args=(free_port(), ret), nprocs=2)
    x, w, b, labels, g = _case(v=38)
    want = _plain(x, w, b, labels)
    dx, dw, db = torch.autograd.grad(want, (x, w, b), g)
    for r in range(2):
        assert torch.allclose(ret[r][0], want, atol=1e-5)
        assert torch.allclose(ret[r][2], dw[19 * r:19 * r + 19], atol=1e-5)
        assert torch.allclose(ret[r][3], db[19 * r:19 * r + 19], atol=1e-5)
    assert torch.allclose(ret[0][1] + ret[1][1], dx, atol=1e-5)


def _head_worker(rank, port, tied, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2")
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        from mist_b200.models.language_model import LMHead
        ret[rank] = _head_step(LMHead, dist.group.WORLD, rank, 2, tied)
    finally:
        dist.destroy_process_group()


def _head_step(LMHead, group, rank, world, tied):
    from mist_b200.config import ModelConfig
    cfg = ModelConfig(name="gpt2-t", hidden_size=16, num_hidden_layers=1, num_attention_heads=2, max_position_embeddings=8,
                      vocab_size=40, params_dtype="float32", add_encoder=True, add_decoder=False,
                      encoder_attn_mask_type="causal", fused_lm_loss=True)
    x, w, _, labels, _ = _case(rows=12, v=40, bias=False)
    labels = labels.clamp(min=0)
    head = LMHead(cfg, group)
    part = w.detach().chunk(world)[rank].clone().requires_grad_(True)
    if not tied:
        with torch.no_grad():
            head.proj.weight.copy_(part)
        part = head.proj.weight
    loss = head(x.view(2, 6, 16), labels.view(2, 6), part if tied else None)
    return [t.detach() for t in (loss, *torch.autograd.grad(loss, (x, part)))]


@pytest.mark.parametrize("tied", [False, True])
def test_head_on_two_ranks(tied):
    from mist_b200.models.language_model import LMHead
    ret = mp.Manager().dict()
    mp.spawn(_head_worker, args=(free_port(), tied, ret), nprocs=2)
    loss, dx, dw = _head_step(LMHead, None, 0, 1, tied)
    for r in range(2):
        assert torch.allclose(ret[r][0], loss, atol=1e-5) and torch.allclose(ret[r][1], dx, atol=1e-5)
        assert torch.allclose(ret[r][2], dw.chunk(2)[r], atol=1e-5)


def _masked_slice_worker(rank, port, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE="2")
    dist.init_process_group("gloo", rank=rank, world_size=2)
    try:
        x, w, b, labels, g = _masked_case()
        half = w.detach()[rank * 19:(rank + 1) * 19].clone().requires_grad_(True)
        hb = b.detach()[rank * 19:(rank + 1) * 19].clone()
        loss = F.linear_cross_entropy(x, half, labels, hb, vocab_start=19 * rank, group=dist.group.WORLD)
        ret[rank] = [t.detach() for t in (loss, *torch.autograd.grad(loss, (x, half), g))]
    finally:
        dist.destroy_process_group()


def _masked_case():
    """All of the second rank's words (the padding of a vocabulary) have the logit -inf."""
    x, w, b, labels, g = _case(v=38)
    with torch.no_grad():
        b[19:] = float("-inf")
    return x, w, b, torch.where(labels >= 0, labels % 19, labels), g


def test_a_slice_of_words_that_are_masked():
    ret = mp.Manager().dict()
    mp.spawn(_masked_slice_worker, args=(free_port(), ret), nprocs=2)
    x, w, b, labels, g = _masked_case()
    want = _plain(x, w, b, labels)
    dx, dw = torch.autograd.grad(want, (x, w), g)
    for r in range(2):
        assert torch.allclose(ret[r][0], want, atol=1e-5)
        assert torch.allclose(ret[r][2], dw[19 * r:19 * r + 19], atol=1e-5)
    assert torch.allclose(ret[0][1] + ret[1][1], dx, atol=1e-5)
