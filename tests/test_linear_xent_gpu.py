"""Vocabulary projection with cross entropy on the GPU against 64 bits.

Tolerances.  A logit is a sum of k products in fp32, taken as off by at most k * 2^-23 of the sum of their magnitudes
(sums that truncate); the loss adds the error of two logits and a few fp32 roundings of the numbers in it (2^-21).  The
gradient of a logit is rounded to bf16, off by at most 2^-8 of it; the gradients of x and of the weight sum those with
signs that have nothing to do with one another, so the 2-norm of their error is held to 2^-8 of the root of the sum of
the squared terms, and 2^-8 of the gradient itself for its own rounding."""
import gc

import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = 2.0 ** -8


def _case(rows, k, v, bias, ignored=0.2, seed=0):
    torch.manual_seed(seed)
    x = torch.randn(rows, k, device=DEV).bfloat16().requires_grad_(True)
    w = (torch.randn(v, k, device=DEV) * (2.0 / k ** 0.5)).bfloat16().requires_grad_(True)
    b = torch.randn(v, device=DEV).bfloat16().requires_grad_(True) if bias else None
    labels = torch.randint(0, v, (rows,), device=DEV)
    labels[torch.rand(rows, device=DEV) < ignored] = -100
    return x, w, b, labels, (torch.rand(rows, device=DEV) + 0.5) / rows



@pytest.fixture(autouse=True, params=["kept", "computed twice"])
def logits(request, monkeypatch):
    """Every test with the logits kept for the backward pass, and with logits that are computed again.  What is kept is
    right to 2^-11 octaves, 3.4e-4 of a probability: a sixth of half a step of bf16, which the bounds below count."""
    from mist_b200.ops import linear_xent
    monkeypatch.setattr(linear_xent, "KEEP_FROM", 0)
    if request.param != "kept":
        monkeypatch.setattr(F.Settings, "xent_keep_bytes", 0)
    return request.param


class _Exact:
    def __init__(self, x, w, b, labels, g):
        xd, wd = x.detach().double(), w.detach().double()
        logits = xd @ wd.t()
        size = (xd.abs() @ wd.abs().t()).amax(-1)
        if b is not None:
            logits, size = logits + b.detach().double(), size + b.detach().double().abs().max()
        lse = torch.logsumexp(logits, -1)
        kept = labels != -100
        at = labels.clamp(min=0)[:, None]
        target = logits.gather(1, at)[:, 0]
        self.loss = (lse - target) * kept
        self.loss_tol = 2 * x.shape[1] * 2.0 ** -23 * size + 2.0 ** -21 * (lse.abs() + target.abs() + 1)
        dl = torch.softmax(logits, -1)
        dl.scatter_add_(1, at, torch.full_like(at, -1.0, dtype=torch.double))
        self.dl = dl * (g.double() * kept)[:, None]
        self.grads = [self.dl @ wd, self.dl.t() @ xd] + ([self.dl.sum(0)] if b is not None else [])
        sq = self.dl.square()
        self.spread = [(sq @ wd.square()).sum(), (sq.t() @ xd.square()).sum(), sq.sum()]

    def check(self, loss, grads):
        assert loss.dtype == torch.float32
        assert ((loss.double() - self.loss).abs() <= self.loss_tol).all()
        assert len(grads) == len(self.grads)
        for got, want, spread in zip(grads, self.grads, self.spread):
            assert (got.double() - want).norm() <= BF * (spread.sqrt() + want.norm()) + 1e-12


@pytest.mark.parametrize("rows,k,v", [(1, 8, 1), (1, 64, 1003), (77, 512, 1003), (129, 72, 257), (300, 264, 5000),
                                      (1000, 128, 255), (513, 1024, 256), (2047, 64, 31999)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("limit", [256 << 20, 1])
def test_loss_and_gradients(rows, k, v, bias, limit, monkeypatch):
    monkeypatch.setattr(F.Settings, "xent_piece_bytes", limit)      # 1: pieces of 256 columns
    x, w, b, labels, g = _case(rows, k, v, bias)
    loss = F.linear_cross_entropy(x, w, labels, b)
    grads = torch.autograd.grad(loss, [t for t in (x, w, b) if t is not None], g)
    native.check_status()
    _Exact(x, w, b, labels, g).check(loss, grads)
    assert not loss[labels == -100].any() and not grads[0][labels == -100].any()


def test_everything_ignored_and_nothing_given():
    x, w, b, labels, g = _case(40, 64, 300, True, ignored=2.0)
    loss = F.linear_cross_entropy(x, w, labels, b)
    grads = torch.autograd.grad(loss, (x, w, b), g)
    assert not loss.any() and all(not t.any() for t in grads)
    loss = F.linear_cross_entropy(x[:0], w, labels[:0], b)
    assert loss.shape == (0,) and all(not t.any() for t in torch.autograd.grad(loss.sum(), (x, w, b)))


def test_large_and_masked_logits():
    """Logits of hundreds, words ruled out by a bias of -inf, a row whose label is one of those."""
    x, w, b, labels, g = _case(200, 64, 700, True, ignored=0.0)
    with torch.no_grad():
        w.mul_(64)
        b[100:400] = float("-inf")
        labels[labels.ge(100) & labels.lt(400)] = 5
        labels[7] = 150
    loss = F.linear_cross_entropy(x, w, labels, b)
    grads = torch.autograd.grad(loss, (x, w, b), g)
    logits = torch.nn.functional.linear(x.detach().double(), w.detach().double(), b.detach().double())
    want = torch.nn.functional.cross_entropy(logits, labels, reduction="none")
    assert torch.isinf(loss[7]) and loss[7] > 0
    keep = torch.arange(200, device=DEV) != 7
    # logits of some hundreds: 64 * 2^-23 of magnitudes that add up to 64 * |x| |w| < 20000
    assert ((loss.double() - want).abs()[keep] < 0.3).all()
    assert all(torch.isfinite(t).all() for t in grads)
    assert not grads[2][100:150].any() and not grads[2][151:400].any() and abs(grads[2][150].item() + g[7].item()) <= BF * g[7]


def test_labels_outside_the_slice_and_slices_that_join():
    """Statistics and gradients of two slices of the vocabulary give those of the whole."""
    rows, k, v, cut = 150, 128, 900, 333
    x, w, b, labels, g = _case(rows, k, v, True)
    exact = _Exact(x, w, b, labels, g)
    lib, stats = native.kernels(), []
    with torch.no_grad():
        for a, e in ((0, cut), (cut, v)):
            tiles = lib.mb_xent_linear_tiles(e - a)
            work, out = torch.empty(tiles, rows, 2, device=DEV), torch.full((rows, 3), float("nan"), device=DEV)
            target, bias = torch.empty(rows, device=DEV), b[a:e].contiguous()
            native.call("mb_xent_linear_fwd", native.ptr(x), native.ptr(w) + 2 * k * a, native.ptr(bias), native.ptr(labels),
                        native.ptr(work), native.ptr(target), 0, 0, native.ptr(out), 0, 0, rows, e - a, k, k, k, a, -100, 0,
                        native.stream())
            stats.append(out)
        top = torch.maximum(stats[0][:, 0], stats[1][:, 0])
        total = sum(s[:, 1] * torch.exp(s[:, 0] - top) for s in stats)
        lse = total.log() + top
        loss = torch.where(labels == -100, torch.zeros_like(lse), lse - stats[0][:, 2] - stats[1][:, 2])
        parts = []
        for a, e in ((0, cut), (cut, v)):
            wa, ba = w[a:e].contiguous(), b[a:e].contiguous()
            dw, db = torch.empty(e - a, k, device=DEV, dtype=torch.bfloat16), torch.empty(e - a, device=DEV)
            dx = torch.empty(rows, k, device=DEV, dtype=torch.bfloat16)
            work = torch.empty(lib.mb_xent_linear_bwd_workspace(rows, e - a, k, e - a, 1, 1, 1, 0, 0, 0), dtype=torch.uint8,
                               device=DEV)
            native.call("mb_xent_linear_bwd", native.ptr(x), native.ptr(wa), native.ptr(ba), native.ptr(labels), native.ptr(lse),
                        native.ptr(g), native.ptr(dx), native.ptr(dw), native.ptr(db), 0, 0, 0, 0, rows, e - a, k, k, k, k, 0,
                        0, 1, a, -100, e - a, 0, native.ptr(work), native.stream())
            parts.append((dx.double(), dw, db))
    exact.check(loss, (parts[0][0] + parts[1][0], torch.cat([p[1] for p in parts]), torch.cat([p[2] for p in parts])))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("limit", [256 << 20, 1])
def test_bucket(dtype, accumulate, limit, monkeypatch):
    monkeypatch.setattr(F.Settings, "xent_piece_bytes", limit)
    x, w, b, labels, g = _case(333, 128, 1500, False)
    exact = _Exact(x, w, None, labels, g)
    before = (torch.randn(1500, 128, device=DEV) * exact.grads[1].abs().mean().float()).to(dtype)
    w.grad_bucket, w.grad_accumulate = before.clone(), accumulate
    F.linear_cross_entropy(x, w, labels).backward(g)
    native.check_status()
    want = exact.grads[1] + (before.double() if accumulate else 0)
    assert w.grad is None and w.grad_accumulate
    assert (w.grad_bucket.double() - want).norm() <= BF * (exact.spread[1].sqrt() + want.norm())


def test_only_what_is_asked_for():
    x, w, b, labels, g = _case(100, 64, 400, True)
    both = torch.autograd.grad(F.linear_cross_entropy(x, w, labels, b), (x, w, b), g)
    for k, leaf in enumerate((x, w, b)):
        args = [t if t is leaf else t.detach() for t in (x, w, b)]
        loss = F.linear_cross_entropy(args[0], args[1], labels, args[2])
        assert torch.equal(torch.autograd.grad(loss, leaf, g)[0], both[k])


def test_an_ignored_word_and_a_limit_on_the_ctas(monkeypatch):
    """The ignored label may be a word of the vocabulary; few CTAs, down to one, give the same."""
    x, w, b, labels, g = _case(300, 128, 600, True, ignored=0.0)
    labels[::3] = 5
    kept = labels.masked_fill(labels == 5, -100)
    leaves = (x, w, b)

    def once(labels, ignore):
        loss = F.linear_cross_entropy(x, w, labels, b, ignore_index=ignore)
        return [loss, *torch.autograd.grad(loss, leaves, g)]

    want = once(kept, -100)
    assert all(torch.equal(a, c) for a, c in zip(once(labels, 5), want))
    for ctas in (1, 2, 7, 64):
        monkeypatch.setattr(F.Settings, "gemm_max_ctas", ctas)
        got = once(kept, -100)
        assert torch.equal(got[0], want[0])
        exact = _Exact(x, w, b, kept, g)
        exact.check(got[0], got[1:])
    native.check_status()


def test_strided_inputs_and_one_gradient_value():
    x, w, b, labels, _ = _case(64, 128, 500, False)
    loss = F.linear_cross_entropy(x, w, labels)
    want = torch.autograd.grad(loss.mean(), (x, w))          # a gradient that is one value, expanded
    wide = torch.randn(64, 300, device=DEV).bfloat16()
    for at in (0, 8, 3):                                      # rows of a wider buffer, on 16 bytes and not
        wide[:, at:at + 128] = x.detach()
        xs = wide[:, at:at + 128].detach().requires_grad_(True)
        again = F.linear_cross_entropy(xs, w, labels)
        assert torch.equal(again, loss)
        assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(again.mean(), (xs, w)), want))
    shaped = F.linear_cross_entropy(x.view(4, 16, 128), w, labels.view(4, 16).int())
    assert torch.equal(shaped, loss.view(4, 16))


def test_repeats_and_streams():
    x, w, b, labels, g = _case(700, 256, 3000, True)

    def once():
        loss = F.linear_cross_entropy(x, w, labels, b)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w, b), g)]

    first = once()
    torch.cuda.synchronize()
    side, got = [torch.cuda.Stream() for _ in range(2)], []
    for k in range(4):
        with torch.cuda.stream(side[k % 2]):
            got.append(once())
    torch.cuda.synchronize()
    native.check_status()
    assert all(torch.equal(a, c) for other in got for a, c in zip(first, other))


def test_two_captured_graphs():
    cases = [_case(200, 64, 1000, True, seed=s) for s in (1, 2)]

    def once(c):
        loss = F.linear_cross_entropy(c[0], c[1], c[3], c[2])
        return [loss.detach(), *torch.autograd.grad(loss, (c[0], c[1], c[2]), c[4])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            once(c)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(once(c))
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):                                        # both under way at once
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    native.check_status()
    for c, o in zip(cases, outs):
        assert all(torch.equal(a, e) for a, e in zip(o, once(c)))


@pytest.mark.parametrize("case", ["type", "hidden", "device"])
def test_refusals(case):
    x, w, b, labels, _ = _case(8, 64, 100, False)
    if case == "type":
        w = w.float()
    elif case == "hidden":
        x, w = x[:, :60], w[:, :60]
    else:
        labels = labels.cpu()
    with pytest.raises(ValueError):
        F.linear_cross_entropy(x, w, labels)


@pytest.mark.parametrize("dtype,start", [(torch.float32, 1), (torch.bfloat16, 4)])
def test_bucket_off_the_stores_alignment(dtype, start):
    """A bucket that the kernels' stores cannot address gets the gradient by way of another tensor."""
    torch.manual_seed(9)
    x = torch.randn(40, 64, device=DEV).bfloat16()
    w = torch.nn.Parameter(torch.randn(96, 64, device=DEV).bfloat16())
    labels = torch.randint(0, 96, (40,), device=DEV)
    want, = torch.autograd.grad(F.linear_cross_entropy(x, w, labels).sum(), w)
    flat = torch.zeros(96 * 64 + 8, device=DEV, dtype=dtype)
    w.grad_bucket = flat[start:start + 96 * 64].view(96, 64)
    for n in (1, 2):
        F.linear_cross_entropy(x, w, labels).sum().backward()
        # an fp32 bucket holds what the bf16 gradient was before its rounding; a second step adds one rounding
        tol = 2 ** -8 * n * want.float().abs() * (1 + n) + 1e-6
        assert ((w.grad_bucket.float() - n * want.float()).abs() <= tol).all()
    assert not flat[:start].any() and not flat[start + 96 * 64:].any()


def test_a_label_that_is_all_but_certain():
    """Its gradient is the small rest to 1, which what is kept of the logit alone would get wrong by a tenth."""
    torch.manual_seed(12)
    rows, k, v = 96, 256, 1000
    w = (torch.randn(v, k, device=DEV) / k ** 0.5).bfloat16().requires_grad_(True)
    labels = torch.arange(rows, device=DEV) * 7
    x = (12.5 * w.detach()[labels].float()).bfloat16().requires_grad_(True)
    g = torch.rand(rows, device=DEV) + 0.5
    exact = _Exact(x, w, None, labels, g)
    rest = -exact.dl.gather(1, labels[:, None])[:, 0] / g
    assert 1e-4 < rest.median() < 2e-2
    loss = F.linear_cross_entropy(x, w, labels)
    grads = torch.autograd.grad(loss, (x, w), g)
    exact.check(loss, grads)
    # row by row: dx of a row is what its own column of dl gives; bf16 of dl (2^-8 of each entry) and of dx
    dl = exact.dl
    for got, want, spread in zip(grads[0].double(), dl @ w.double(), (dl.square() @ w.double().square()).sum(1)):
        assert (got - want).norm() <= BF * (2 * spread.sqrt() + want.norm())


def test_a_second_backward_pass_gets_the_same(logits):
    x, w, b, labels, g = _case(130, 72, 700, True)
    loss = F.linear_cross_entropy(x, w, labels, b)
    first = torch.autograd.grad(loss, (x, w, b), g, retain_graph=True)
    again = torch.autograd.grad(loss, (x, w, b), g)
    assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_what_is_kept(logits, monkeypatch):
    """16 bits per logit, and not without need: no gradient wanted, or more than the limit."""
    x, w, _, labels, g = _case(256, 64, 4096, False)

    def asked():              # (a block that the allocator hands out may be larger)
        return torch.cuda.memory_stats()["requested_bytes.all.current"]

    def held(fn):
        gc.collect()              # what earlier tests left
        torch.cuda.synchronize()
        before = asked()
        out = fn()
        return asked() - before, out

    size = 2 * 256 * 4096
    small = 4 * 256 * 16 * 8
    n, loss = held(lambda: F.linear_cross_entropy(x, w, labels))
    assert (size <= n <= size + small) if logits == "kept" else n <= small
    del loss
    with torch.no_grad():
        n, loss = held(lambda: F.linear_cross_entropy(x, w, labels))
    assert n <= small
    monkeypatch.setattr(F.Settings, "xent_keep_bytes", size - 1)
    n, loss = held(lambda: F.linear_cross_entropy(x, w, labels))
    assert n <= small


def test_rows_that_are_not_numbers():
    """An ignored row of NaN has the loss 0 and no gradient of its own; a row of NaN with a label is NaN, the others are not."""
    x, w, b, labels, g = _case(70, 64, 600, True, ignored=0.0)
    with torch.no_grad():
        x[5] = float("nan")
        x[9] = float("nan")
    labels[5] = -100
    loss = F.linear_cross_entropy(x, w, labels, b)
    dx, = torch.autograd.grad(loss, (x,), g)
    assert loss[5] == 0 and not dx[5].any() and torch.isnan(loss[9]) and torch.isnan(dx[9]).all()
    others = [i for i in range(70) if i not in (5, 9)]
    assert torch.isfinite(loss[others]).all() and torch.isfinite(dx[others]).all()


def test_slices_that_join_with_logits_kept():
    """As above for slices of the vocabulary, each keeping its own logits; the log-sum-exp is that of all of them."""
    rows, k, v, cut = 150, 128, 900, 333
    x, w, b, labels, g = _case(rows, k, v, True)
    exact = _Exact(x, w, b, labels, g)
    lib, held, outs = native.kernels(), [], []
    p = native.ptr
    for a, e in ((0, cut), (cut, v)):
        wide = (e - a + 7) // 8 * 8
        stats, target = torch.empty(2 * lib.mb_xent_linear_tiles(e - a), rows, 2, device=DEV), torch.empty(rows, device=DEV)
        kept, out = torch.empty(rows, wide, device=DEV, dtype=torch.int16), torch.full((rows, 3), float("nan"), device=DEV)
        wa, ba = w.detach()[a:e].contiguous(), b.detach()[a:e].contiguous()
        native.call("mb_xent_linear_fwd", p(x), p(wa), p(ba), p(labels), p(stats), p(target), 0, 0, p(out), p(kept), wide, rows,
                    e - a, k, k, k, a, -100, 0, native.stream())
        held.append((a, e, wa, ba, stats, target, kept, wide))
        outs.append(out)
    top = torch.maximum(outs[0][:, 0], outs[1][:, 0])
    lse = sum(o[:, 1] * torch.exp(o[:, 0] - top) for o in outs).log() + top
    loss = torch.where(labels == -100, torch.zeros_like(lse), lse - outs[0][:, 2] - outs[1][:, 2])
    parts = []
    for a, e, wa, ba, stats, target, kept, wide in held:
        dw, db = torch.empty(e - a, k, device=DEV, dtype=torch.bfloat16), torch.empty(e - a, device=DEV)
        dx = torch.empty(rows, k, device=DEV, dtype=torch.bfloat16)
        work = torch.empty(lib.mb_xent_linear_bwd_workspace(rows, e - a, k, 256, 1, 1, 1, 0, 0, 0), dtype=torch.uint8, device=DEV)
        native.call("mb_xent_linear_bwd", p(x), p(wa), p(ba), p(labels), p(lse), p(g), p(dx), p(dw), p(db), p(kept), wide,
                    p(stats), p(target), rows, e - a, k, k, k, k, 0, 0, 1, a, -100, 256, 0, p(work), native.stream())
        parts.append((dx.double(), dw, db))
    native.check_status()
    exact.check(loss, (parts[0][0] + parts[1][0], torch.cat([q[1] for q in parts]), torch.cat([q[2] for q in parts])))
