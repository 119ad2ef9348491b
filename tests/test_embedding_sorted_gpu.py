"""Embedding lookup and its gradient by sorted tokens against sums in 64 bits.

Tolerances: the lookup is one fp32 multiply-add and one rounding to bf16 (2^-8 of the value, and 2^-23 of the larger
summand).  A gradient is a sum of n products in fp32, off by at most n * 2^-24 of the sum of the magnitudes, and rounded
once (2^-8; to an fp32 bucket 2^-24)."""
import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = 2.0 ** -8


def _ids(kind, b, s, v, start):
    if kind == "uniform":
        return torch.randint(0, v + 2 * start, (b, s), device=DEV)
    if kind == "one":
        return torch.full((b, s), start + v - 1, device=DEV)
    if kind == "none":
        return torch.full((b, s), start + v, device=DEV)
    if kind == "ends":                                    # two long rows that share a tile, and nothing between
        return start + (torch.arange(b * s, device=DEV).view(b, s) * 2 >= b * s).long() * (v - 1)
    assert kind == "skewed"
    u = torch.rand(b, s, device=DEV)
    return start + (u ** 6 * v).long().clamp(max=v - 1)


@pytest.mark.parametrize("kind", ["uniform", "one", "none", "ends", "skewed"])
@pytest.mark.parametrize("b,s,h,v", [(1, 1, 8, 3), (2, 65, 24, 255), (1, 64, 128, 256), (3, 777, 520, 1003),
                                     (1, 5003, 1024, 70001), (4, 2048, 64, 300), (2, 17001, 16, 500)])
@pytest.mark.parametrize("positions", ["none", "row", "given"])
def test_forward_and_gradients(kind, b, s, h, v, positions):
    torch.manual_seed(7)
    start, scale, p = 2, 1.75, max(s, 9)
    ids = _ids(kind, b, s, v, start)
    wte = torch.randn(v, h, device=DEV).bfloat16().requires_grad_(True)
    wpe = torch.randn(p, h, device=DEV).bfloat16().requires_grad_(True) if positions != "none" else None
    pos = torch.randint(-1, p + 1, (b, s), device=DEV) if positions == "given" else None
    out = F.embedding(ids, wte, wpe, start, scale=scale, position_ids=pos)
    loc = (ids - start).reshape(-1)
    inside = (loc >= 0) & (loc < v)
    at = (pos if pos is not None else torch.arange(s, device=DEV).expand(b, s)).reshape(-1)
    known = (at >= 0) & (at < p)
    want = wte.detach().double()[loc.clamp(0, v - 1)] * inside[:, None] * scale
    size = want.abs()
    if wpe is not None:
        more = wpe.detach().double()[at.clamp(0, p - 1)] * known[:, None]
        want, size = want + more, size + more.abs()
    assert ((out.detach().double().view(-1, h) - want).abs() <= BF * want.abs() + 2.0 ** -23 * size).all()

    g = torch.randn(b, s, h, device=DEV).bfloat16()
    grads = torch.autograd.grad(out, (wte,) if wpe is None else (wte, wpe), g)
    native.check_status()
    g2 = g.double().view(-1, h)

    def check(got, rows, index, keep, factor):
        n = torch.zeros(rows, device=DEV, dtype=torch.double).index_add_(0, index[keep], torch.ones_like(index[keep]).double())
        ref = torch.zeros(rows, h, device=DEV, dtype=torch.double).index_add_(0, index[keep], g2[keep] * factor)
        mag = torch.zeros(rows, h, device=DEV, dtype=torch.double).index_add_(0, index[keep], (g2[keep] * factor).abs())
        assert got.dtype == torch.bfloat16
        assert ((got.double() - ref).abs() <= BF * ref.abs() * 1.01 + (n[:, None] + 2) * 2.0 ** -24 * mag).all()

    check(grads[0], v, loc, inside, scale)
    if wpe is not None:
        check(grads[1], p, at, known, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("kind", ["skewed", "ends"])
def test_bucket_rows_without_tokens(dtype, accumulate, kind):
    """Long rows in a bucket; rows that get nothing are zero, or left to the bit where the bucket is added to."""
    torch.manual_seed(3)
    v, h, b, s = 501, 72, 2, 600
    w = torch.nn.Parameter(torch.randn(v, h, device=DEV).bfloat16())
    ids = _ids(kind, b, s, v, 0)
    g = torch.randn(b, s, h, device=DEV).bfloat16()
    before = torch.randn(v, h, device=DEV).to(dtype)
    w.grad_bucket, w.grad_accumulate = before.clone(), accumulate
    F.embedding(ids, w, scale=0.5).backward(g)
    native.check_status()
    old = before.double() if accumulate else torch.zeros(v, h, device=DEV, dtype=torch.double)
    want = old.index_add(0, ids.reshape(-1), g.double().view(-1, h) * 0.5)
    mag = old.abs().index_add(0, ids.reshape(-1), g.double().view(-1, h).abs() * 0.5)
    step = BF if dtype == torch.bfloat16 else 2.0 ** -24
    assert ((w.grad_bucket.double() - want).abs() <= 1.01 * step * want.abs() + 1300 * 2.0 ** -24 * mag).all()
    free = torch.ones(v, dtype=torch.bool, device=DEV)
    free[ids.reshape(-1)] = False
    assert free.any() and torch.equal(w.grad_bucket[free], before[free] if accumulate else torch.zeros_like(before[free]))


def test_repeats_bit_for_bit_and_on_other_streams():
    torch.manual_seed(4)
    v, h, s = 2000, 256, 9000
    wte = torch.randn(v, h, device=DEV).bfloat16().requires_grad_(True)
    ids = _ids("skewed", 1, s, v, 0)
    g = torch.randn(1, s, h, device=DEV).bfloat16()

    def once():
        return torch.autograd.grad(F.embedding(ids, wte), wte, g)[0]

    first = once()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k in range(6):                                     # two calls under way at once
        with torch.cuda.stream(side[k % 2]):
            got.append(once())
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in got)


def test_captured_into_a_graph():
    torch.manual_seed(5)
    v, h, s = 300, 64, 700
    wte = torch.randn(v, h, device=DEV).bfloat16().requires_grad_(True)
    ids, g = _ids("skewed", 1, s, v, 0), torch.randn(1, s, h, device=DEV).bfloat16()

    def once():
        out = F.embedding(ids, wte, scale=2.0)
        return out, torch.autograd.grad(out, wte, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = once()
    for _ in range(3):                                     # other tokens at each replay
        ids.copy_(_ids("uniform", 1, s, v, 0))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, once()):
            assert torch.equal(a, b)


def test_other_integer_types_and_strides():
    torch.manual_seed(6)
    v, h = 50, 16
    wte = torch.randn(v, h, device=DEV).bfloat16()
    ids = torch.randint(0, v, (6, 10), device=DEV)
    want = F.embedding(ids, wte)
    assert torch.equal(F.embedding(ids.int(), wte), want)
    assert torch.equal(F.embedding(ids.t().contiguous().t(), wte), want)
    w = wte.clone().requires_grad_(True)
    wide = torch.randn(6, 10, 2 * h, device=DEV).bfloat16()
    a = torch.autograd.grad(F.embedding(ids, w), w, wide[..., 3:h + 3])[0]           # an odd start, strided rows
    b = torch.autograd.grad(F.embedding(ids, w), w, wide[..., 3:h + 3].contiguous())[0]
    assert torch.equal(a, b)


@pytest.mark.parametrize("shape", [(0, 5), (3, 0)])
@pytest.mark.parametrize("given", [False, True])
def test_no_tokens(shape, given):
    wte, wpe = (torch.randn(n, 16, device=DEV).bfloat16().requires_grad_(True) for n in (20, 9))
    ids = torch.zeros(shape, device=DEV, dtype=torch.long)
    out = F.embedding(ids, wte, wpe, position_ids=ids if given else None)
    assert out.shape == (*shape, 16)
    assert all(not g.any() for g in torch.autograd.grad(out.sum(), (wte, wpe)))


@pytest.mark.parametrize("given", [False, True])
def test_one_table_frozen(given):
    torch.manual_seed(8)
    ids, pos = torch.randint(0, 40, (2, 90), device=DEV), torch.randint(0, 90, (2, 90), device=DEV) if given else None
    g = torch.randn(2, 90, 24, device=DEV).bfloat16()
    tables = [torch.randn(n, 24, device=DEV).bfloat16() for n in (40, 90)]
    both = [t.clone().requires_grad_(True) for t in tables]
    want = torch.autograd.grad(F.embedding(ids, *both, position_ids=pos), both, g)
    for k in range(2):
        only = [t.clone().requires_grad_(i == k) for i, t in enumerate(tables)]
        assert torch.equal(torch.autograd.grad(F.embedding(ids, *only, position_ids=pos), only[k], g)[0], want[k])


@pytest.mark.parametrize("case", ["type", "width", "stride", "device"])
def test_refusals(case):
    wte = torch.zeros(10, 16, device=DEV, dtype=torch.bfloat16)
    ids = torch.zeros(1, 3, device=DEV, dtype=torch.long)
    if case == "type":
        wte = wte.float()
    elif case == "width":
        wte = torch.zeros(10, 12, device=DEV, dtype=torch.bfloat16)
    elif case == "stride":
        wte = torch.zeros(10, 32, device=DEV, dtype=torch.bfloat16)[:, :16]
    else:
        ids = ids.cpu()
    with pytest.raises(ValueError):
        F.embedding(ids, wte)


def test_tables_on_sixteen_bytes():
    """Tables that begin between two 32-byte sectors: another width of accesses, the same bits."""
    torch.manual_seed(4)
    flat = torch.randn(8 + 300 * 64, device=DEV).bfloat16()
    off = flat[8:].view(300, 64).requires_grad_(True)
    on = flat[8:].view(300, 64).clone().requires_grad_(True)
    assert off.data_ptr() % 32 == 16 and on.data_ptr() % 32 == 0
    ids = torch.randint(0, 300, (2, 90), device=DEV)
    g = torch.randn(2, 90, 64, device=DEV).bfloat16()
    a, b = F.embedding(ids, off, off, scale=1.5), F.embedding(ids, on, on, scale=1.5)
    assert torch.equal(a, b)
    assert torch.equal(a, (1.5 * on[ids].float() + on[:90].float()).bfloat16())
    assert torch.equal(*(torch.autograd.grad(x, t, g)[0] for x, t in ((a, off), (b, on))))
