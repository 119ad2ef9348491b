"""One packing on several streams: whoever comes second waits for what the first one made."""
import math

import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native

pytestmark = pytest.mark.gpu
DEV = "cuda"
DELAY = 40_000_000        # cycles, some 20 ms: what is made behind it is not there when the other stream begins
LENS = [100, 30, 257]
CU = [0, 100, 130, 387]


def _run(x, seqs, g):
    leaf = x.clone().requires_grad_(True)
    out = F.attention_projected(leaf.clone(), 2, 1 / math.sqrt(64), True, seqs.rotary(64, 1e4), packed=seqs)
    return out.detach(), torch.autograd.grad(out, leaf, g)[0]


def _same(a, b):
    """dQ of three key blocks is summed in no fixed order, and rotated in bf16 afterwards."""
    assert torch.equal(a[0], b[0])
    assert ((a[1].float() - b[1].float()).norm() <= 2 * 2 ** -8 * b[1].float().norm())


@pytest.mark.parametrize("offsets", ["host", "device"])
def test_two_streams_share_a_packing(offsets):
    torch.manual_seed(0)
    x, g = torch.randn(1, 387, 8, 64, device=DEV).bfloat16(), torch.randn(1, 387, 4, 64, device=DEV).bfloat16()
    cu = CU if offsets == "host" else torch.tensor(CU, device=DEV, dtype=torch.int32)

    def make():
        return F.PackedSequences(cu, 387, device=DEV)

    want = _run(x, make(), g)
    torch.cuda.synchronize()
    first, second, third = (torch.cuda.Stream() for _ in range(3))
    with torch.cuda.stream(first):
        torch.cuda._sleep(DELAY)
        seqs = make()
    with torch.cuda.stream(second):             # the plan, and then the tables, are not there yet
        at = seqs.positions + 0
        torch.cuda._sleep(DELAY)
        seqs.rotary(64, 1e4)
    with torch.cuda.stream(third):
        got = _run(x, seqs, g)
    with torch.cuda.stream(first):
        again = _run(x, seqs, g)
    torch.cuda.synchronize()
    native.check_status()
    assert at.tolist() == [i for n in LENS for i in range(n)]
    _same(got, want)
    _same(again, want)


def test_memory_of_a_packing_is_not_handed_out_under_another_stream():
    """Dropped while a kernel of another stream still has to read it: its block waits for that stream."""
    torch.manual_seed(1)
    x, g = torch.randn(1, 387, 8, 64, device=DEV).bfloat16(), torch.randn(1, 387, 4, 64, device=DEV).bfloat16()
    want = _run(x, F.PackedSequences(CU, 387, device=DEV), g)
    side = torch.cuda.Stream()
    seqs = F.PackedSequences(CU, 387, device=DEV)
    size = seqs.plan.numel()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(DELAY)
        with torch.no_grad():
            out = F.attention_projected(x.clone(), 2, 1 / math.sqrt(64), True, seqs.rotary(64, 1e4), packed=seqs)
    del seqs
    junk = [torch.zeros(size, dtype=torch.uint8, device=DEV) for _ in range(20)]       # empty plans: no items, in bounds
    torch.cuda.synchronize()
    assert len(junk) == 20 and torch.equal(out, want[0])


def test_a_packing_of_before_in_a_captured_graph():
    torch.manual_seed(2)
    x = torch.randn(1, 387, 8, 64, device=DEV).bfloat16()
    seqs = F.PackedSequences(CU, 387, device=DEV)

    def run():
        with torch.no_grad():
            return F.attention_projected(x.clone(), 2, 1 / math.sqrt(64), True, seqs.rotary(64, 1e4), packed=seqs)

    want = run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
        inside = F.PackedSequences(torch.tensor(CU, device="cpu"), 387, device=DEV)
        other = F.attention_projected(x.clone(), 2, 1 / math.sqrt(64), True, inside.rotary(64, 1e4), packed=inside)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(other.detach(), want)
