"""Offsets of packed attention, on the host and on the GPU: the same rows, the same refusals."""
import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tensors(rows, heads=2, d=64, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(rows, heads, d, device=DEV, generator=g).bfloat16().requires_grad_(True) for _ in range(3)]


@pytest.mark.parametrize("cu,rows", [([0, 30, 70], 70), ([0, 30, 70], 100), ([0, 1], 100), ([0, 0], 100), ([0], 100)])
def test_rows_do_not_depend_on_where_the_offsets_are(cu, rows):
    t = _tensors(rows)
    outs = [F.attention_varlen(*t, c) for c in (cu, torch.tensor(cu), torch.tensor(cu, device=DEV),
                                                torch.tensor(cu, device=DEV, dtype=torch.int32))]
    assert outs[0].shape[0] == (cu[-1] or rows)
    grads = [torch.autograd.grad(o, t, torch.ones_like(o)) for o in outs]
    for o, g in zip(outs[1:], grads[1:]):
        assert torch.equal(o, outs[0]) and all(torch.equal(a, b) for a, b in zip(g, grads[0]))
    other = F.attention_varlen(*t, torch.tensor(cu, device=DEV), cu, causal=False)
    assert torch.equal(other, F.attention_varlen(*t, cu, torch.tensor(cu, device=DEV), causal=False))
    assert other.shape[0] == (cu[-1] or rows)
    native.check_status()


@pytest.mark.parametrize("cu", [[1, 70], [0, 50, 20, 70], [0, 71], [-5, 70]])
def test_impossible_offsets_on_the_gpu_are_refused(cu):
    """The kernels clamp them (which keeps them inside the tensors); the call raises."""
    t = _tensors(70)
    ends = [0] * (len(cu) - 1) + [70]
    for bad, keys in ((torch.tensor(cu, device=DEV), None), (torch.tensor(cu, device=DEV), ends), (ends, torch.tensor(cu, device=DEV))):
        with pytest.raises(ValueError):
            F.attention_varlen(*t, bad, keys)
    native.check_status()


def test_a_captured_call_reads_nothing_back():
    t, cu = _tensors(100), torch.tensor([0, 30, 70], device=DEV, dtype=torch.int32)
    with torch.no_grad():
        want = F.attention_varlen(*t, cu)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            F.attention_varlen(*t, cu)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = F.attention_varlen(*t, cu)
        graph.replay()
    torch.cuda.synchronize()
    assert out.shape[0] == 100 and torch.equal(out[:70], want) and not out[70:].any()


@pytest.mark.parametrize("n", [1, 991, 992, 993, 2500])
def test_offsets_of_the_host_reach_the_device(n):
    cu = [3 * i for i in range(n)]
    seqs = F.PackedSequences(cu, device=DEV)
    assert seqs.cu_q.tolist() == cu and seqs.cu_q.dtype == torch.int32


@pytest.mark.parametrize("causal", [True, False])
def test_offsets_of_the_host_in_a_captured_graph(causal):
    """Nothing of the host's is read when the graph is replayed, and capturing waits for nothing."""
    t, cu = _tensors(70), [0, 30, 70]
    with torch.no_grad():
        want = F.attention_varlen(*t, cu, causal=causal)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            F.attention_varlen(*t, cu, causal=causal)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = F.attention_varlen(*t, torch.tensor(cu), causal=causal)
            other = F.attention_varlen(*t, cu, [0, 10, 70], causal=causal)
        del cu
        for _ in range(2):
            out.fill_(7.0)
            graph.replay()
        assert torch.equal(out, want)
        assert torch.equal(other, F.attention_varlen(*t, [0, 30, 70], [0, 10, 70], causal=causal))


def test_the_ends_of_calls_on_two_streams_are_their_own():
    """Calls on both streams at once, behind a delay on the first: each reads back its own ends."""
    t = _tensors(100)
    cus = [torch.tensor([0, 30, 70], device=DEV), torch.tensor([0, 10, 90], device=DEV)]
    with torch.no_grad():
        want = [F.attention_varlen(*t, cu) for cu in cus]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        for _ in range(3):
            for s, cu, w in zip(streams, cus, want):
                with torch.cuda.stream(s):
                    torch.cuda._sleep(1_000_000)
                    out = F.attention_varlen(*t, cu)
                assert out.shape == w.shape
                s.synchronize()
                assert torch.equal(out, w)


def test_a_call_that_raises_keeps_its_pinned_numbers():
    """Tensors that do not fit are refused behind the launch of the plan, which writes them when its turn comes."""
    from mist_b200.ops import packed
    q, k, v = _tensors(70)
    cu = torch.tensor([0, 30, 70], device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    free = packed._ends.setdefault(q.device.index, [])
    kept = list(free)
    free.clear()                                        # the call takes new ones
    with torch.cuda.stream(side):
        torch.cuda._sleep(40_000_000)
        with pytest.raises(ValueError):
            F.attention_varlen(q, k, v[:, :1], cu)
    others = [torch.full((2,), 7, dtype=torch.int32, pin_memory=True) for _ in range(50)]
    torch.cuda.synchronize()
    assert all(t.tolist() == [7, 7] for t in others)
    import gc
    gc.collect()
    assert len(free) == 1 and free[0][0].tolist() == [70, 70]
    free.extend(kept)


def test_offsets_on_the_gpu_of_tensors_on_the_host():
    x = torch.randn(100, 2, 16)
    for cu in (torch.tensor([0, 30, 70]), torch.tensor([0, 30, 70], device=DEV)):
        assert torch.equal(F.attention_varlen(x, x, x, cu), F.attention_varlen(x, x, x, [0, 30, 70]))
    with pytest.raises(ValueError):
        F.attention_varlen(x, x, x, torch.tensor([1, 70], device=DEV))
