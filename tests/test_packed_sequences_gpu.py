"""Attention over packed sequences on the GPU, forward and backward, against 64 bits, sequence by sequence.

Tolerances, element by element.  The probabilities are rounded to bf16 for the product with V, the output once more: off by
at most 2^-8 (sum_j p_j |v_j| + |o|).  dV has the same form with |dO| in the place of |v|.  dS = P (dP - delta) is rounded
(2^-8 |dS|), and delta is a sum over the rounded output: off by at most E = sum_d |dO| (the bound on o); so
|error of dS| <= 2^-8 |dS| + P E, which dQ and dK carry on as sums over |K| and |Q|, rounded once themselves.  Where a group's
heads are added from several parts, those are rounded too: one more 2^-8 of the sum of the magnitudes.  Scores are sums of
d products in fp32 (d * 2^-23 of the sum of their magnitudes, as an exponent), far below the rest; 1.1 times all covers it."""
import math

import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = 2.0 ** -8
ITEM, HEAD = 32, 16


def _cu(lens):
    return [0] + torch.tensor(lens).cumsum(0).tolist() if len(lens) else [0]


def _exact(q, k, v, g, scale, causal):
    """o, dq, dk, dv of one sequence in 64 bits, each with its bound."""
    n, nh, d = q.shape
    m, hk = k.shape[0], k.shape[1]
    rep = nh // hk
    qd, gd = (t.double().transpose(0, 1) for t in (q, g))
    kd, vd = (t.double().transpose(0, 1).repeat_interleave(rep, 0) for t in (k, v))
    s = qd @ kd.transpose(1, 2) * scale
    if causal:
        s.masked_fill_(torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1), float("-inf"))
    p = torch.softmax(s, -1).nan_to_num(0.0)
    o, o_err = p @ vd, BF * (p @ vd.abs())
    o_err = o_err + BF * o.abs()
    dv, dv_err = p.transpose(1, 2) @ gd, BF * (p.transpose(1, 2) @ gd.abs())
    ds = p * (gd @ vd.transpose(1, 2) - (gd * o).sum(-1, keepdim=True))
    ds_err = BF * ds.abs() + p * (gd.abs() * o_err).sum(-1, keepdim=True)
    dq, dq_err = ds @ kd * scale, ds_err @ kd.abs() * scale
    dk, dk_err = ds.transpose(1, 2) @ qd * scale, ds_err.transpose(1, 2) @ qd.abs() * scale
    dk_mag, dv_mag = ds.abs().transpose(1, 2) @ qd.abs() * scale, p.transpose(1, 2) @ gd.abs()

    def groups(t):
        return t.view(hk, rep, m, d).sum(1)

    def back(t):
        return t.transpose(0, 1)

    dk, dv, dk_err, dv_err, dk_mag, dv_mag = (groups(t) for t in (dk, dv, dk_err, dv_err, dk_mag, dv_mag))
    more = BF if rep > 1 else 0.0
    return [(back(a), 1.1 * back(e) + 1e-6) for a, e in
            ((o, o_err), (dq, dq_err + BF * dq.abs()), (dk, dk_err + BF * dk.abs() + more * dk_mag),
             (dv, dv_err + BF * dv.abs() + more * dv_mag))]


def _check(got, want_err, what):
    want, err = want_err
    bad = (got.double() - want).abs() > err
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / err).max()))


def _run(lens_q, lens_k, nh, hk, d, causal, seed=0, extra=0):
    torch.manual_seed(seed)
    cu_q, cu_k = _cu(lens_q), _cu(lens_k)
    tq, tk = cu_q[-1] + extra, cu_k[-1] + extra
    q = torch.randn(tq, nh, d, device=DEV).bfloat16().requires_grad_(True)
    k, v = (torch.randn(tk, hk, d, device=DEV).bfloat16().requires_grad_(True) for _ in range(2))
    g = torch.randn(tq, nh, d, device=DEV).bfloat16()
    seqs = F.PackedSequences(torch.tensor(cu_q, device=DEV), tq, None if lens_q is lens_k else torch.tensor(cu_k, device=DEV),
                             None if lens_q is lens_k else tk)
    o = F.attention_varlen(q, k, v, seqs, causal=causal)
    grads = torch.autograd.grad(o, (q, k, v), g)
    native.check_status()
    scale = 1 / math.sqrt(d)
    for i in range(len(lens_q)):
        a, b = slice(cu_q[i], cu_q[i + 1]), slice(cu_k[i], cu_k[i + 1])
        want = _exact(q.detach()[a], k.detach()[b], v.detach()[b], g[a], scale, causal)
        for name, t, at, w in zip(("o", "dq", "dk", "dv"), (o, *grads), (a, a, b, b), want):
            _check(t.detach()[at], w, (name, i, lens_q[i], lens_k[i]))
    for t, end in zip((o, *grads), (cu_q[-1], cu_q[-1], cu_k[-1], cu_k[-1])):
        assert not t[end:].any()
    return q, k, v, g, seqs, o, grads


SHORT = [1, 2, 15, 16, 17, 0, 63, 64, 65]
EDGES = [127, 128, 129, 0, 255, 256, 257, 1, 300]


@pytest.mark.parametrize("lens", [[1], [40], SHORT, EDGES, [700, 3, 1025]])
@pytest.mark.parametrize("nh,hk,d", [(2, 2, 64), (4, 1, 128), (6, 2, 80), (3, 3, 16), (2, 1, 112)])
@pytest.mark.parametrize("causal", [True, False])
def test_self_attention(lens, nh, hk, d, causal):
    _run(lens, lens, nh, hk, d, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("extra", [0, 5, 300])
def test_other_lengths_of_keys_and_rows_behind_the_end(causal, extra):
    """Sequences without keys or without queries, more queries than keys (the first of them see nothing), and fewer."""
    _run([5, 0, 130, 64, 257, 7, 0], [9, 33, 128, 0, 100, 400, 0], 4, 2, 64, causal, extra=extra)


def test_nothing_at_all():
    for lens in ([], [0, 0]):
        seqs = F.PackedSequences(torch.tensor(_cu(lens), device=DEV), 0)
        x = torch.zeros(0, 2, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        o = F.attention_varlen(x, x, x, seqs)
        assert o.shape == (0, 2, 64) and torch.autograd.grad(o.sum(), x)[0].shape == x.shape
    _run([3, 4], [0, 0], 2, 2, 64, False)          # queries without any key, keys without any query
    _run([0, 0], [3, 4], 2, 2, 64, True)


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), 3e38])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [64, 128])
def test_a_sequence_reaches_no_other(poison, causal, d):
    """What stands in one sequence, or behind the last one, changes nothing in the others."""
    lens, bad = [70, 33, 200, 129, 300, 20], (1, 3)
    cu = _cu(lens)
    torch.manual_seed(2)
    t = [torch.randn(cu[-1] + 40, 2, d, device=DEV).bfloat16() for _ in range(4)]

    def run(q, k, v, g):
        q, k, v = (x.clone().requires_grad_(True) for x in (q, k, v))
        o = F.attention_varlen(q, k, v, F.PackedSequences(torch.tensor(cu, device=DEV), cu[-1] + 40), causal=causal)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), g)]

    clean = run(*t)
    dirty = [x.clone() for x in t]
    for x in dirty:
        for i in bad:
            x[cu[i]:cu[i + 1]] = poison
        x[cu[-1]:] = poison
    got = run(*dirty)
    native.check_status()
    for i in range(len(lens)):
        if i in bad:
            continue
        a = slice(cu[i], cu[i + 1])
        for name, x, y in zip(("o", "dq", "dk", "dv"), got, clean):
            if name == "dq":      # summed over the key blocks in no fixed order: a rounding of the bf16 result apart
                assert ((x[a].float() - y[a].float()).abs() <= 2 * BF * y[a].float().abs() + 1e-5).all(), (name, i)
            else:
                assert torch.equal(x[a], y[a]), (name, i)
    assert not got[0][cu[-1]:].any() and all(not x[cu[-1]:].any() for x in got[2:])


def _lists(seqs):
    """(backward, causal) -> items of a plan, as the kernels read them."""
    plan, n = seqs.plan.cpu(), seqs.n
    fwd, bwd = HEAD + ITEM * (seqs.total_q // 256 + n + 1), HEAD + ITEM * (seqs.total_k // 128 + n + 1)
    assert plan.numel() == 2 * (fwd + bwd) + 9 * seqs.total_q
    single = plan[2 * (fwd + bwd) + 8 * seqs.total_q:].tolist()      # a byte per query row
    out, heads = {}, {}
    for backward in (0, 1):
        for causal in (0, 1):
            at = 2 * fwd + causal * bwd if backward else causal * fwd
            size = bwd if backward else fwd
            words = plan[at:at + size].view(torch.int32)
            count = int(words[0])
            assert 0 <= count <= (size - HEAD) // ITEM
            out[backward, causal] = words[4:4 + 8 * count].view(-1, 8)[:, :5].tolist()
            heads[backward, causal] = words[:4].tolist()
    return out, heads, single


@pytest.mark.parametrize("lens_q,lens_k,extra", [(SHORT, SHORT, 0), (EDGES, EDGES, 7), ([], [], 10), ([5000], [5000], 0),
                                                  ([3, 0, 900], [700, 2, 0], 300), ([1] * 2000, [1] * 2000, 0)])
def test_plan_covers_every_row_once(lens_q, lens_k, extra):
    cu_q, cu_k = _cu(lens_q), _cu(lens_k)
    tq, tk = cu_q[-1] + extra, cu_k[-1] + extra
    seqs = F.PackedSequences(torch.tensor(cu_q, device=DEV), tq, torch.tensor(cu_k, device=DEV), tk)
    assert seqs.positions.tolist() == [i for n in lens_q for i in range(n)] + list(range(extra))
    lists, heads, single = _lists(seqs)
    want = []
    for n, m in [*zip(lens_q, lens_k), (extra, 0)]:         # at most one block of keys seen: whole (1), causal (2)
        for i in range(n):
            keys = min(m, i // 128 * 128 + 128 + m - n)
            want.append((1 if m <= 128 else 0) + (2 if keys <= 128 else 0))
    assert single == want
    for (backward, causal), items in lists.items():
        step, total = (128, tk) if backward else (256, tq)
        seen, costs = torch.zeros(total, dtype=torch.int32), []
        for q_row, sq, k_row, sk, first in items:
            row, n = (k_row, sk) if backward else (q_row, sq)
            assert first % step == 0 and first < n
            seen[row + first:row + min(n, first + step)] += 1
            off = sk - sq
            if backward:
                costs.append(max(0, -(-sq // 128) - (max(0, first - off) // 128 if causal else 0)))
            else:
                costs.append(max(0, -(-(min(sk, min(sq, first + 256) + off) if causal else sk) // 128)))
        assert (seen == 1).all()
        assert costs == sorted(costs, reverse=True)
        assert heads[backward, causal] == [len(items), sum(costs), max(costs, default=0), 0]


@pytest.mark.parametrize("cu", [[0, 50, 20, 90], [3, 10, 200, 400], [0, -7, 60, 2 ** 31 - 1], [5, 4, 3, 2]])
def test_plan_of_impossible_offsets_stays_inside(cu):
    total = 100
    seqs = F.PackedSequences(torch.tensor(cu, device=DEV), total)
    for items in _lists(seqs)[0].values():
        for q_row, sq, k_row, sk, first in items:
            assert 0 <= q_row and 0 <= sq and q_row + sq <= total
            assert 0 <= k_row and 0 <= sk and k_row + sk <= total and first >= 0


def test_projected_strides_rotary_and_groups():
    torch.manual_seed(4)
    h, hk, d, lens = 8, 2, 128, [130, 1, 65, 300]
    cu = _cu(lens)
    x = torch.randn(2, cu[-1] // 2, h + 2 * hk, d, device=DEV).bfloat16()
    seqs = F.PackedSequences(torch.tensor(cu, device=DEV), cu[-1])
    rotary = seqs.rotary(64, 1e4)
    g = torch.randn(2, cu[-1] // 2, h, d, device=DEV).bfloat16()
    leaf = x.clone().requires_grad_(True)
    out = F.attention_projected(leaf.clone(), hk, 1 / math.sqrt(d), True, rotary, packed=seqs)
    (grad,) = torch.autograd.grad(out, leaf, g)
    flat, parts, grads = x.view(1, cu[-1], -1, d), [], []
    for a, b in zip(cu, cu[1:]):              # the documents one by one on the kernels of whole sequences
        leaf = flat[:, a:b].clone().requires_grad_(True)
        o = F.attention_projected(leaf.clone(), hk, 1 / math.sqrt(d), True, (*F.rope_tables(b - a, 64, 1e4, x.device), 64))
        parts.append(o)
        grads.append(torch.autograd.grad(o, leaf, g.view(1, cu[-1], h, d)[:, a:b])[0])
    native.check_status()
    # the same kernels on the same numbers, in blocks of the same rows: the order of the fp32 sums of dQ, and the number of
    # heads that one CTA adds, may differ, each a rounding to bf16 at most
    ref, ref_g = torch.cat(parts, 1).view(out.shape), torch.cat(grads, 1).view(grad.shape)
    assert ((out.float() - ref.float()).abs() <= 2 * BF * ref.float().abs() + 1e-3).all()
    assert ((grad.float() - ref_g.float()).norm() <= 2 * BF * ref_g.float().norm()).all()


def test_views_and_offsets_of_other_types():
    torch.manual_seed(5)
    lens = [33, 100, 7]
    cu = _cu(lens)
    qkv = torch.randn(cu[-1], 3, 4, 72, device=DEV).bfloat16()[..., 4:68]           # 64 of 72, an odd start
    q, k, v = qkv.unbind(1)
    want = F.attention_varlen(*(t.contiguous() for t in (q, k, v)), torch.tensor(cu, device=DEV, dtype=torch.int32))
    for offsets in (cu, torch.tensor(cu), torch.tensor(cu, device=DEV), torch.tensor(cu, device=DEV, dtype=torch.int32)):
        assert torch.equal(F.attention_varlen(q, k, v, offsets), want)
    one = k[:, :1].expand(-1, 4, -1)                                                # heads that are one
    assert torch.equal(F.attention_varlen(q, one, v, cu), F.attention_varlen(q, one.contiguous(), v, cu))


def test_streams_and_captured_graphs():
    lens = [[100, 30, 257], [64, 200, 123]]
    torch.manual_seed(6)
    t = [torch.randn(387, 4, 64, device=DEV).bfloat16().requires_grad_(True) for _ in range(3)]
    g = torch.randn(387, 4, 64, device=DEV).bfloat16()

    def once(cu):
        o = F.attention_varlen(*t, F.PackedSequences(cu, 387))
        return [o.detach(), *torch.autograd.grad(o, t, g)]

    offsets = [torch.tensor(_cu(x), device=DEV, dtype=torch.int32) for x in lens]
    want = [once(cu) for cu in offsets]
    torch.cuda.synchronize()
    side, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(4):
        with torch.cuda.stream(side[i % 2]):
            got.append(once(offsets[i % 2]))
    torch.cuda.synchronize()

    def same(a, b):
        for i, (x, y) in enumerate(zip(a, b)):
            if i == 1:
                assert ((x.float() - y.float()).abs() <= 2 * BF * y.float().abs() + 1e-5).all()
            else:
                assert torch.equal(x, y)

    for i in range(4):
        same(got[i], want[i % 2])
    graphs, outs, held = [], [], [cu.clone() for cu in offsets]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for cu in held:
            once(cu)
    torch.cuda.current_stream().wait_stream(s)
    for cu in held:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(once(cu))
    for swap in (0, 1):                        # both under way at once; then with the other's offsets
        for i in range(2):
            held[i].copy_(offsets[i ^ swap])
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        native.check_status()
        for i in range(2):
            same(outs[i], want[i ^ swap])


@pytest.mark.parametrize("case", ["type", "head", "device", "total"])
def test_refusals(case):
    x = torch.zeros(10, 2, 64, device=DEV, dtype=torch.bfloat16)
    cu = torch.tensor([0, 10], device=DEV)
    if case == "type":
        x = x.float()
    elif case == "head":
        x = torch.zeros(10, 2, 136, device=DEV, dtype=torch.bfloat16)
    elif case == "device":
        cu = F.PackedSequences([0, 10])
    else:
        cu = F.PackedSequences(cu, 11)
    with pytest.raises(ValueError):
        F.attention_varlen(x, x, x, cu)


def test_rotary_tables_of_a_captured_graph_stay_in_it():
    """Tables that a graph computes are not there for anyone before it is replayed."""
    seqs = F.PackedSequences([0, 30, 70], device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        F.PackedSequences([0, 30, 70], device=DEV).rotary(32, 10000.0)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = seqs.rotary(32, 10000.0)
    at = torch.cat([torch.arange(30), torch.arange(40)]).double()
    angles = torch.outer(at, 10000.0 ** (-torch.arange(0, 32, 2).double() / 32))
    outside = seqs.rotary(32, 10000.0)
    graph.replay()
    torch.cuda.synchronize()
    for cos, sin, rot in (outside, inside):
        assert rot == 32
        # angles up to 40 in fp32: half a step is 2^-19, three roundings of it on the way
        assert (cos.double().cpu() - angles.cos()).abs().max() < 2 ** -17
        assert (sin.double().cpu() - angles.sin()).abs().max() < 2 ** -17
