"""Packed attention where every CTA takes many work items one after another: claims, the ring of items, the phases of every
barrier across items, and several query heads of a group in one CTA.  Bounds and reference as in test_packed_sequences_gpu."""
import math
import random

import pytest
import torch

from mist_b200.ops import functional as F
from mist_b200.ops import native
from mist_b200.ops import packed as P
from tests.test_packed_sequences_gpu import BF, DEV, _cu, _run

pytestmark = pytest.mark.gpu
CTAS = 148


def _lengths(n, longest, seed=0):
    """Uneven, most of them short and no multiple of 16, a few empty or of a single token."""
    r = random.Random(seed)
    return [r.choice([0, 1, 17, 127, 129]) if r.random() < 0.15 else 1 + int(longest ** r.random()) for _ in range(n)]


def _items(lens, heads, step):
    return sum(-(-n // step) for n in lens) * heads


@pytest.mark.parametrize("d", [64, 80, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_many_items_per_cta(d, causal):
    lens = _lengths(300, 300, seed=d)
    assert _items(lens, 16, 256) > 5 * CTAS and _items(lens, 16, 128) > 5 * CTAS
    _run(lens, lens, 16, 16, d, causal, seed=d, extra=3)


@pytest.mark.parametrize("causal", [True, False])
def test_many_items_with_keys_of_other_lengths(causal):
    lens_q, lens_k = _lengths(200, 300, seed=1), _lengths(200, 400, seed=2)
    assert _items(lens_q, 12, 256) > 5 * CTAS and _items(lens_k, 12, 128) > 5 * CTAS
    _run(lens_q, lens_k, 12, 4, 64, causal)


@pytest.mark.parametrize("nh,hk,d,unit", [(32, 8, 128, 4), (32, 8, 64, 4), (24, 8, 80, 3), (16, 8, 128, 2), (32, 4, 64, 4)])
@pytest.mark.parametrize("causal", [True, False])
def test_several_heads_of_a_group_in_one_cta(nh, hk, d, unit, causal):
    """Documents of one, two, three and more blocks of queries: what a head sees is odd, even and 1."""
    lens = [700, 1, 128, 256, 384, 385, 100, 0, 513, 90, 640, 17] + _lengths(40, 300, seed=3)
    lens.append(max(0, 5300 - sum(lens)))
    assert P._backward_sizes(sum(lens), sum(lens), nh, hk, d)[0] == unit
    assert _items(lens, nh // unit, 128) > CTAS
    _run(lens, lens, nh, hk, d, causal, seed=nh)


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("nh,hk,d,causal", [(16, 16, 64, True), (16, 16, 128, False), (32, 8, 128, True)])
def test_a_sequence_reaches_no_other_behind_many_items(poison, nh, hk, d, causal):
    lens = _lengths(250, 250, seed=5) + [300, 33, 200, 129]
    cu = _cu(lens)
    r = random.Random(6)
    bad = set(r.sample(range(len(lens)), 80))
    torch.manual_seed(2)
    t = [torch.randn(cu[-1] + 40, n, d, device=DEV).bfloat16() for n in (nh, hk, hk, nh)]

    def run(q, k, v, g):
        q, k, v = (x.clone().requires_grad_(True) for x in (q, k, v))
        o = F.attention_varlen(q, k, v, F.PackedSequences(torch.tensor(cu, device=DEV), cu[-1] + 40), causal=causal)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v), g)]

    clean = run(*t)
    dirty = [x.clone() for x in t]
    rows = torch.zeros(cu[-1] + 40, dtype=torch.bool, device=DEV)
    rows[cu[-1]:] = True
    for i in bad:
        rows[cu[i]:cu[i + 1]] = True
    for x in dirty:
        x[rows] = poison
    got = run(*dirty)
    native.check_status()
    good = ~rows
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, clean):
        if name == "dq":      # summed over the key blocks in no fixed order: a rounding of the bf16 result apart
            assert ((x[good].float() - y[good].float()).abs() <= 2 * BF * y[good].float().abs() + 1e-5).all()
        else:
            assert torch.equal(x[good], y[good]), name
    assert not got[0][cu[-1]:].any() and all(not x[cu[-1]:].any() for x in got[2:])


def test_many_items_through_the_projection():
    """The form that training takes: one gradient tensor, rotated heads, several heads of a group in a CTA."""
    torch.manual_seed(7)
    h, hk, d = 32, 8, 128
    lens = _lengths(60, 300, seed=8)
    lens.append(max(0, 5300 - sum(lens)))
    cu = _cu(lens)
    x = torch.randn(1, cu[-1], h + 2 * hk, d, device=DEV).bfloat16()
    g = torch.randn(1, cu[-1], h, d, device=DEV).bfloat16()
    seqs = F.PackedSequences(cu, device=DEV)
    leaf = x.clone().requires_grad_(True)
    out = F.attention_projected(leaf.clone(), hk, 1 / math.sqrt(d), True, seqs.rotary(d, 1e4), packed=seqs)
    grad = torch.autograd.grad(out, leaf, g)[0]
    ref, ref_g = torch.zeros_like(out), torch.zeros_like(grad)
    for a, b in zip(cu, cu[1:]):
        if b == a:
            continue
        leaf = x[:, a:b].clone().requires_grad_(True)
        o = F.attention_projected(leaf.clone(), hk, 1 / math.sqrt(d), True, (*F.rope_tables(b - a, d, 1e4, x.device), d))
        ref[:, a:b] = o.detach()
        ref_g[:, a:b] = torch.autograd.grad(o, leaf, g[:, a:b])[0]
    native.check_status()
    # as in test_projected_strides_rotary_and_groups: the same numbers, other orders of a few fp32 sums
    assert ((out.float() - ref.float()).abs() <= 2 * BF * ref.float().abs() + 1e-3).all()
    assert (grad.float() - ref_g.float()).norm() <= 2 * BF * ref_g.float().norm()
