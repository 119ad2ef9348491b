"""Packed sequences on the reference path: positions, attention inside each sequence, the packed projection with rotary
positions that start again, refusals."""
import math

import pytest
import torch

from mist_b200.ops import functional as F

LENS = [5, 0, 1, 9, 3]
CU = [0, 5, 5, 6, 15, 18]


def test_positions_and_rows_behind_the_last_sequence():
    seqs = F.PackedSequences(CU, 20)
    assert seqs.n == 5 and seqs.total_q == seqs.total_k == 20
    want = [i for n in LENS for i in range(n)] + [0, 1]
    assert seqs.positions.tolist() == want
    assert F.PackedSequences(torch.tensor(CU)).total_q == 18
    assert F.PackedSequences([0]).positions.numel() == 0


@pytest.mark.parametrize("causal", [True, False])
def test_cross_lengths_and_padding_rows(causal):
    torch.manual_seed(0)
    cu_k = [0, 2, 8, 8, 12, 19]
    q = torch.randn(20, 4, 16, requires_grad=True)
    k, v = (torch.randn(19, 2, 16, requires_grad=True) for _ in range(2))
    seqs = F.PackedSequences(CU, 20, cu_k, 19)
    out = F.attention_varlen(q, k, v, seqs, causal=causal)
    assert out.shape == q.shape and not out[18:].any() and not out[5:6].any()       # behind the end; no keys
    ref = torch.zeros_like(q)
    for i in range(5):
        a, b = slice(CU[i], CU[i + 1]), slice(cu_k[i], cu_k[i + 1])
        if CU[i + 1] > CU[i] and cu_k[i + 1] > cu_k[i]:
            ref = ref.index_copy(0, torch.arange(20)[a], F._ref_attention(q[None, a], k[None, b], v[None, b], 0.25, causal)[0][0])
    assert torch.allclose(out, ref, atol=1e-5)
    g = torch.randn_like(out)
    got, want = torch.autograd.grad(out, (q, k, v), g), torch.autograd.grad(ref, (q, k, v), g)
    assert all(torch.allclose(a, b, atol=1e-4) for a, b in zip(got, want))
    host = F.attention_varlen(q, k, v, CU, cu_k, causal=causal)                    # offsets known here: no rows behind them
    assert host.shape[0] == 18 and torch.equal(host, out[:18])


@pytest.mark.parametrize("kv_heads,rot", [(4, 0), (2, 8), (1, 16)])
@pytest.mark.parametrize("batch", [1, 2])
def test_projection_is_the_documents_one_by_one(kv_heads, rot, batch):
    torch.manual_seed(1)
    h, d = 4, 16
    qkv = torch.randn(batch, 18 // batch, h + 2 * kv_heads, d, requires_grad=True)
    seqs = F.PackedSequences(CU, 18)
    out = F.attention_projected(qkv, kv_heads, 1 / math.sqrt(d), True, seqs.rotary(rot, 1e4) if rot else None, packed=seqs)
    assert out.shape == (batch, 18 // batch, h, d)
    parts, flat = [], qkv.reshape(1, 18, -1, d)
    for a, b in zip(CU, CU[1:]):
        if b > a:
            tables = (*F.rope_tables(b - a, rot, 1e4, "cpu"), rot) if rot else None
            parts.append(F.attention_projected(flat[:, a:b], kv_heads, 1 / math.sqrt(d), True, tables))
    ref = torch.cat(parts, 1).view(out.shape)
    assert torch.allclose(out, ref, atol=1e-5)
    g = torch.randn_like(out)
    assert torch.allclose(torch.autograd.grad(out, qkv, g)[0], torch.autograd.grad(ref, qkv, g)[0], atol=1e-4)


@pytest.mark.parametrize("cu,total", [([1, 4], None), ([0, 4, 3], None), ([0, 9], 8), ([], None), (torch.zeros(2, 2), None),
                                      (torch.tensor([0.0, 2.0]), None), ([0, 4], -1)])
def test_offsets_that_are_refused(cu, total):
    with pytest.raises(ValueError):
        F.PackedSequences(cu, total)


def test_tensors_that_do_not_fit():
    q = torch.randn(18, 4, 16)
    seqs = F.PackedSequences(CU)
    with pytest.raises(ValueError):
        F.attention_varlen(q[:17], q[:17], q[:17], seqs)
    with pytest.raises(ValueError):
        F.attention_varlen(q, q[:, :3], q[:, :3], seqs)
    with pytest.raises(ValueError):
        F.attention_varlen(q, q, q[:, :2], seqs)
    with pytest.raises(ValueError):
        F.PackedSequences(CU, None, [0, 5])
    with pytest.raises(ValueError):
        F.attention_projected(q[None], 1, 0.25, True, seqlens=torch.tensor([18]), packed=seqs)
    with pytest.raises(ValueError):
        F.attention_projected(q[None], 2, 0.25, True, packed=seqs)


@pytest.mark.parametrize("case", ["rows", "width", "type", "strided", "more than a head"])
def test_rotary_tables_that_do_not_fit_are_refused(case):
    """Each token has a row; a table of positions, as the batched form takes it, is too short."""
    seqs = F.PackedSequences([0, 5, 12])
    qkv = torch.randn(1, 12, 3, 2, 16)
    cos, sin, rot = seqs.rotary(16, 10000.0)
    F.attention_projected(qkv, 2, 0.25, True, (cos, sin, rot), packed=seqs)
    if case == "rows":
        cos, sin = cos[:7].contiguous(), sin[:7].contiguous()
    elif case == "width":
        rot = 8
    elif case == "type":
        cos = cos.double()
    elif case == "strided":
        sin = torch.cat([sin, sin], 1)[:, ::2]
    else:
        cos, sin, rot = seqs.rotary(32, 10000.0)
    with pytest.raises(ValueError):
        F.attention_projected(qkv, 2, 0.25, True, (cos, sin, rot), packed=seqs)
