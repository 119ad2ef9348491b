"""Sequences packed back to back in one row of tokens, and attention inside each of them.

A :class:`PackedSequences` is made once per batch.  It holds the offsets, every token's position in its sequence, and the
work lists that the attention kernels walk (csrc/packed_plan.cu); all layers, forward and backward, use the same one, and
nothing is read back to the host (reference: csrc/flash_attn/flash_api.cpp:427, 814 ``varlen_fwd`` / ``varlen_bwd``, called
with offsets that mist/modules/mha.py:1233-1243 derives from a padding mask)."""
from __future__ import annotations

from typing import Optional

import torch

from . import native
from .native import call, ptr, stream, use_native


def _offsets(cu, device):
    """Offsets as int32 on the device, and as a list where they are known on the host (then checked)."""
    if isinstance(cu, torch.Tensor):
        if cu.dim() != 1 or cu.numel() < 1 or cu.is_floating_point():
            raise ValueError(f"offsets: a vector of integers expected, got {tuple(cu.shape)} of {cu.dtype}")
        if cu.is_cuda:
            return cu.to(device=device, dtype=torch.int32).contiguous(), None
    host = [int(x) for x in (cu.tolist() if isinstance(cu, torch.Tensor) else cu)]
    if not host or host[0] != 0 or any(b < a for a, b in zip(host, host[1:])):
        raise ValueError("offsets: they begin with 0 and do not fall")
    return torch.tensor(host, dtype=torch.int32, device=device), host


class PackedSequences:
    """``n`` sequences packed back to back: ``cu_seqlens`` holds the ``n + 1`` offsets (0 first), as a tensor or a list.

    ``total``: rows of the packed tensors, at least the last offset; rows behind it belong to no sequence.  It may be left
    out where the offsets are known on the host.  ``cu_seqlens_k`` / ``total_k``: offsets of the keys, where they are others
    than those of the queries.  Offsets on the GPU are not read back and not checked: ones that fall or pass ``total`` are
    clamped, which keeps every access inside the tensors, and what comes out is unspecified.  The object's tensors are made
    on the stream that is current then."""

    def __init__(self, cu_seqlens, total: Optional[int] = None, cu_seqlens_k=None, total_k: Optional[int] = None, device=None):
        if device is None:
            device = cu_seqlens.device if isinstance(cu_seqlens, torch.Tensor) else torch.device("cpu")
        device = torch.device(device)
        self.same = cu_seqlens_k is None
        self.cu_q, self.host_q = _offsets(cu_seqlens, device)
        self.cu_k, self.host_k = (self.cu_q, self.host_q) if self.same else _offsets(cu_seqlens_k, device)
        if self.cu_k.numel() != self.cu_q.numel():
            raise ValueError("as many sequences of keys as of queries expected")
        self.n = self.cu_q.numel() - 1
        self.total_q = self._total(total, self.host_q)
        self.total_k = self.total_q if self.same and total_k is None else self._total(total_k, self.host_k)
        self.device = self.cu_q.device
        self._rotary = {}
        self.plan = None
        if use_native(self.cu_q):
            size = native.kernels().mb_packed_plan_bytes(self.n, self.total_q, self.total_k)
            self.plan = torch.empty(size, dtype=torch.uint8, device=self.device)
            #: every query row's place in its sequence, int64 ``[total]``
            self.positions = torch.empty(self.total_q, dtype=torch.int64, device=self.device)
            if self.device.index == torch._C._cuda_getDevice():
                self._make_plan()
            else:
                with torch.cuda.device(self.device):
                    self._make_plan()
        else:
            at = torch.arange(self.total_q)
            self.positions = at - self.cu_q.long()[torch.searchsorted(self.cu_q, at, right=True) - 1]

    def _make_plan(self):
        call("mb_packed_plan", ptr(self.cu_q), ptr(self.cu_k), self.n, self.total_q, self.total_k, ptr(self.plan),
             ptr(self.positions), stream())

    @staticmethod
    def _total(total, host):
        if total is None:
            if host is None:
                raise ValueError("offsets on the GPU need the number of packed rows beside them")
            total = host[-1]
        if total < 0 or (host is not None and host[-1] > total):
            raise ValueError(f"{total} rows, but the offsets end at {host and host[-1]}")
        return int(total)

    def check(self, q, k):
        if q.shape[0] != self.total_q or k.shape[0] != self.total_k:
            raise ValueError(f"{q.shape[0]} query and {k.shape[0]} key rows, but the packing is of {self.total_q} and {self.total_k}")
        if q.device != self.device:
            raise ValueError(f"tensors on {q.device}, offsets on {self.device}")

    def rotary(self, rot_dim: int, base: float):
        """``(cos, sin, rot_dim)`` with a row for each packed token, that of its position."""
        key = (rot_dim, base)
        if key not in self._rotary:
            from .functional import rope_tables
            cos, sin = rope_tables(max(self.total_q, 1), rot_dim, base, self.device)
            self._rotary[key] = (cos[self.positions].contiguous(), sin[self.positions].contiguous(), rot_dim)
        return self._rotary[key]

    def _each(self):
        """``(queries, keys)`` slices of every sequence (reference path: reads the offsets)."""
        q, k = self.host_q or self.cu_q.tolist(), self.host_k or self.cu_k.tolist()
        return [(slice(q[i], q[i + 1]), slice(k[i], k[i + 1])) for i in range(self.n)]


def _rows(t):
    """``t`` ``[rows, heads, d]`` as the kernels' copies can address it."""
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or ptr(t) % 16 or (t.shape[0] > 1 and t.stride(0) == 0) \
            or (t.shape[1] > 1 and t.stride(1) == 0):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def forward(q, k, v, packed: PackedSequences, scale: float, causal: bool):
    """Attention of ``q`` ``[total_q, heads, d]`` over ``k``, ``v`` ``[total_k, kv heads, d]`` inside each sequence:
    ``(o, lse [heads, total_q])``."""
    total, nh, d = q.shape
    if not use_native(q):
        from .functional import _ref_attention
        o = torch.zeros_like(q, memory_format=torch.contiguous_format)
        lse = torch.full((nh, total), float("-inf"), dtype=torch.float32)
        for a, b in packed._each():
            if a.stop > a.start and b.stop > b.start:
                oi, li = _ref_attention(q[None, a], k[None, b], v[None, b], scale, causal)
                o[a], lse[:, a] = oi[0], li[0]
        return o, lse
    o = torch.empty(total, nh, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(nh * total + 1, dtype=torch.float32, device=q.device)      # and the count of claimed work items
    claimed = ptr(lse) + 4 * nh * total
    lse = lse[:nh * total].view(nh, total)
    call("mb_attn_fwd_packed", ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(packed.plan),
         claimed if native.kernels().mb_attn_fwd_packed_counters(packed.n, total, nh) else 0, packed.n, total, k.shape[0], nh,
         k.shape[1], d, q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), nh * d, d, scale,
         int(causal), stream())
    return o, lse


def backward(dout, q, k, v, o, lse, packed: PackedSequences, scale: float, causal: bool, out=None):
    """``(dq, dk, dv)``; with ``out`` written into those (possibly strided) tensors."""
    from . import attention_bwd
    if out is None:
        out = tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    dq, dk, dv = out
    if not use_native(q):
        for t in out:
            t.zero_()
        for a, b in packed._each():
            if a.stop > a.start and b.stop > b.start:
                for t, at, g in zip(out, (a, b, b), attention_bwd._reference(dout[None, a], q[None, a], k[None, b], v[None, b],
                                                                            scale, causal)):
                    t[at] = g[0]
        return out
    total, nh, d = q.shape
    nkv = k.shape[1]
    dout = dout.contiguous()
    if ptr(dout) % 16:
        dout = dout.clone()
    unit = attention_bwd._unit_heads(q[None], k[None])
    parts = nh // nkv // unit
    gk, gv = dk, dv
    if parts > 1:        # a CTA sums `unit` heads of a group; the rest is added from a copy per unit
        gk, gv = (torch.empty(k.shape[0], nkv * parts, d, dtype=q.dtype, device=q.device) for _ in range(2))
    delta = torch.empty(nh * total + 1, dtype=torch.float32, device=q.device)    # and the count of claimed work items
    dq_acc = torch.empty(nh, total, d, dtype=torch.float32, device=q.device)
    call("mb_attn_bwd_packed", ptr(dout), ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(delta), ptr(dq_acc),
         ptr(delta) + 4 * nh * total, ptr(dq), ptr(gk), ptr(gv), ptr(packed.plan), packed.n, total, k.shape[0], nh, nkv, unit, d, q.stride(0), q.stride(1), k.stride(0),
         k.stride(1), v.stride(0), v.stride(1), dq.stride(0), dq.stride(1), gk.stride(0), gk.stride(1), gv.stride(0),
         gv.stride(1), scale, int(causal), stream())
    if parts > 1:
        call("mb_attn_sum_parts", ptr(gk), ptr(gv), ptr(dk), ptr(dv), 1, k.shape[0], nkv, parts, d, 0, dk.stride(0),
             dk.stride(1), 0, dv.stride(0), dv.stride(1), stream())
    return out


def check_kernel_types(*tensors):
    for t in tensors:
        if t.dtype != torch.bfloat16 or t.shape[-1] % 16 or not 16 <= t.shape[-1] <= 128:
            raise ValueError(f"the attention kernels take bf16 and head sizes of 16, 32, ... 128, not {t.dtype} of {t.shape[-1]}")


class _PackedSequencesAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, packed, scale, causal):
        o, lse = forward(q, k, v, packed, scale, causal)
        ctx.packed, ctx.scale, ctx.causal = packed, scale, causal
        ctx.save_for_backward(q, k, v, o, lse)
        return o

    @staticmethod
    def backward(ctx, dout):
        dq, dk, dv = backward(dout, *ctx.saved_tensors, ctx.packed, ctx.scale, ctx.causal)
        return dq, dk, dv, None, None, None


def attention(q, k, v, packed: PackedSequences, scale: float, causal: bool):
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2] or q.shape[1] % max(k.shape[1], 1):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    packed.check(q, k)
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v have to be on one device")
    if use_native(q):
        check_kernel_types(q, k, v)
        q, k, v = _rows(q), _rows(k), _rows(v)
    return _PackedSequencesAttnFn.apply(q, k, v, packed, float(scale), bool(causal))
