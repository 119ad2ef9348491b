"""Sequences packed back to back in one row of tokens, and attention inside each of them.

A :class:`PackedSequences` is made once per batch.  It holds the offsets, every token's position in its sequence, and the
work lists that the attention kernels walk (csrc/packed_plan.cu); all layers, forward and backward, use the same one, and
nothing is read back to the host, but by ``attention_varlen`` with bare offsets on the GPU (reference:
csrc/flash_attn/flash_api.cpp:427, 814 ``varlen_fwd`` / ``varlen_bwd``, called with offsets that mist/modules/mha.py:1233-1243
derives from a padding mask)."""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import native
from .native import INT32_MAX, call, ptr, stream, use_native


# what the library says of sizes alone
@functools.lru_cache(maxsize=1024)
def _plan_bytes(n, total_q, total_k):
    return native.kernels().mb_packed_plan_bytes(n, total_q, total_k)


@functools.lru_cache(maxsize=1024)
def _counters(n, total_q, heads):
    return native.kernels().mb_attn_fwd_packed_counters(n, total_q, heads)


@functools.lru_cache(maxsize=1024)
def _backward_sizes(total_q, total_k, nh, nkv, d):
    """Query heads of a group that a CTA sums, bytes of workspace."""
    from .attention_bwd import unit_heads
    unit = unit_heads(nh // nkv, total_k, nh)
    return unit, native.kernels().mb_attn_bwd_packed_workspace(total_q, total_k, nh, nkv, unit, d)


def _offsets(cu, device):
    """Offsets as int32 on the device, and as a list where they are known on the host (then checked)."""
    if isinstance(cu, torch.Tensor):
        if cu.dim() != 1 or cu.numel() < 1 or cu.is_floating_point():
            raise ValueError(f"offsets: a vector of integers expected, got {tuple(cu.shape)} of {cu.dtype}")
        if cu.is_cuda and device.type == "cuda":
            if cu.dtype != torch.int32 or cu.device != device or not cu.is_contiguous():
                cu = cu.to(device=device, dtype=torch.int32).contiguous()
            return cu, None
    host = [int(x) for x in (cu.tolist() if isinstance(cu, torch.Tensor) else cu)]
    _check_offsets(host)
    if host[-1] > INT32_MAX:
        raise ValueError(f"offsets up to {host[-1]}: 32 bits hold them")
    if device.type == "cuda":      # they go there as arguments of a kernel: nothing waits, and a captured graph holds them
        return torch.empty(len(host), dtype=torch.int32, device=device), host
    return torch.tensor(host, dtype=torch.int32), host


def _check_offsets(host):
    if not host or host[0] != 0 or any(b < a for a, b in zip(host, host[1:])):
        raise ValueError("offsets: they begin with 0 and do not fall")


_streams = {}


def _current_stream(index: int):
    """The current stream of a device as an object; one for each raw handle is kept, because making it takes 3 us."""
    handle = torch._C._cuda_getCurrentRawStream(index)
    stream = _streams.get((index, handle))
    if stream is None:
        stream = _streams[index, handle] = torch.cuda.current_stream(index)
    return stream


_events = {}      # of each device: those of packings that are gone (making and destroying one takes 5 us)


class _Made:
    """Tensors that were made on the stream that was current then.  Others wait for that once, where they first use them; the
    allocator learns of them.  Tensors of a graph being captured belong to it: nobody outside waits for them."""

    def __init__(self, device, *tensors):
        self.index, self.tensors, self.event = device.index, tensors, None
        self.seen = {torch._C._cuda_getCurrentRawStream(device.index)}
        if not torch.cuda.is_current_stream_capturing():
            free = _events.setdefault(device.index, [])
            self.event = free.pop() if free else torch.cuda.Event()
            self.event.record(_current_stream(device.index))

    def __del__(self):
        if self.event is not None and _events is not None:      # (nothing is left of the module when the process ends)
            _events[self.index].append(self.event)

    def here(self):
        now = torch._C._cuda_getCurrentRawStream(self.index)
        # (an event of outside cannot be waited for under capture; a graph is replayed after its capture, which itself begins
        # when the device is idle)
        if now in self.seen or self.event is None or torch.cuda.is_current_stream_capturing():
            return
        current = _current_stream(self.index)
        current.wait_event(self.event)
        for t in self.tensors:
            t.record_stream(current)
        self.seen.add(now)


class PackedSequences:
    """``n`` sequences packed back to back: ``cu_seqlens`` holds the ``n + 1`` offsets (0 first), as a tensor or a list.

    ``total``: rows of the packed tensors, at least the last offset; rows behind it belong to no sequence.  It may be left
    out where the offsets are known on the host.  ``cu_seqlens_k`` / ``total_k``: offsets of the keys, where they are others
    than those of the queries.  Offsets on the GPU are not read back and not checked: ones that fall or pass ``total`` are
    clamped, which keeps every access inside the tensors, and what comes out is unspecified.  The object may be used on any
    stream: its tensors are made on one and waited for on others (under capture they have to be there, as after
    ``torch.cuda.graph`` has begun)."""

    def __init__(self, cu_seqlens, total: Optional[int] = None, cu_seqlens_k=None, total_k: Optional[int] = None, device=None):
        self._set_up(cu_seqlens, total, cu_seqlens_k, total_k, device)
        if self.plan is not None:
            self._made = _Made(self.device, self.cu_q, self.cu_k, self.plan)

    def _set_up(self, cu_seqlens, total, cu_seqlens_k, total_k, device, ends=0):
        if device is None and isinstance(cu_seqlens, torch.Tensor):
            device = cu_seqlens.device
        else:
            device = torch.device("cpu" if device is None else device)
            if device.type == "cuda" and device.index is None:
                device = torch.device("cuda", torch.cuda.current_device())
        self.same = cu_seqlens_k is None
        self.cu_q, self.host_q = _offsets(cu_seqlens, device)
        self.cu_k, self.host_k = (self.cu_q, self.host_q) if self.same else _offsets(cu_seqlens_k, device)
        if self.cu_k.numel() != self.cu_q.numel():
            raise ValueError("as many sequences of keys as of queries expected")
        self.n = self.cu_q.numel() - 1
        self.total_q = self._total(total, self.host_q)
        self.total_k = self.total_q if self.same and total_k is None else self._total(total_k, self.host_k)
        self.device = device
        self._rotary = {}
        self._positions = self.plan = self._made = None
        if use_native(self.cu_q):
            size = _plan_bytes(self.n, self.total_q, self.total_k)
            if torch.is_inference_mode_enabled():      # autograd keeps none that were made under it
                with torch.inference_mode(False):
                    self.plan = torch.empty(size, dtype=torch.uint8, device=device)
            else:
                self.plan = torch.empty(size, dtype=torch.uint8, device=device)
            if device.index == torch._C._cuda_getDevice():
                self._make_plan(ends)
            else:
                with torch.cuda.device(device):
                    self._make_plan(ends)

    def _make_plan(self, ends):
        def ints(host):
            return None if host is None else (ctypes.c_int * len(host))(*host)

        call("mb_packed_plan", ptr(self.cu_q), ptr(self.cu_k), ints(self.host_q), None if self.same else ints(self.host_k),
             self.n, self.total_q, self.total_k, ptr(self.plan), ends, stream())

    def here(self):
        """The plan and the offsets, for kernels of the current stream."""
        if self._made is not None:
            self._made.here()

    @property
    def positions(self):
        """Every query row's place in its sequence, int64 ``[total]``."""
        self.here()
        if self._positions is None:
            with torch.inference_mode(False):
                if self.plan is not None:
                    at = native.kernels().mb_packed_plan_positions(self.n, self.total_q, self.total_k)
                    self._positions = self.plan[at:at + 8 * self.total_q].view(torch.int64)
                else:
                    rows = torch.arange(self.total_q)
                    self._positions = rows - self.cu_q.long()[torch.searchsorted(self.cu_q, rows, right=True) - 1]
        return self._positions

    def limit_lengths(self, most: int):
        """Refuses sequences of queries longer than ``most``: here where the offsets are known on the host, else by a status
        that :func:`~mist_b200.ops.native.check_status` raises.  Rows behind the last sequence do not count."""
        host = self.host_q
        if host is None and self.plan is None:
            host = self.cu_q.tolist()
        if host is not None:
            longest = max((b - a for a, b in zip(host, host[1:])), default=0)
            if longest > most:
                raise ValueError(f"a sequence of {longest} tokens, but the table of positions has {most}")
        else:
            self.here()
            with torch.cuda.device(self.device):
                call("mb_packed_limit", ptr(self.cu_q), self.n, self.total_q, most, stream())

    @staticmethod
    def _total(total, host):
        if total is None:
            if host is None:
                raise ValueError("offsets on the GPU need the number of packed rows beside them")
            total = host[-1]
        if total < 0 or (host is not None and host[-1] > total):
            raise ValueError(f"{total} rows, but the offsets end at {host and host[-1]}")
        if total > INT32_MAX:
            raise ValueError(f"{total} rows: 32 bits hold their number")
        return int(total)

    def check(self, q, k):
        if q.shape[0] != self.total_q or k.shape[0] != self.total_k:
            raise ValueError(f"{q.shape[0]} query and {k.shape[0]} key rows, but the packing is of {self.total_q} and {self.total_k}")
        if q.device != self.device:
            raise ValueError(f"tensors on {q.device}, offsets on {self.device}")
        self.here()

    def rotary(self, rot_dim: int, base: float):
        """``(cos, sin, rot_dim)`` with a row for each packed token, that of its position; made on the stream of the first call,
        kept, and waited for on others, or made for the graph alone while one is captured."""
        key = (rot_dim, base)
        tables, made = self._rotary.get(key, (None, None))
        if made is not None:
            made.here()
        if tables is None:
            # the angles of functional.rope_tables; what it keeps is by length, and packings come in every length
            with torch.inference_mode(False):
                inv = 1.0 / (base ** (torch.arange(0, rot_dim, 2, dtype=torch.float32, device=self.device) / rot_dim))
                angles = torch.outer(self.positions.float(), inv)
                tables = (angles.cos(), angles.sin(), rot_dim)
            # (tables that a graph being captured computes belong to it: outside it nobody has computed them)
            if self.plan is None or not torch.cuda.is_current_stream_capturing():
                self._rotary[key] = tables, None if self.plan is None else _Made(self.device, *tables[:2])
        return tables

    def _each(self):
        """``(queries, keys)`` slices of every sequence (reference path: reads the offsets)."""
        q, k = self.host_q or self.cu_q.tolist(), self.host_k or self.cu_k.tolist()
        return [(slice(q[i], q[i + 1]), slice(k[i], k[i + 1])) for i in range(self.n)]


_ends = {}      # of each device: pinned numbers and events of calls that are over


class PackedCall(PackedSequences):
    """The packing of one call on one stream: nobody else waits for it, and the ends of its offsets come to the host."""

    def __init__(self, cu_q, total_q, cu_k, total_k, device):
        self._reads, self._index = None, device.index
        if (device.type == "cuda" and any(isinstance(cu, torch.Tensor) and cu.is_cuda for cu in (cu_q, cu_k))
                and not torch.cuda.is_current_stream_capturing()):
            free = _ends.setdefault(device.index, [])
            self._reads = free.pop() if free else (torch.empty(2, dtype=torch.int32, pin_memory=True), torch.cuda.Event())
        self._set_up(cu_q, total_q, cu_k, total_k, device, 0 if self._reads is None else ptr(self._reads[0]))
        if self._reads is not None:
            self._reads[1].record(_current_stream(device.index))

    def __del__(self):
        """A call that raised: its plan may still be about to write the numbers."""
        if self._reads is not None:
            self._reads[1].synchronize()
            _ends[self._index].append(self._reads)

    def end(self):
        """Where the queries' last sequence ends, or ``None`` where that is only known on the GPU and a graph is being captured.
        Impossible offsets raise; waits for the plan, but not for what was launched behind it."""
        if self._reads is None:
            return None if self.host_q is None else self.host_q[-1]
        pinned, event = self._reads
        event.synchronize()
        ends = pinned.tolist()
        _ends[self._index].append(self._reads)
        self._reads = None
        if min(ends) < 0:
            raise ValueError("offsets: they begin with 0, do not fall, and end within the tensors")
        return ends[0]


def _rows(t):
    """``t`` ``[rows, heads, d]`` as the kernels' copies can address it."""
    rows, heads, inner = t.stride()
    if inner != 1 or rows % 8 or heads % 8 or ptr(t) % 16 or (rows == 0 and t.shape[0] > 1) or (heads == 0 and t.shape[1] > 1):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _reference_forward(q, k, v, packed, scale, causal):
    from .functional import _ref_attention
    o = torch.zeros(q.shape, dtype=q.dtype)
    lse = torch.full((q.shape[1], q.shape[0]), float("-inf"), dtype=torch.float32)
    for a, b in packed._each():
        if a.stop > a.start and b.stop > b.start:
            oi, li = _ref_attention(q[None, a], k[None, b], v[None, b], scale, causal)
            o[a], lse[:, a] = oi[0], li[0]
    return o, lse


def _reference_backward(dout, q, k, v, packed, scale, causal, out):
    from .attention_bwd import _reference
    for t in out:
        t.zero_()
    for a, b in packed._each():
        if a.stop > a.start and b.stop > b.start:
            grads = _reference(dout[None, a], q[None, a], k[None, b], v[None, b], scale, causal)
            for t, at, g in zip(out, (a, b, b), grads):
                t[at] = g[0]


def _launch_forward(tensors, strides, o, heads, packed, scale, causal):
    """``tensors``: addresses of q, k, v; ``strides``: of their rows and heads.  Returns lse, ``[heads, total]`` and one more
    number behind (the count of claimed work items)."""
    nh, nkv, d = heads
    total = packed.total_q
    lse = torch.empty(nh * total + 1, dtype=torch.float32, device=o.device)
    claimed = ptr(lse) + 4 * nh * total if _counters(packed.n, total, nh) else 0
    call("mb_attn_fwd_packed", *tensors, ptr(o), ptr(lse), ptr(packed.plan), claimed, packed.n, total, packed.total_k, nh, nkv,
         d, *strides, nh * d, d, scale, int(causal), stream())
    return lse


def _launch_backward(dout, tensors, strides, o, lse, grads, grad_strides, heads, packed, scale, causal):
    nh, nkv, d = heads
    dout = dout.contiguous()
    if ptr(dout) % 16:
        dout = dout.clone()
    unit, size = _backward_sizes(packed.total_q, packed.total_k, nh, nkv, d)
    workspace = torch.empty(size, dtype=torch.uint8, device=o.device)
    call("mb_attn_bwd_packed", ptr(dout), *tensors, ptr(o), ptr(lse), *grads, ptr(packed.plan), ptr(workspace), packed.n,
         packed.total_q, packed.total_k, nh, nkv, unit, d, *strides, *grad_strides, scale, int(causal), stream())


def check_kernel_types(*tensors):
    for t in tensors:
        if t.dtype != torch.bfloat16 or t.shape[-1] % 16 or not 16 <= t.shape[-1] <= 128:
            raise ValueError(f"the attention kernels take bf16 and head sizes of 16, 32, ... 128, not {t.dtype} of {t.shape[-1]}")


def _forward(q, k, v, packed, scale, causal):
    if not use_native(q):
        return _reference_forward(q, k, v, packed, scale, causal)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = _launch_forward((ptr(q), ptr(k), ptr(v)), (*q.stride()[:2], *k.stride()[:2], *v.stride()[:2]), o,
                          (q.shape[1], k.shape[1], q.shape[2]), packed, scale, causal)
    return o, lse


class _PackedSequencesAttnFn(torch.autograd.Function):
    """q ``[total_q, heads, d]``, k and v ``[total_k, kv heads, d]``."""

    @staticmethod
    def forward(ctx, q, k, v, packed, scale, causal):
        ctx.packed, ctx.scale, ctx.causal = packed, scale, causal
        o, lse = _forward(q, k, v, packed, scale, causal)
        ctx.save_for_backward(q, k, v, o, lse)
        return o

    @staticmethod
    def backward(ctx, dout):
        q, k, v, o, lse = ctx.saved_tensors
        out = tuple(torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        if use_native(q):
            _launch_backward(dout, (ptr(q), ptr(k), ptr(v)), (*q.stride()[:2], *k.stride()[:2], *v.stride()[:2]), o, lse,
                             tuple(ptr(t) for t in out), tuple(x for t in out for x in t.stride()[:2]),
                             (q.shape[1], k.shape[1], q.shape[2]), ctx.packed, ctx.scale, ctx.causal)
        else:
            _reference_backward(dout, q, k, v, ctx.packed, ctx.scale, ctx.causal, out)
        return (*out, None, None, None)


class _ProjectedAttnFn(torch.autograd.Function):
    """Rotary embedding and self attention on a projection output ``[b, s, q heads + 2 * kv heads, d]`` of packed sequences,
    whose gradient is one tensor.  On the device the projection output is rotated in place."""

    @staticmethod
    def forward(ctx, qkv, cos, sin, rot, packed, kv_heads, scale, causal):
        from .functional import _PackedAttnFn
        b, s, n, d = qkv.shape
        if rot:
            qkv = _PackedAttnFn._rotate(qkv.view(1, b * s, n, d), cos, sin, rot, False, kv_heads)
        ctx.args = rot, packed, kv_heads, scale, causal
        ctx.shape = b, s, n, d
        if use_native(qkv):
            o = torch.empty(b, s, n - 2 * kv_heads, d, dtype=qkv.dtype, device=qkv.device)
            lse = _launch_forward(_ProjectedAttnFn._parts(ptr(qkv), n, kv_heads, d), (n * d, d) * 3, o,
                                  (n - 2 * kv_heads, kv_heads, d), packed, scale, causal)
        else:
            o, lse = _reference_forward(*_ProjectedAttnFn._split(qkv.view(b * s, n, d), kv_heads), packed, scale, causal)
            o = o.view(b, s, n - 2 * kv_heads, d)
        ctx.save_for_backward(qkv, o, lse, cos, sin)
        return o

    @staticmethod
    def _parts(at, n, kv_heads, d):
        """Addresses of the q, the k and the v heads of the first token."""
        return at, at + 2 * d * (n - 2 * kv_heads), at + 2 * d * (n - kv_heads)

    @staticmethod
    def _split(t, kv_heads):
        n = t.shape[1]
        return t[:, :n - 2 * kv_heads], t[:, n - 2 * kv_heads:n - kv_heads], t[:, n - kv_heads:]

    @staticmethod
    def backward(ctx, dout):
        from .functional import _PackedAttnFn
        qkv, o, lse, cos, sin = ctx.saved_tensors
        rot, packed, kv_heads, scale, causal = ctx.args
        b, s, n, d = ctx.shape
        dqkv = torch.empty(ctx.shape, dtype=qkv.dtype, device=qkv.device)
        if use_native(qkv):
            strides = (n * d, d) * 3
            _launch_backward(dout, _ProjectedAttnFn._parts(ptr(qkv), n, kv_heads, d), strides, o, lse,
                             _ProjectedAttnFn._parts(ptr(dqkv), n, kv_heads, d), strides, (n - 2 * kv_heads, kv_heads, d),
                             packed, scale, causal)
        else:
            _reference_backward(dout.reshape(b * s, -1, d), *_ProjectedAttnFn._split(qkv.view(b * s, n, d), kv_heads), packed,
                                scale, causal, _ProjectedAttnFn._split(dqkv.view(b * s, n, d), kv_heads))
        if rot:
            dqkv = _PackedAttnFn._rotate(dqkv.view(1, b * s, n, d), cos, sin, rot, True, kv_heads).view(ctx.shape)
        return dqkv, None, None, None, None, None, None, None


def attention(q, k, v, packed: PackedSequences, scale: float, causal: bool):
    """Attention of ``q`` ``[total_q, heads, d]`` over ``k``, ``v`` ``[total_k, kv heads, d]`` inside each sequence."""
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2] or q.shape[1] % max(k.shape[1], 1):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    packed.check(q, k)
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v have to be on one device")
    if use_native(q):
        check_kernel_types(q, k, v)
        q, k, v = _rows(q), _rows(k), _rows(v)
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)):
        return _forward(q, k, v, packed, float(scale), bool(causal))[0]
    return _PackedSequencesAttnFn.apply(q, k, v, packed, float(scale), bool(causal))


def projected_attention(qkv, kv_heads: int, packed: PackedSequences, scale: float, causal: bool, rotary):
    """Self attention on a projection output ``[b, s, q heads + 2 * kv heads, d]`` or ``[b, s, 3, kv heads, d]``."""
    cos, sin, rot = rotary if rotary is not None else (None, None, 0)
    if qkv.dim() == 5:
        qkv = qkv.flatten(2, 3)
    if qkv.dim() != 4 or kv_heads < 1 or qkv.shape[2] <= 2 * kv_heads or (qkv.shape[2] - 2 * kv_heads) % kv_heads or not packed.same:
        raise ValueError(f"{tuple(qkv.shape)} with {kv_heads} key heads: self attention over one packing expected")
    if qkv.shape[0] * qkv.shape[1] != packed.total_q or packed.total_k != packed.total_q:
        raise ValueError(f"{tuple(qkv.shape[:2])} tokens, but the packing is of {packed.total_q}")
    if qkv.device != packed.device:
        raise ValueError(f"tensors on {qkv.device}, offsets on {packed.device}")
    packed.here()
    if rot:
        for t in (cos, sin):
            if t.shape != (packed.total_q, rot // 2) or t.dtype != torch.float32 or not t.is_contiguous() or t.device != qkv.device:
                raise ValueError(f"rotary tables: fp32 {(packed.total_q, rot // 2)} on {qkv.device} expected, a row for every token")
        if rot % 2 or rot > qkv.shape[3]:
            raise ValueError(f"{rot} rotated values of heads of {qkv.shape[3]}")
    if use_native(qkv):
        check_kernel_types(qkv)
        if not qkv.is_contiguous() or ptr(qkv) % 16:
            if rot:
                raise ValueError("the rotation in place needs a contiguous projection output")
            qkv = qkv.clone(memory_format=torch.contiguous_format)
    elif not qkv.is_contiguous():
        qkv = qkv.contiguous()
    return _ProjectedAttnFn.apply(qkv, cos, sin, int(rot), packed, int(kv_heads), float(scale), bool(causal))
