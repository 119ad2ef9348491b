"""Vocabulary projection and cross entropy as one operator, whose logits are never stored as numbers of their own.

``loss[t] = log sum_v exp(x_t . w_v + b_v) - (x_t . w_label + b_label)``.  The forward pass is one GEMM whose epilogue
keeps a maximum and a sum per row and tile.  The backward pass goes over the vocabulary piece by piece, gets the gradient
of a piece's logits and multiplies it into the gradients of ``x`` and of the weight.  It has the logits from the forward
pass, which keeps 16 bits of each while all that it keeps takes no more than ``Settings.xent_keep_bytes`` and the hidden
size makes it worth while, or computes them again.

So by default this operator saves no memory: 16 bits per logit are what the two separate steps hold too, whose gradient
overwrites their logits.  ``xent_keep_bytes = 0`` is the form that holds two numbers per row and one piece of the gradient.
Both passes of 8192 tokens of 2560, vocabulary 50304 (time; held between the passes; at most, the gradients included):
separate steps 5.4 ms, 786 MiB, 1072 MiB; logits kept 5.3 ms, 811, 1395; computed twice 6.4 ms, 0, 584.  What the first form
has over the separate steps is the loss of fp32 logits instead of bf16 ones (reference: the projection of
mist/modules/fused_dense.py:221-327 followed by mist/modules/losses.py:48-176, which hold ``[tokens, vocabulary]`` logits
between the two).
"""
from __future__ import annotations

import functools

import torch

from . import functional as F
from . import native
from .native import INT32_MAX, call, ptr, stream, use_native

# Hidden sizes from which a logit is kept and not computed again.  Both passes, vocabulary 50304 (kept, twice, us): 4096 tokens of
# 4096 3952, 5145; of 2048 2197, 2574; of 1024 1250, 1474; of 512 766, 875; 256 tokens of 4096 482, 571; of 1024 294, 309; of 512
# 266, 270; 16384 of 1024 5033, 5758; of 512 3377, 3775.  Vocabulary 8192: 4096 tokens of 1024 209, 234; of 512 159, 163; up to 1024
# tokens of 2048 the host decides (140, 136).  Below 1024 a tenth of the time is not worth memory of 16 bits per logit.
KEEP_FROM = 1024


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """``t`` as ``[rows, cols]`` that the kernels' copies can address: unit stride, rows on 16 bytes."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if t.stride(1) != 1 or t.stride(0) % 8 or not cols <= t.stride(0) <= INT32_MAX or ptr(t) % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def piece_columns(rows: int, vocab: int) -> int:
    """Columns of the vocabulary whose gradient the backward pass holds at a time: as many multiples of 256 as
    ``Settings.xent_piece_bytes`` allows, in pieces of equal size."""
    most = max(256, F.Settings.xent_piece_bytes // (2 * max(rows, 1)) // 256 * 256)
    pieces = -(-vocab // most)
    return min(vocab, -(-(-(-vocab // pieces)) // 256) * 256)


def kept_bytes(rows: int, vocab: int) -> int:
    """Bytes that live from the forward to the backward pass where logits are kept: of each row 16 bits per logit, a maximum
    and a sum per 128 columns, the label's logit, the loss and the log-sum-exp."""
    return rows * (2 * (-(-vocab // 8) * 8) + 16 * -(-vocab // 256) + 12)


def keeps_logits(rows: int, vocab: int, k: int) -> bool:
    """Whether the forward pass keeps 16 bits of every logit for the backward pass instead of computing the logits twice."""
    return k >= KEEP_FROM and rows <= 2 ** 20 and kept_bytes(rows, vocab) <= F.Settings.xent_keep_bytes


@functools.lru_cache(maxsize=1024)
def _backward_bytes(*sizes):
    """Workspace of the backward pass: a function of the sizes alone."""
    return native.kernels().mb_xent_linear_bwd_workspace(*sizes)


def _combine_over_group(stats, labels, ignore_index, group):
    """Per-row loss and log-sum-exp from ``{maximum, sum, label's logit}`` of every slice of the vocabulary."""
    top = stats[:, 0].clone()
    torch.distributed.all_reduce(top, op=torch.distributed.ReduceOp.MAX, group=group)
    rest = stats[:, 1:].clone()
    rest[:, 0] *= torch.exp(stats[:, 0] - top)
    torch.distributed.all_reduce(rest, group=group)
    lse = rest[:, 0].log() + top
    return torch.where(labels == ignore_index, torch.zeros_like(lse), lse - rest[:, 1]), lse


class _LinearXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, labels, v0, group, ignore_index, backward):
        ctx.v0, ctx.ignore, ctx.x_shape = v0, ignore_index, x.shape
        ctx.param = F._bucket_owner(weight)
        vocab, k = weight.shape
        x2, w2 = _rows(x, k), weight
        rows = x2.shape[0]
        split = group is not None and torch.distributed.get_world_size(group) > 1
        kept = None, None
        if not use_native(x2):
            logits = x2.float() @ weight.float().t()
            if bias is not None:
                logits += bias.float()
            at = labels - v0
            inside = (at >= 0) & (at < vocab)
            top = logits.max(-1).values
            target = torch.where(inside, logits.gather(1, at.clamp(0, vocab - 1)[:, None])[:, 0], torch.zeros_like(top))
            # (a slice that is all -inf adds nothing: the others may have more)
            total = torch.exp(logits - top.masked_fill(top == float("-inf"), 0.0)[:, None]).sum(-1)
            if split:
                loss, lse = _combine_over_group(torch.stack([top, total, target], 1), labels, ignore_index, group)
            else:
                lse = total.log() + top
                loss = torch.where(labels == ignore_index, torch.zeros_like(lse), lse - target)
        else:
            w2 = _rows(weight, k)
            tiles = native.kernels().mb_xent_linear_tiles(vocab)
            keeps = backward and keeps_logits(rows, vocab, k)
            # [tile, or half of one][row] statistics, labels' logits, and per row: loss and lse, or what the group combines
            entries = tiles * (2 if keeps else 1)
            work = torch.empty((2 * entries + 1) * rows, dtype=torch.float32, device=x.device)
            out = torch.empty(3 if split else 2, rows, dtype=torch.float32, device=x.device)
            loss, lse = out[0], out[1]
            if keeps:
                wide = -(-vocab // 8) * 8
                kept = torch.empty(rows, wide, dtype=torch.int16, device=x.device), work
            call("mb_xent_linear_fwd", ptr(x2), ptr(w2), ptr(bias), ptr(labels), ptr(work), ptr(work) + 8 * entries * rows,
                 ptr(loss), ptr(lse), ptr(out) if split else 0, ptr(kept[0]), wide if keeps else 0, rows, vocab, k, x2.stride(0),
                 w2.stride(0), v0, ignore_index, F.Settings.gemm_max_ctas, stream())
            if split:
                loss, lse = _combine_over_group(out.view(rows, 3), labels, ignore_index, group)
        ctx.save_for_backward(x2, weight, bias, labels, lse, *kept)
        return loss

    @staticmethod
    def backward(ctx, gloss):
        x2, weight, bias, labels, lse, kept, stats = ctx.saved_tensors
        rows, k = x2.shape
        vocab = weight.shape[0]
        want_x, want_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        want_b = bias is not None and ctx.needs_input_grad[2]
        bucket = getattr(ctx.param, "grad_bucket", None) if want_w else None
        accumulate = bucket is not None and bool(getattr(ctx.param, "grad_accumulate", False))
        direct = bucket is not None and bucket.dtype in (torch.float32, weight.dtype) and bucket.stride(1) == 1
        if direct and use_native(x2):      # what the products' stores can address
            direct = bucket.stride(0) % 8 == 0 and k <= bucket.stride(0) <= INT32_MAX and ptr(bucket) % 16 == 0
        dw = None
        if direct:
            dw = bucket
        elif want_w:
            dw = torch.empty(vocab, k, dtype=weight.dtype if bucket is None else torch.float32, device=x2.device)
        dx = torch.empty(rows, k, dtype=x2.dtype, device=x2.device) if want_x else None
        db = torch.empty(vocab, dtype=bias.dtype, device=x2.device) if want_b else None
        add = direct and accumulate
        gloss = gloss.float().contiguous()
        if rows == 0:
            for t in (db, None if add else dw):
                if t is not None:
                    t.zero_()
        elif use_native(x2):
            w2, piece, ctas = _rows(weight, k), piece_columns(rows, vocab), F.Settings.gemm_max_ctas
            fp32 = int(dw is not None and dw.dtype == torch.float32)
            area = _backward_bytes(rows, vocab, k, piece, want_x, want_w, want_b, fp32, add, ctas)
            workspace = torch.empty(area, dtype=torch.uint8, device=x2.device)
            wide, target = (0, 0) if kept is None else (kept.shape[1], ptr(stats) + 4 * (stats.numel() - rows))
            call("mb_xent_linear_bwd", ptr(x2), ptr(w2), ptr(bias), ptr(labels), ptr(lse), ptr(gloss), ptr(dx), ptr(dw),
                 ptr(db), ptr(kept), wide, ptr(stats), target, rows, vocab, k, x2.stride(0), w2.stride(0), 0 if dw is None else dw.stride(0), fp32, add, 0, ctx.v0, ctx.ignore,
                 piece, ctas, ptr(workspace), stream())
        else:
            _reference_backward(x2, weight, bias, labels, lse, gloss, ctx.v0, ctx.ignore, dx, dw, add, db)
        if bucket is not None:
            if not direct:
                bucket.add_(dw) if accumulate else bucket.copy_(dw)      # any type and order
            ctx.param.grad_accumulate = True
        if dx is not None and dx.shape != ctx.x_shape:
            dx = dx.reshape(ctx.x_shape)
        return (dx, dw if bucket is None else None, db, None, None, None, None, None)


def _reference_backward(x2, weight, bias, labels, lse, gloss, v0, ignore, dx, dw, accumulate, db):
    logits = x2.float() @ weight.float().t()
    if bias is not None:
        logits += bias.float()
    p = torch.exp(logits - lse[:, None])
    at = labels - v0
    inside = (at >= 0) & (at < weight.shape[0])
    p[inside, at[inside]] -= 1.0
    p = torch.where((labels == ignore)[:, None], torch.zeros_like(p), p * gloss[:, None])
    if dw is not None:
        g = p.t() @ x2.float()
        dw.add_(g.to(dw.dtype)) if accumulate else dw.copy_(g)
    if db is not None:
        db.copy_(p.sum(0))
    if dx is not None:
        dx.copy_(p @ weight.float())


def linear_cross_entropy(x, weight, labels, bias=None, vocab_start: int = 0, group=None, ignore_index: int = -100):
    """Loss (fp32) of every row of ``x`` ``[..., hidden]`` against ``labels`` ``[...]``: the cross entropy of the logits
    ``x @ weight.T + bias``, which are computed in fp32 and never stored as such.  For the backward pass 16 bits of each are
    kept while all that is kept takes no more than ``Settings.xent_keep_bytes`` (2 GiB; 0: never); otherwise it computes them
    again.  Rows labelled
    ``ignore_index`` have loss 0 and give no gradient.  A label outside the vocabulary counts as one whose logit is 0; no one checks for it.

    ``weight`` ``[vocab, hidden]`` (and ``bias`` ``[vocab]``) may be this rank's slice of the vocabulary, starting at
    ``vocab_start``; ``group`` is then the group of the slices, and ``x`` is the same on every rank of it (its gradient is
    this slice's share).  The weight's gradient goes into its bucket where it has one."""
    if F._sym(x):
        return F._rules().linear_cross_entropy(x, weight, labels, bias)
    if F._elsewhere(x):
        with torch.cuda.device(x.device):
            return linear_cross_entropy(x, weight, labels, bias, vocab_start, group, ignore_index)
    if weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.shape[0] == 0:
        raise ValueError(f"x {tuple(x.shape)} does not fit a weight {tuple(weight.shape)}")
    if labels.shape != x.shape[:-1] or labels.is_floating_point():
        raise ValueError(f"labels: integers of shape {tuple(x.shape[:-1])} expected, got {tuple(labels.shape)} of {labels.dtype}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias {tuple(bias.shape)} does not fit a weight {tuple(weight.shape)}")
    for t in (weight, labels, bias):
        if t is not None and t.device != x.device:
            raise ValueError("x, weight, labels and bias have to be on one device")
    if use_native(x):
        if max(labels.numel(), *weight.shape) > INT32_MAX:
            raise ValueError(f"{labels.numel()} rows, weight {tuple(weight.shape)}: the kernels count them in 32 bits")
        if any(t is not None and t.dtype != torch.bfloat16 for t in (x, weight, bias)) or x.shape[-1] % 8:
            raise ValueError("the kernels take bf16 of a hidden size that is a multiple of 8")
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
    flat = labels if labels.dim() == 1 else labels.reshape(-1)
    loss = _LinearXentFn.apply(x, weight, bias, flat.long().contiguous(), int(vocab_start), group, int(ignore_index),
                               torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)))
    return loss if labels.dim() == 1 else loss.reshape(labels.shape)
