"""Distillation from a teacher's top log probabilities, forward and backward.

``topk_distillation_loss(logits, teacher_ids, teacher_logprobs)`` is
KL(teacher || student) where the teacher is known by its k best entries per
position, as ``logprobs.token_logprobs(teacher_logits, top_k=k,
temperature=t)`` returns them. It stands beside ``fused_linear_cross_entropy``,
the loss against labels. The loss and the gradient of the logits come from one
kernel (``dwarf_topk_distill`` in the C ABI).

Where the loss is reduced (``"mean"``, ``"sum"``) and the logits require grad,
the forward launch writes the gradient for an upstream gradient of 1 in the same
pass over the logits; backward's launch leaves it as it is when the upstream
gradient is 1, and otherwise computes it anew from the logits and the sums that the
forward launch has left (one rounding either way). Where the two do not run alike (one
captured into a CUDA graph and the other not) backward always computes it.
``weight`` scales the loss without leaving the one-pass form.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib, _rows

__all__ = ["TopKDistillationLoss", "topk_distillation_loss"]


def _launch(logits, ids, logprobs, mask, inv_temperature, tail, *, loss=None, grad=None, stats=None, grad_scale=None,
            grad_rows=None, skip_if_one=False, loss_scale=1.0, scale=1.0) -> None:
    logits, outer, inner, so, si = _rows.addressed(logits)
    args = _lib.TopkDistillArgs(
        version=_lib.ABI_VERSION, dtype=_lib.dtype_code(logits.dtype), logits=logits.data_ptr(), outer=outer,
        inner=inner, vocab=logits.shape[-1], so=so, si=si, teacher_ids=ids.data_ptr(),
        teacher_logprobs=logprobs.data_ptr(), k=ids.shape[-1], tail=int(tail), row_mask=_lib.ptr(mask),
        inv_temperature=inv_temperature, grad_rows_stride=int(grad_rows is not None and grad_rows.ndim > 0),
        grad_scale=_lib.ptr(grad_scale), grad_rows=_lib.ptr(grad_rows), loss=_lib.ptr(loss), grad=_lib.ptr(grad),
        stats=_lib.ptr(stats), skip_if_one=int(skip_if_one), loss_scale=loss_scale, scale=scale)
    if outer * inner:
        _rows.launch("dwarf_topk_distill", args, logits.device)


def _reduce(out, *, values=None, mask=None, host_scale=1.0) -> None:
    rows = (values if values is not None else mask).numel()
    args = _lib.RowReduceArgs(version=_lib.ABI_VERSION, rows=rows, values=_lib.ptr(values), mask=_lib.ptr(mask),
                              host_scale=host_scale, out=out.data_ptr())
    _rows.launch("dwarf_row_reduce", args, out.device)


class _TopKDistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, logprobs, mask, inv_temperature, tail, reduction, weight):
        stats = torch.empty(*logits.shape[:-1], 8, dtype=torch.float32, device=logits.device)
        ctx.save_for_backward(logits, ids, logprobs, mask, stats)
        ctx.scalars = (inv_temperature, tail)
        ctx.grad = None
        if reduction != "none":
            ctx.grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            ctx.capture = _lib.capture_id(logits.device)
        loss, ctx.scale, ctx.grad_scale = _forward(logits, ids, logprobs, mask, inv_temperature, tail, reduction,
                                                   weight, ctx.grad, stats)
        return loss

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():  # create_graph: a second derivative is refused, not left out
            return _once_more(ctx, g)
        logits, ids, logprobs, mask, stats = ctx.saved_tensors
        grad, ctx.grad = ctx.grad, None  # a second backward gets a buffer of its own
        # Where only one of forward and backward is captured, or each into a graph of its own, they are not
        # replayed in step, and what forward wrote is not this backward's to hand out.
        written = grad is not None and ctx.capture == _lib.capture_id(logits.device)
        if not written:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _launch(logits, ids, logprobs, mask, *ctx.scalars, grad=grad, stats=stats, grad_scale=ctx.grad_scale,
                grad_rows=_rows.in_memory(g).contiguous(), skip_if_one=written, scale=ctx.scale)
        return grad, None, None, None, None, None, None, None


_once_more = torch.autograd.function.once_differentiable(_TopKDistillationFn.backward)


def _forward(logits, ids, logprobs, mask, inv_temperature, tail, reduction, weight, grad=None, stats=None):
    """(loss, host and device factors of the gradient)."""
    dev = logits.device
    rows = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
    scale, grad_scale = weight, None
    if rows.numel() == 0:
        return rows if reduction == "none" else rows.new_zeros(()), scale, grad_scale
    if reduction == "mean":
        if mask is None:
            scale = weight / rows.numel()
        elif stats is not None:  # the gradient needs the number of rows before the loss is there
            grad_scale = torch.empty((), dtype=torch.float32, device=dev)
            _reduce(grad_scale, mask=mask)
    _launch(logits, ids, logprobs, mask, inv_temperature, tail, loss=rows, grad=grad, stats=stats, grad_scale=grad_scale,
            loss_scale=weight, scale=scale)
    if reduction == "none":
        return rows, scale, grad_scale
    loss = torch.empty((), dtype=torch.float32, device=dev)
    if reduction == "sum":
        _reduce(loss, values=rows)
    elif mask is None:
        _reduce(loss, values=rows, host_scale=1.0 / rows.numel())
    else:
        _reduce(loss, values=rows, mask=mask)
    return loss, scale, grad_scale


def topk_distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                           temperature: float = 1.0, tail: bool = True, row_mask: torch.Tensor | None = None,
                           reduction: str = "mean", weight: float = 1.0) -> torch.Tensor:
    """``weight`` * KL(teacher || softmax(logits / temperature)) over a teacher's listed entries.

    ``logits`` [..., V] float32, bfloat16 or float16 (``logits[:, :-1]`` is read in
    place); ``teacher_ids`` [..., k] int64 or int32 and ``teacher_logprobs`` [..., k]
    floating point, k in 1..128, the teacher's log probabilities at the same
    temperature (constants: no gradient flows to the teacher).

    * ``tail=True``: what the listed probabilities leave of 1 is one more event, the
      ids not listed, whose student probability is the sum over those ids.
      ``tail=False``: the listed values are normalised among themselves (any
      ``logits / temperature`` of the teacher will do; a list of -inf alone is NaN).
    * A slot with an id below 0 is not used; an id >= V makes its row NaN; an id
      listed twice counts with both probabilities.
    * ``row_mask`` [...] bool: rows where it is False, and rows without a used slot,
      have loss 0 and gradient exactly 0 whatever their logits hold. A NaN or +inf among
      another row's logits makes its loss and gradient NaN.
    * Where the student gives a listed id, or all the ids not listed, nothing (-inf) and the
      teacher gives them something, the loss is inf and the gradient finite: -p / temperature
      at such a listed id, 0 at the ids not listed. A counted row without a finite logit has
      loss inf and gradient 0.
    * ``reduction``: "mean" over the rows that ``row_mask`` keeps, "sum", or "none"
      ([...]). The loss is fp32; no factor temperature**2 is applied.

    The same call gives the same bits every time; a row's last bits may change with the number
    of rows beside it. Second and forward-mode derivatives and torch.func transforms are
    refused. Runs on the current stream, without synchronising.
    """
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    _rows.refuse_transforms(logits=logits, teacher_ids=teacher_ids, teacher_logprobs=teacher_logprobs,
                            row_mask=row_mask)
    logits = _rows.in_memory(logits)
    inv_temperature = _rows.check_logits(logits, temperature)
    weight = float(weight)
    if not math.isfinite(weight):
        raise ValueError(f"weight must be finite, got {weight}")
    k = teacher_ids.shape[-1] if teacher_ids.ndim else 0
    if not 1 <= k <= _rows.TOP_K_MAX:
        raise ValueError(f"the teacher must list 1..{_rows.TOP_K_MAX} entries, got {k}")
    shape = (*logits.shape[:-1], k)
    teacher_ids = _rows.ids64(teacher_ids, shape, "teacher_ids")
    if not teacher_logprobs.dtype.is_floating_point:
        raise TypeError(f"teacher_logprobs must be floating point, got {teacher_logprobs.dtype}")
    if tuple(teacher_logprobs.shape) != shape:
        raise ValueError(f"teacher_logprobs must be {shape}, got {tuple(teacher_logprobs.shape)}")
    grad = torch.is_grad_enabled()
    if grad and teacher_logprobs.requires_grad:
        raise NotImplementedError("no gradient flows to the teacher: pass teacher_logprobs.detach()")
    if row_mask is not None:
        if row_mask.dtype != torch.bool:
            raise TypeError(f"row_mask must be bool, got {row_mask.dtype}")
        if tuple(row_mask.shape) != shape[:-1]:
            raise ValueError(f"row_mask must be {shape[:-1]}, got {tuple(row_mask.shape)}")
        row_mask = row_mask.contiguous()
    _rows.same_device(logits, teacher_ids=teacher_ids, teacher_logprobs=teacher_logprobs, row_mask=row_mask)
    teacher_logprobs = _rows.in_memory(teacher_logprobs).to(torch.float32).contiguous()
    if grad and logits.requires_grad:
        return _TopKDistillationFn.apply(logits, teacher_ids, teacher_logprobs, row_mask, inv_temperature, bool(tail),
                                         reduction, weight)
    return _forward(logits, teacher_ids, teacher_logprobs, row_mask, inv_temperature, bool(tail), reduction, weight)[0]


class TopKDistillationLoss(nn.Module):
    """``topk_distillation_loss`` with its options held: ``loss(logits, teacher_ids, teacher_logprobs, row_mask=None)``."""

    def __init__(self, temperature: float = 1.0, tail: bool = True, reduction: str = "mean",
                 weight: float = 1.0) -> None:
        super().__init__()
        self.temperature = float(temperature)
        self.tail = bool(tail)
        self.reduction = reduction
        self.weight = float(weight)

    def forward(self, logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logprobs: torch.Tensor,
                row_mask: torch.Tensor | None = None) -> torch.Tensor:
        return topk_distillation_loss(logits, teacher_ids, teacher_logprobs, temperature=self.temperature,
                                      tail=self.tail, row_mask=row_mask, reduction=self.reduction, weight=self.weight)
