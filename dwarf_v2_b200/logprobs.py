"""Log probabilities of given tokens, the entropy and the best alternatives of logit rows.

``token_logprobs(logits, targets, top_k=..., temperature=...)`` stands beside
``gemm.linear_lse`` (which reduces the lm_head's logits without writing them) for
logits that exist: a decoding step's (``DwarfForCausalLM.decode_step``,
``DecodeGraph.step``), a scoring pass's, a trainer's. It is differentiable: a
policy-gradient or entropy loss gets the gradient of the logits from one kernel
(``dwarf_token_logprobs`` / ``dwarf_token_logprobs_bwd`` in the C ABI). Its top
alternatives at a temperature are what ``distillation.topk_distillation_loss``
takes from a teacher.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, _rows

__all__ = ["TokenLogprobs", "token_logprobs"]


class TokenLogprobs(NamedTuple):
    """Outputs of ``token_logprobs``; [...] stands for the logits' leading dimensions."""

    logprob: torch.Tensor | None        # fp32 [...]: of the given tokens (None without targets)
    entropy: torch.Tensor               # fp32 [...]
    lse: torch.Tensor                   # fp32 [...]: logsumexp(logits / temperature)
    top_logprobs: torch.Tensor | None   # fp32 [..., top_k], falling (None with top_k=0)
    top_ids: torch.Tensor | None        # int64 [..., top_k]


def _forward(logits: torch.Tensor, targets: torch.Tensor | None, top_k: int, inv_temperature: float,
             ignore_index: int, want_stats: bool):
    dev, lead = logits.device, logits.shape[:-1]
    logits, outer, inner, so, si = _rows.addressed(logits)
    if targets is None:
        logprob, entropy = None, torch.empty(lead, dtype=torch.float32, device=dev)
    else:
        logprob = torch.empty_like(targets, dtype=torch.float32)
        entropy = torch.empty_like(logprob)
    lse = torch.empty_like(entropy)
    stats = torch.empty(*lead, 2, dtype=torch.float32, device=dev) if want_stats else None
    top_logprobs = top_ids = None
    if top_k:
        top_logprobs = torch.empty(*lead, top_k, dtype=torch.float32, device=dev)
        top_ids = torch.empty_like(top_logprobs, dtype=torch.int64)
    args = _lib.TokenLogprobsArgs(
        version=_lib.ABI_VERSION, dtype=_lib.dtype_code(logits.dtype), logits=logits.data_ptr(), outer=outer,
        inner=inner, vocab=logits.shape[-1], so=so, si=si, targets=_lib.ptr(targets), ignore_index=ignore_index,
        inv_temperature=inv_temperature, top_k=top_k, logprob=_lib.ptr(logprob), entropy=entropy.data_ptr(),
        lse=lse.data_ptr(), stats=_lib.ptr(stats), top_logprobs=_lib.ptr(top_logprobs), top_ids=_lib.ptr(top_ids))
    if outer * inner:
        _rows.launch("dwarf_token_logprobs", args, dev)
    return logprob, entropy, lse, stats, top_logprobs, top_ids


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top_k, inv_temperature, ignore_index):
        logprob, entropy, lse, stats, top_logprobs, top_ids = _forward(logits, targets, top_k, inv_temperature,
                                                                       ignore_index, True)
        ctx.save_for_backward(logits, targets, entropy, stats, top_ids)
        ctx.scalars = (top_k, inv_temperature, ignore_index)
        if top_ids is not None:
            ctx.mark_non_differentiable(top_ids)
        ctx.set_materialize_grads(False)
        return logprob, entropy, lse, top_logprobs, top_ids

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, g_lse, g_top, no_grad):
        if torch.is_grad_enabled():  # create_graph: a second derivative is refused, not left out
            return _once_more(ctx, g_logprob, g_entropy, g_lse, g_top, no_grad)
        logits, targets, entropy, stats, top_ids = ctx.saved_tensors
        top_k, inv_temperature, ignore_index = ctx.scalars
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        logits, outer, inner, so, si = _rows.addressed(logits)
        g_logprob, g_entropy, g_lse, g_top = (None if g is None else _rows.in_memory(g).contiguous()
                                              for g in (g_logprob, g_entropy, g_lse, g_top))
        args = _lib.TokenLogprobsBwdArgs(
            version=_lib.ABI_VERSION, dtype=_lib.dtype_code(logits.dtype), logits=logits.data_ptr(), outer=outer,
            inner=inner, vocab=logits.shape[-1], so=so, si=si, targets=_lib.ptr(targets), ignore_index=ignore_index,
            inv_temperature=inv_temperature, top_k=top_k, stats=stats.data_ptr(), entropy=entropy.data_ptr(),
            top_ids=_lib.ptr(top_ids), g_logprob=_lib.ptr(g_logprob), g_entropy=_lib.ptr(g_entropy),
            g_lse=_lib.ptr(g_lse), g_top=_lib.ptr(g_top), grad=grad.data_ptr())
        if outer * inner:
            _rows.launch("dwarf_token_logprobs_bwd", args, logits.device)
        return grad, None, None, None, None


_once_more = torch.autograd.function.once_differentiable(_TokenLogprobsFn.backward)


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top_k: int = 0,
                   temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities under ``softmax(logits / temperature)``.

    ``logits`` [..., V] float32, bfloat16 or float16 (``logits[:, :-1]`` is read in
    place); ``targets`` [...] int64 or int32, or None. All statistics are fp32.

    * ``logprob``: of the targets; 0 where ``targets == ignore_index``, NaN for any
      other target outside [0, V).
    * ``entropy`` of each row and ``lse``, both at the temperature.
    * ``top_ids`` / ``top_logprobs``: the ``top_k`` (0..128) largest logits, ties to
      the lowest id.

    A row without a finite logit gives logprob, lse and top_logprobs -inf, entropy 0
    and a gradient of zeros; a row with NaN or +inf gives NaN. Every float output is
    differentiable with respect to the logits; a row whose output gradients are all
    zero gets exact zeros. The same call gives the same bits every time; a row's last bits
    may change with the number of rows beside it, which decides how many threads share a row.
    Second and forward-mode derivatives and torch.func transforms
    are refused. Runs on the current stream, without synchronising.
    """
    _rows.refuse_transforms(logits=logits, targets=targets)
    logits = _rows.in_memory(logits)
    inv_temperature = _rows.check_logits(logits, temperature)
    top_k = int(top_k)
    if not 0 <= top_k <= min(_rows.TOP_K_MAX, logits.shape[-1]):
        raise ValueError(f"top_k must be in [0, {min(_rows.TOP_K_MAX, logits.shape[-1])}], got {top_k}")
    if targets is not None:
        targets = _rows.ids64(targets, logits.shape[:-1], "targets")
    _rows.same_device(logits, targets=targets)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, targets, top_k, inv_temperature, int(ignore_index)))
    logprob, entropy, lse, _, top_logprobs, top_ids = _forward(logits, targets, top_k, inv_temperature,
                                                               int(ignore_index), False)
    return TokenLogprobs(logprob, entropy, lse, top_logprobs, top_ids)
