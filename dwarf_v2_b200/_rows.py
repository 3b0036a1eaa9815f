"""What the vocabulary-row operators share: how a logit tensor's rows are addressed, and their checks."""

from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _lib

TOP_K_MAX = 128
VOCAB_MAX = 1 << 20
_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def check_logits(logits: torch.Tensor, temperature: float) -> float:
    """1 / temperature, after the checks of a [..., vocab] logit tensor."""
    if logits.ndim < 1:
        raise ValueError("logits must be [..., vocab]")
    if logits.dtype not in _TYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if not 1 <= logits.shape[-1] <= VOCAB_MAX:
        raise ValueError(f"the vocabulary must hold 1..{VOCAB_MAX} entries, got {logits.shape[-1]}")
    if logits.numel() // logits.shape[-1] >= 1 << 28:
        raise ValueError("too many rows")
    temperature = float(temperature)
    if not (math.isfinite(temperature) and 1e-30 <= temperature <= 1e30):
        raise ValueError(f"temperature must be positive and finite (1e-30..1e30), got {temperature}")
    return 1.0 / temperature


def refuse_transforms(**tensors: torch.Tensor | None) -> None:
    """Forward-mode derivatives and torch.func transforms are refused: a kernel reads a tensor's memory, where
    a tangent or a batch dimension would be left out unseen."""
    if forward_ad._current_level < 0 and torch._C._functorch.peek_interpreter_stack() is None:
        return  # neither is under way
    for name, t in tensors.items():
        if t is None:
            continue
        if torch._C._functorch.is_functorch_wrapped_tensor(t):
            raise NotImplementedError(f"{name}: torch.func transforms (vmap, grad, jvp, ...) are not supported")
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name}: forward-mode derivatives are not supported")


def in_memory(t: torch.Tensor) -> torch.Tensor:
    """``t`` with its sign applied: a lazily negated view (the imaginary part of a conjugate) is copied."""
    return t.resolve_neg() if t.is_neg() else t


def same_device(logits: torch.Tensor, **others: torch.Tensor | None) -> None:
    """Every tensor on the logits' CUDA device."""
    _lib.require_cuda(logits, *others.values())
    for name, t in others.items():
        if t is not None and t.device != logits.device:
            raise ValueError(f"{name} is on {t.device}, the logits are on {logits.device}")


def ids64(t: torch.Tensor, shape, name: str) -> torch.Tensor:
    """A contiguous int64 tensor of ``shape``."""
    if t.dtype is torch.int64 and t.shape == shape and t.is_contiguous():
        return t
    if t.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{name} must be int64 or int32, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    return t.to(torch.int64).contiguous()


def addressed(logits: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """(logits, outer, inner, outer stride, inner stride) of a [..., vocab] tensor.

    Leading dimensions that lie one behind the other are merged; up to two groups
    (``logits[:, :-1]``) are read in place, anything else is copied first."""
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if logits.is_contiguous():
        vocab = logits.shape[-1]
        return logits, 1, logits.numel() // vocab, 0, vocab
    groups: list[list[int]] = []
    for n, stride in zip(logits.shape[:-1], logits.stride()[:-1]):
        if n == 1:
            continue
        if groups and groups[-1][1] == stride * n:
            groups[-1] = [groups[-1][0] * n, stride]
        else:
            groups.append([n, stride])
    if len(groups) > 2:
        return addressed(logits.contiguous())
    groups = [[1, 0]] * (2 - len(groups)) + groups
    (outer, so), (inner, si) = groups
    return logits, outer, inner, so, si


def launch(name: str, args, device: torch.device) -> None:
    """``_lib.call`` with ``device`` current (a launch goes to the current device)."""
    if torch.cuda.current_device() == device.index:
        _lib.call(name, args, device)
    else:
        with torch.cuda.device(device):
            _lib.call(name, args, device)
