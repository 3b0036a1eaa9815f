"""Vocabulary-row operators in 64 bits: token log probabilities (with entropy and top
alternatives) and distillation from a teacher's listed entries, with their gradients.

The reference has neither; both are restated from their definitions:

* q = softmax(x / t); logprob, entropy = -sum q log q, lse = logsumexp(x / t), the top
  entries by value with ties to the lowest id; d(logprob_v)/dx = (1[v] - q) / t,
  d(entropy)/dx = -q (log q + entropy) / t, d(lse)/dx = q / t.
* KL(p || q) over the listed ids and, with a tail, the event "none of them";
  dKL/dx = (q W - sum p at the listed ids - p_* q / q_* at the others) / t, W = sum p + p_*.
"""

from __future__ import annotations

import math

import torch


def _log_softmax(x):
    """(log softmax, logsumexp), shifted by the maximum first: at the type's lowest value x - lse would lose log V."""
    top = x.amax(-1, keepdim=True)
    z = x - torch.where(top == -math.inf, torch.zeros_like(top), top)
    lse = torch.logsumexp(z, -1, keepdim=True)
    return z - lse, (top + lse).squeeze(-1)


def token_logprobs(x, targets=None, *, top_k=0, temperature=1.0, ignore_index=-100):
    """Dict of logprob, entropy, lse, top_logprobs, top_ids for x [R, V] (any floating type)."""
    raw = x.double()
    x = raw / temperature
    V = x.shape[-1]
    bad = (torch.isnan(x) | (x == math.inf)).any(-1)
    empty = (x == -math.inf).all(-1)
    safe = torch.where((bad | empty).unsqueeze(-1), torch.zeros_like(x), x)
    logq, lse = _log_softmax(safe)
    entropy = -torch.where(logq > -math.inf, torch.exp(logq) * logq, torch.zeros_like(logq)).sum(-1)

    def special(t, empty_value):
        t = torch.where(empty.reshape(-1, *[1] * (t.ndim - 1)), torch.full_like(t, empty_value), t)
        return torch.where(bad.reshape(-1, *[1] * (t.ndim - 1)), torch.full_like(t, math.nan), t)

    out = {"lse": special(lse, -math.inf), "entropy": special(entropy, 0.0)}
    if targets is not None:
        inside = (targets >= 0) & (targets < V)
        lp = special(logq.gather(-1, targets.clamp(0, V - 1).unsqueeze(-1)).squeeze(-1), -math.inf)
        lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
        out["logprob"] = torch.where(targets == ignore_index, torch.zeros_like(lp), lp)
    if top_k:
        order = torch.where(torch.isnan(raw), torch.full_like(raw, math.inf), raw)
        order = torch.sort(order, dim=-1, descending=True, stable=True).indices
        # NaN before +inf: a second stable pass over what the first left in value order
        nan_first = torch.sort((~torch.isnan(raw)).gather(-1, order).int(), dim=-1, stable=True).indices
        ids = order.gather(-1, nan_first)[:, :top_k]
        out["top_ids"] = ids
        out["top_logprobs"] = special(logq.gather(-1, ids), -math.inf)
    return out


def token_logprobs_grad(x, targets=None, *, top_ids=None, g_logprob=None, g_entropy=None, g_lse=None, g_top=None,
                        temperature=1.0, ignore_index=-100):
    """(gradient of x [R, V], the sum of the magnitudes of its terms) for rows of finite or -inf logits."""
    out = token_logprobs(x, targets, temperature=temperature, ignore_index=ignore_index)
    x = x.double() / temperature
    empty = (x == -math.inf).all(-1, keepdim=True)
    logq = _log_softmax(torch.where(empty, torch.zeros_like(x), x))[0]
    q = torch.exp(logq)
    zero = torch.zeros(x.shape[0], 1, dtype=torch.float64, device=x.device)
    weight, sparse, size = zero, torch.zeros_like(x), torch.zeros_like(x)
    if g_logprob is not None:
        counted = targets != ignore_index
        g = torch.where(counted, g_logprob.double(), 0.0).unsqueeze(-1)
        at = torch.where(counted, targets, 0).unsqueeze(-1)
        weight = weight + g
        sparse.scatter_add_(-1, at, g)
        size.scatter_add_(-1, at, g.abs())
    if g_top is not None:
        weight = weight + g_top.double().sum(-1, keepdim=True)
        sparse.scatter_add_(-1, top_ids, g_top.double())
        size.scatter_add_(-1, top_ids, g_top.double().abs())
    if g_lse is not None:
        weight = weight - g_lse.double().unsqueeze(-1)
    absolute = sum((g.double().abs().reshape(x.shape[0], -1).sum(-1, keepdim=True)
                    for g in (g_logprob, g_top, g_lse) if g is not None), zero)
    dense, dense_size = -q * weight, q * absolute
    if g_entropy is not None:
        gh = g_entropy.double().unsqueeze(-1)
        h = out["entropy"].unsqueeze(-1)
        lq = torch.where(q > 0, logq, torch.zeros_like(logq))
        dense = dense - q * gh * (lq + h)
        dense_size = dense_size + q * gh.abs() * (lq.abs() + h)
    grad = torch.where(empty, torch.zeros_like(x), (sparse + dense) / temperature)
    return grad, (size + dense_size) / temperature


def topk_distillation(x, ids, logprobs, *, temperature=1.0, tail=True, row_mask=None, upstream=None):
    """(loss [R], gradient of x [R, V] under ``upstream`` [R], size of the gradient's terms, size of the loss's terms)."""
    x = x.double() / temperature
    R, V = x.shape
    used = ids >= 0
    keep = used.any(-1)
    if row_mask is not None:
        keep = keep & row_mask
    off = (ids >= V).any(-1) & keep
    empty = (x == -math.inf).all(-1) & keep
    x = torch.where((keep & ~empty).unsqueeze(-1), x, torch.zeros_like(x))
    at = ids.clamp(0, V - 1)
    l = torch.where(used, logprobs.double(), torch.full_like(logprobs, -math.inf, dtype=torch.float64))
    if tail:
        p = torch.exp(l)
        rest = (1.0 - p.sum(-1, keepdim=True)).clamp(min=0.0)
    else:
        l = l - torch.logsumexp(torch.where(keep.unsqueeze(-1), l, torch.zeros_like(l)), -1, keepdim=True)
        p = torch.exp(l)
        rest = torch.zeros(R, 1, dtype=torch.float64, device=x.device)
    hit = torch.zeros(R, V, dtype=torch.float64, device=x.device).scatter_add_(-1, at, used.double()) > 0
    rest = torch.where(hit.all(-1, keepdim=True), torch.zeros_like(rest), rest)
    logq = _log_softmax(x)[0]
    logq_rest = torch.logsumexp(torch.where(hit, torch.full_like(x, -math.inf), logq), -1, keepdim=True)
    some = used & (p > 0)
    zero = torch.zeros_like(p)
    terms = torch.where(some, p * (torch.where(some, l, zero) - torch.where(some, logq.gather(-1, at), zero)), zero)
    rest_term = torch.where(rest > 0, rest * (torch.log(rest.clamp(min=1e-300)) - logq_rest), torch.zeros_like(rest))
    loss = terms.sum(-1) + rest_term.squeeze(-1)
    loss = torch.where(torch.isnan(p.sum(-1)), torch.full_like(loss, math.nan), loss)  # nothing to normalise
    loss_size = (torch.where(some, p * (l.clamp(min=-1e4).abs() + logq.gather(-1, at).abs()), zero).sum(-1)
                 + rest_term.abs().squeeze(-1) + rest.squeeze(-1) * logq_rest.clamp(min=-1e4).abs().squeeze(-1))
    q = torch.exp(logq)
    mass = torch.zeros_like(x).scatter_add_(-1, at, torch.where(used, p, zero))
    # (where the student gives the ids not listed nothing, the loss is inf and their gradient 0)
    share = torch.where(hit | (rest == 0) | (logq_rest == -math.inf), torch.zeros_like(x),
                        rest * torch.exp(logq - logq_rest))
    weight = p.sum(-1, keepdim=True) + rest
    grad, size = q * weight - mass - share, q * weight + mass + share
    up = torch.ones(R, dtype=torch.float64, device=x.device) if upstream is None else upstream.double()
    up = up.unsqueeze(-1) / temperature
    dead = ~keep.unsqueeze(-1)
    grad = torch.where(dead, torch.zeros_like(grad), grad * up)
    # without a finite logit every q is 0, as its logarithm in token_logprobs says: the loss is inf, the gradient 0
    given = weight.squeeze(-1)
    nothing = torch.where(given > 0, torch.full_like(given, math.inf), given)  # (NaN stays NaN)
    grad = torch.where(empty.unsqueeze(-1), torch.zeros_like(grad) * weight, grad)
    loss = torch.where(empty, nothing, loss)
    loss = torch.where(keep, loss, torch.zeros_like(loss))
    grad = torch.where(off.unsqueeze(-1), torch.full_like(grad, math.nan), grad)
    loss = torch.where(off, torch.full_like(loss, math.nan), loss)
    return loss, grad, size * up.abs(), loss_size
