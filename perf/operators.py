"""Cases of the vocabulary-row operators: log probabilities of given tokens (with entropy and top alternatives) and
distillation from a teacher's top log probabilities, forward and backward.

``run`` computes them in a plain form (elementary torch operations in 32 bits) or, where ``own`` is true, through
``dwarf_v2_b200``'s entry points. ``exact`` computes them from their definitions in 64 bits.
"""

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, op, rows, vocab, dtype, k, *, grad=False, batch=0, tau=1.0, tail=True, allowed=1.0, unused=0.0,
          reduction="mean"):
    """op: "logprobs" or "distill"; rows x vocab logits; k: top alternatives / teacher entries per row; grad: the
    backward pass too; batch > 0: the rows are logits[:, :-1] of ``batch`` sequences; allowed: the share of the
    vocabulary that a constrained decoder leaves; unused: the share of ignored rows and of unused teacher slots."""
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "grad": grad, "batch": batch, "tau": tau,
            "tail": tail, "allowed": allowed, "unused": unused, "reduction": reduction}
    return {"name": name, **case} if name else case


def listed():
    return [
        # a decoding step of one sequence that reports 20 alternatives: latency counts
        _case("decode 1 row", "logprobs", 1, 32768, "bf16", 20),
        # a decoding step of 64 sequences under a grammar that leaves 2% of the vocabulary, fp32 logits
        _case("decode 64 rows constrained", "logprobs", 64, 32768, "fp32", 20, allowed=0.02),
        # the log probabilities of one prompt of 2048 tokens with 5 alternatives each
        _case("prompt 2047 rows", "logprobs", 2047, 32768, "bf16", 5),
        # a teacher's pass over a batch of 8 x 2048 tokens: the 64 entries that a student learns from
        _case("teacher 16384 rows", "logprobs", 16384, 32768, "bf16", 64, tau=2.0),
        # scoring 32 sequences of 2048 tokens: rows of logits[:, :-1]
        _case("scoring 32 x 2047 rows", "logprobs", 32 * 2047, 32768, "bf16", 0, batch=32, unused=0.1),
        # a policy-gradient step: log probability and entropy of 8 x 1024 sampled tokens, with gradient
        _case("policy 8192 rows", "logprobs", 8192, 32768, "bf16", 0, grad=True, unused=0.2),
        # the same at an odd vocabulary in fp32, with the alternatives' gradients
        _case("policy 1000 rows odd", "logprobs", 1000, 32003, "fp32", 4, grad=True, unused=0.2),
        # a small student on a small vocabulary (the sizes of a test run)
        _case("student 128 rows small", "distill", 128, 512, "fp32", 8, grad=True),
        # the loss on held-out tokens, without gradient
        _case("held-out 2047 rows", "distill", 2047, 32768, "fp16", 32, tail=False, unused=0.1),
        # a training step of a student on 8 x 2048 tokens
        _case("student 16384 rows", "distill", 16384, 32768, "bf16", 64, grad=True, tau=2.0, unused=0.05),
        # a wide odd vocabulary, packed sequences with padding, and a loss for each row
        _case("student 3001 rows odd", "distill", 3001, 65003, "bf16", 100, grad=True, unused=0.3, reduction="none"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["logprobs", "distill"])
    grad = rng.random() < 0.5
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    vocab = rng.choice([32768, spread(500, 131072), spread(500, 131072) | 1, 16 * spread(32, 8192)])
    rows = max(1, min(spread(1, 32768), (1 << 28) // vocab))
    batch = 0
    if rows >= 64 and rng.random() < 0.25:
        batch = rng.choice([2, 4, 8])
        rows -= rows % batch
    k = spread(1, 128) if op == "distill" or rng.random() < 0.7 else 0
    return _case("", op, rows, vocab, dtype, k, grad=grad, batch=batch, tau=rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]),
                 tail=rng.random() < 0.6, unused=rng.choice([0.0, 0.1, 0.4]),
                 allowed=rng.choice([1.0, 0.05, 0.5]) if op == "logprobs" and not grad else 1.0,
                 reduction=rng.choice(["mean", "sum", "none"]))


def _logits(case, gen):
    """Rows of a language model's kind: a bias per token that falls with its (shuffled) frequency rank, and noise."""
    rows, vocab, batch = case["rows"], case["vocab"], case["batch"]
    rank = torch.randperm(vocab, generator=gen, device="cuda")
    bias = -1.2 * torch.log(rank.float() + 3.0) + 6.0
    shape = (batch, rows // batch + 1, vocab) if batch else (rows, vocab)
    x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=gen)
    x.mul_(1.6).add_(bias)
    if case["allowed"] < 1.0:
        x.masked_fill_(torch.rand(vocab, generator=gen, device="cuda") >= case["allowed"], -math.inf)
        x[..., 0] = 1.0  # the end of the text is allowed always
    return x.to(_TYPES[case["dtype"]])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    logits = _logits(case, gen)
    lead = (case["batch"], rows // case["batch"]) if case["batch"] else (rows,)
    if case["grad"]:
        logits.requires_grad_()
    state = {"case": case, "logits": logits}
    off = torch.rand(lead, generator=gen, device="cuda") < case["unused"]
    if case["op"] == "logprobs":
        targets = torch.randint(0, vocab, lead, generator=gen, device="cuda")
        if case["allowed"] < 1.0:
            targets.zero_()
        state["targets"] = targets.masked_fill_(off, -100)
        if case["grad"]:  # advantages, the entropy bonus, and the alternatives' weights
            state["g_logprob"] = torch.randn(lead, generator=gen, device="cuda") / rows
            state["g_entropy"] = torch.full(lead, -0.01 / rows, device="cuda")
            state["g_top"] = torch.randn((*lead, k), generator=gen, device="cuda") / rows if k else None
        return state
    # the teacher's entries: distinct ids and falling log probabilities that leave a tail
    first = torch.randint(0, vocab, (*lead, 1), generator=gen, device="cuda")
    ids = (first + torch.arange(k, device="cuda") * (vocab // k)) % vocab
    raw = torch.randn((*lead, k), generator=gen, device="cuda").mul_(1.5).sub_(0.05 * torch.arange(k, device="cuda"))
    mass = 0.6 + 0.39 * torch.rand((*lead, 1), generator=gen, device="cuda")
    logprobs = torch.log_softmax(raw, -1) + torch.log(mass)
    logprobs, order = logprobs.sort(-1, descending=True)
    ids = ids.gather(-1, order)
    slot = torch.arange(k, device="cuda")
    cut = torch.where(off.unsqueeze(-1), k // 2, k)  # rows with fewer entries
    state["ids"] = ids.masked_fill(slot >= cut.clamp(min=1), -1)
    state["logprobs"] = logprobs
    state["row_mask"] = torch.rand(lead, generator=gen, device="cuda") >= case["unused"] if case["unused"] else None
    if case["grad"] and case["reduction"] == "none":
        state["g_loss"] = torch.rand(lead, generator=gen, device="cuda") / rows
    return state


def _rows_of(state):
    logits = state["logits"]
    return logits[:, :-1] if state["case"]["batch"] else logits


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    with torch.no_grad():
        out = _plain_logprobs(state) if case["op"] == "logprobs" else _plain_distill(state)
        if case["grad"] and case["batch"]:  # the gradient of logits[:, :-1] in that of the logits
            grad = torch.zeros_like(state["logits"])
            grad[:, :-1] = out["grad"]
            out["grad"] = grad
    return out


def _run_own(state):
    from dwarf_v2_b200.distillation import topk_distillation_loss
    from dwarf_v2_b200.logprobs import token_logprobs

    case = state["case"]
    rows = _rows_of(state)
    if case["op"] == "logprobs":
        got = token_logprobs(rows, state["targets"], top_k=case["k"], temperature=case["tau"])
        out = {"logprob": got.logprob, "entropy": got.entropy, "lse": got.lse}
        if case["k"]:
            out |= {"top_logprobs": got.top_logprobs, "top_ids": got.top_ids}
        if case["grad"]:
            ends, weights = [got.logprob, got.entropy], [state["g_logprob"], state["g_entropy"]]
            if case["k"]:
                ends, weights = ends + [got.top_logprobs], weights + [state["g_top"]]
            out["grad"], = torch.autograd.grad(ends, state["logits"], weights)
        return out
    loss = topk_distillation_loss(rows, state["ids"], state["logprobs"], temperature=case["tau"], tail=case["tail"],
                                  row_mask=state["row_mask"], reduction=case["reduction"])
    out = {"loss": loss}
    if case["grad"]:
        out["grad"], = torch.autograd.grad(loss, state["logits"], state.get("g_loss"))
    return out


# ------------------------------------------------------------------ the plain forms, in 32 bits


def _plain_top(x, k):
    """The k largest values' ids, ties to the lowest: a whole-number key that orders (value, -id)."""
    vocab = x.shape[-1]
    bits = (x.float() + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    key = key * (1 << 24) + (vocab - 1 - torch.arange(vocab, device=x.device))
    return vocab - 1 - torch.topk(key, k, dim=-1).values % (1 << 24)


def _plain_logprobs(state):
    case = state["case"]
    raw = _rows_of(state)
    targets, k, c = state["targets"], case["k"], 1.0 / case["tau"]
    x = raw.float()
    top = x.amax(-1, keepdim=True)
    d = (x - top) * c
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    mean = torch.where(e > 0, e * d, 0.0).sum(-1, keepdim=True) / total
    entropy = log_total - mean
    counted = targets != -100
    index = torch.where(counted, targets, 0).unsqueeze(-1)
    logprob = torch.where(counted, (d.gather(-1, index) - log_total).squeeze(-1), 0.0)
    out = {"logprob": logprob, "entropy": entropy.squeeze(-1), "lse": (top * c + log_total).squeeze(-1)}
    if k:
        ids = _plain_top(raw, k)
        out |= {"top_logprobs": d.gather(-1, ids) - log_total, "top_ids": ids}
    if case["grad"]:
        q = e / total
        g = torch.where(counted, state["g_logprob"], 0.0).unsqueeze(-1)
        weight = g + state["g_top"].sum(-1, keepdim=True) if k else g
        grad = -q * (weight + state["g_entropy"].unsqueeze(-1) * (d - log_total + entropy))
        grad.scatter_add_(-1, index, g)
        if k:
            grad.scatter_add_(-1, ids, state["g_top"])
        out["grad"] = (grad * c).to(raw.dtype)
    return out


def _plain_distill(state):
    case = state["case"]
    raw, ids, teacher, mask = _rows_of(state), state["ids"], state["logprobs"], state["row_mask"]
    c = 1.0 / case["tau"]
    used = ids >= 0
    index = torch.where(used, ids, 0)
    l = torch.where(used, teacher, -math.inf)
    if case["tail"]:
        p = torch.exp(l)
        rest = (1.0 - p.sum(-1, dtype=torch.float64, keepdim=True)).clamp(min=0.0).float()
    else:
        top = l.amax(-1, keepdim=True)
        l = l - top - torch.log(torch.exp(l - top).sum(-1, keepdim=True))
        p = torch.exp(l)
        rest = torch.zeros_like(p[..., :1])
    x = raw.float()
    d = (x - x.amax(-1, keepdim=True)) * c
    e = torch.exp(d)
    listed_ids = torch.zeros_like(e).scatter_add_(-1, index, used.float()) > 0
    total = e.sum(-1, keepdim=True)
    total_rest = torch.where(listed_ids, 0.0, e).sum(-1, keepdim=True)
    log_total = torch.log(total)
    loss = torch.where(used, p * (l - d.gather(-1, index) + log_total), 0.0).sum(-1)
    tail = torch.where(rest > 0, rest * (torch.log(rest) - torch.log(total_rest) + log_total), 0.0)
    loss = loss + tail.squeeze(-1)
    count = float(loss.numel())
    if mask is not None:
        loss = torch.where(mask, loss, 0.0)
        count = mask.sum().clamp(min=1).float()
    out = {"loss": loss if case["reduction"] == "none" else loss.sum(dtype=torch.float64).float()}
    if case["reduction"] == "mean":
        out["loss"] = out["loss"] / count
    if case["grad"]:
        weight = p.sum(-1, keepdim=True) + rest
        grad = e / total * weight - torch.where(listed_ids, 0.0, e / total_rest * rest)
        grad.scatter_add_(-1, index, torch.where(used, -p, 0.0))
        if mask is not None:
            grad = torch.where(mask.unsqueeze(-1), grad, 0.0)
        if case["reduction"] == "none":
            grad = grad * state["g_loss"].unsqueeze(-1)
        elif case["reduction"] == "mean":
            grad = grad / count
        out["grad"] = (grad * c).to(raw.dtype)
    return out


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    size = _TYPES[case["dtype"]].itemsize
    whole = rows * vocab
    grad_values = (rows + case["batch"]) * vocab if case["grad"] else 0
    total = (whole + grad_values) * size
    if case["op"] == "logprobs":
        total += rows * (8 + 3 * 4 + k * (8 + 4)) + (rows * (8 + 4 * k) if case["grad"] else 0)
        flops = whole * 6 + (whole * 6 if case["grad"] else 0)
    else:
        total += rows * (k * (8 + 4) + 4)
        flops = whole * 4 + (whole * 3 if case["grad"] else 0)
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------ the definitions, in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    parts, step = [], max(1, (1 << 27) // case["vocab"])
    rows = _rows_of(state).detach()
    flat = {n: state[n].reshape(case["rows"], *state[n].shape[rows.dim() - 1:])
            for n in ("targets", "g_logprob", "g_entropy", "g_top", "ids", "logprobs", "row_mask", "g_loss")
            if state.get(n) is not None}
    rows = rows.reshape(case["rows"], case["vocab"])
    one = _exact_logprobs if case["op"] == "logprobs" else _exact_distill
    for at in range(0, case["rows"], step):
        parts.append(one(case, rows[at:at + step], {n: t[at:at + step] for n, t in flat.items()}))
    out = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    lead = (case["batch"], case["rows"] // case["batch"]) if case["batch"] else (case["rows"],)
    if case["op"] == "distill" and case["reduction"] != "none":
        count = 1.0
        if case["reduction"] == "mean":
            count = max(1, int(flat["row_mask"].sum())) if "row_mask" in flat else case["rows"]
        total = out.pop("loss").sum() / count
        out = {"loss": total, **{n: t / count for n, t in out.items()}}
    out = {n: t.reshape(*lead, *t.shape[1:]) if t.dim() else t for n, t in out.items()}
    if case["grad"] and case["batch"]:
        out["grad"] = torch.nn.functional.pad(out["grad"], (0, 0, 0, 1))
    return out


def _exact_logprobs(case, rows, given):
    x = rows.double() / case["tau"]
    x.requires_grad_(case["grad"])
    with torch.set_grad_enabled(case["grad"]):
        logq = torch.log_softmax(x, -1)
        entropy = torch.special.entr(logq.exp()).sum(-1) if not case["grad"] else -(logq.exp() * logq).sum(-1)
        counted = given["targets"] != -100
        logprob = logq.gather(-1, given["targets"].clamp(min=0).unsqueeze(-1)).squeeze(-1) * counted
        if not case["grad"]:
            logprob = torch.where(counted, logprob, torch.zeros_like(logprob))
        out = {"logprob": logprob, "entropy": entropy, "lse": torch.logsumexp(x, -1)}
        if case["k"]:
            ids = torch.sort(rows.float(), dim=-1, descending=True, stable=True).indices[..., :case["k"]]
            out |= {"top_logprobs": logq.gather(-1, ids), "top_ids": ids}
        if case["grad"]:
            score = (logprob * given["g_logprob"].double()).sum() + (entropy * given["g_entropy"].double()).sum()
            if case["k"]:
                score = score + (out["top_logprobs"] * given["g_top"].double()).sum()
            out["grad"] = torch.autograd.grad(score, x)[0] / case["tau"]
    return {n: t.detach() for n, t in out.items()}


def _exact_distill(case, rows, given):
    x = rows.double() / case["tau"]
    x.requires_grad_(case["grad"])
    ids, used = given["ids"].clamp(min=0), given["ids"] >= 0
    l = given["logprobs"].double().masked_fill(~used, -math.inf)
    if not case["tail"]:
        l = torch.log_softmax(l, -1)
    p = l.exp()
    with torch.set_grad_enabled(case["grad"]):
        logq = torch.log_softmax(x, -1)
        loss = (p * (l.masked_fill(~used, 0.0) - logq.gather(-1, ids))).sum(-1)
        if case["tail"]:
            drop = torch.zeros_like(x, dtype=torch.int32).scatter_add_(-1, ids, used.int()) > 0
            rest = (1.0 - p.sum(-1)).clamp(min=0.0)
            loss = loss + torch.special.xlogy(rest, rest) - rest * torch.logsumexp(
                logq.masked_fill(drop, -math.inf), -1)
        weight = torch.ones_like(loss)
        if "row_mask" in given:
            weight = weight * given["row_mask"]
        out = {"loss": loss * weight}
        if case["grad"]:
            up = weight * given["g_loss"].double() if "g_loss" in given else weight
            out["grad"] = torch.autograd.grad((loss * up).sum(), x)[0] / case["tau"]
    return {n: t.detach() for n, t in out.items()}
