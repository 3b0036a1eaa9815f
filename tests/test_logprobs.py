"""Token log probabilities, entropy and top alternatives of logit rows, and their gradient,
against the 64-bit oracle (oracle/vocab.py).

Tolerances. One exponential is off by at most 2^-22 (ex2.approx) plus the rounding of its
exponent d = c (x - m) log2 e (three roundings of 2^-24 relative: |d| ln2 3 2^-24). A sum over V
entries adds at most N 2^-24 where N is the number of additions that one value passes: under
V / 128 + 64 in any split of a row over threads. So a sum of exponentials is off by
``rel = 2^-21 + (V / 128 + 64) 2^-24`` at the weight e (1 + |d|) <= 1 of its terms, a logarithm of it by
the same absolute amount, and lse, logprob by that and two roundings (2^-23) of their own size and of the
row maximum's. The entropy is a quotient of two such sums: rel (2 + entropy).
Gradients are held entry by entry to rel times the sum of the magnitudes of their terms, with |d| ln2 2^-22
for the exponent, plus the one rounding of the type (eps / 2 of the value; the smallest subnormal of fp16).
"""

import math

import pytest
import torch

from oracle import vocab as oracle

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def rel_of(V):
    return 2.0 ** -21 + (V / 128 + 64) * 2.0 ** -24


def close(got, want, tol, what=""):
    got, want = got.double().cpu(), want.double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu().expand(want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine] - tol[fine]
    assert off.numel() == 0 or off.max() <= 0, (what, float(off.max()), float((got - want).abs()[fine].max()))


def check_forward(out, x, targets, k, t, ignore_index=-100):
    R, V = x.numel() // x.shape[-1], x.shape[-1]
    want = oracle.token_logprobs(x.reshape(R, V), None if targets is None else targets.reshape(R), top_k=k,
                                 temperature=t, ignore_index=ignore_index)
    rel = rel_of(V)
    # a row without a finite logit has a maximum of 0 here: its outputs are exact values
    top = torch.nan_to_num(x.double().reshape(R, V).amax(-1) / t, nan=0.0, posinf=0.0, neginf=0.0).abs()

    def tol(v):
        return rel + 2.0 ** -22 * torch.nan_to_num(want[v], nan=0.0, posinf=0.0, neginf=0.0).abs()

    close(out.lse.reshape(R), want["lse"], tol("lse") + 2.0 ** -23 * top, "lse")
    h = torch.nan_to_num(want["entropy"], nan=0.0)
    close(out.entropy.reshape(R), want["entropy"], rel * (2.0 + 2.0 * h + math.log(V)), "entropy")
    if targets is None:
        assert out.logprob is None
    else:
        close(out.logprob.reshape(R), want["logprob"], tol("logprob"), "logprob")
    if k:
        assert torch.equal(out.top_ids.reshape(R, k).cpu(), want["top_ids"].cpu())
        close(out.top_logprobs.reshape(R, k), want["top_logprobs"], tol("top_logprobs"), "top_logprobs")
    else:
        assert out.top_ids is None and out.top_logprobs is None
    return want


def grad_tolerance(x, t, grad, size):
    V = x.shape[-1]
    d = torch.nan_to_num((x.double() - x.double().amax(-1, keepdim=True)) / t, neginf=0.0).abs()
    # an exponential below 2^-126 counts as 0: a term q (G + gH (|log q| + H)) is then left out whole, at most
    # 2^-126 (2 + 88 + 12) < 2^-119 of gradients whose c G and c gH are 2 and 1 (the others have no such terms)
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -119
    return size * (4 * rel_of(V) + d * 2.0 ** -21) + torch.finfo(x.dtype).eps / 2 * grad.abs() * 1.01 + tiny


def logits(R, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * spread).to(TYPES[dtype])


# ------------------------------------------------------------------ CPU: the oracle, refusals


def test_oracle_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 11, generator=g, dtype=torch.float64)
    targets = torch.tensor([4, -100, 0])
    gl, gh, gz = (torch.randn(3, generator=g, dtype=torch.float64) for _ in range(3))
    gt = torch.randn(3, 2, generator=g, dtype=torch.float64)
    out = oracle.token_logprobs(x, targets, top_k=2, temperature=1.7)

    def value(v):
        o = oracle.token_logprobs(v, targets, temperature=1.7)
        logq = v / 1.7 - o["lse"].unsqueeze(-1)
        return ((gl * o["logprob"] + gh * o["entropy"] + gz * o["lse"]).sum()
                + (gt * logq.gather(-1, out["top_ids"])).sum())

    grad, _ = oracle.token_logprobs_grad(x, targets, top_ids=out["top_ids"], g_logprob=gl, g_entropy=gh, g_lse=gz,
                                         g_top=gt, temperature=1.7)
    for i in range(3):
        for v in range(11):
            step = torch.zeros_like(x)
            step[i, v] = 1e-5
            diff = (value(x + step) - value(x - step)) / 2e-5
            assert abs(diff - grad[i, v]) < 1e-8


def test_refuses_what_it_does_not_take():
    from dwarf_v2_b200.logprobs import token_logprobs

    x = torch.zeros(4, 10)
    with pytest.raises(RuntimeError):
        token_logprobs(x)
    with pytest.raises(TypeError):
        token_logprobs(x.double())
    with pytest.raises(TypeError):
        token_logprobs(x, torch.zeros(4))
    for bad in (-1, 11, 129):
        with pytest.raises(ValueError):
            token_logprobs(x, top_k=bad)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(4, 300), top_k=129)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            token_logprobs(x, temperature=bad)
    with pytest.raises(ValueError):
        token_logprobs(x, torch.zeros(5, dtype=torch.int64))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(4, 0))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(()))
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(1, (1 << 20) + 1))


def test_row_addressing():
    from dwarf_v2_b200._rows import addressed

    x = torch.zeros(4, 6, 10)
    assert addressed(x)[1:] == (1, 24, 0, 10)
    assert addressed(x[:, :-1])[1:] == (4, 5, 60, 10)
    assert addressed(x[:, -1])[1:] == (1, 4, 0, 60)
    assert addressed(x[0, 0])[1:4] == (1, 1, 0)
    assert addressed(x[:1, :-1])[1:] == (1, 5, 0, 10)
    assert addressed(x[..., :7])[1:] == (1, 24, 0, 10)
    assert addressed(torch.zeros(1, 10).expand(5, 10))[1:] == (1, 5, 0, 0)
    y = torch.zeros(3, 4, 5, 10)[:, :-1, :-1]
    got, *rest = addressed(y)
    assert got.is_contiguous() and rest == [1, 36, 0, 10]
    got, *rest = addressed(torch.zeros(10, 4).t())
    assert got.is_contiguous() and rest == [1, 4, 0, 10]
    assert addressed(torch.zeros(2, 0, 10))[1] * addressed(torch.zeros(2, 0, 10))[2] == 0


def test_launches_on_the_tensors_device(monkeypatch):
    """A launch goes to the current device: the tensors' one is made current for it, and only where it is not."""
    from dwarf_v2_b200 import _lib, _rows

    current, seen = [0], []

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "call", lambda name, args, device: seen.append((name, current[0], device.index)))
    for index in (0, 3):
        _rows.launch("dwarf_row_reduce", None, torch.device("cuda", index))
    assert seen == [("dwarf_row_reduce", 0, 0), ("dwarf_row_reduce", 3, 3)] and current == [0]


def test_c_entry_refuses_bad_arguments():
    import ctypes

    from dwarf_v2_b200 import _lib

    lib = _lib.load()

    def status(name, struct, **fields):
        base = dict(version=_lib.ABI_VERSION, dtype=1, logits=4096, outer=1, inner=2, vocab=64, so=0, si=64,
                    inv_temperature=1.0)
        return getattr(lib, name)(ctypes.byref(struct(**{**base, **fields})), None)

    fwd = dict(lse=4096, entropy=4096)
    name, struct = "dwarf_token_logprobs", _lib.TokenLogprobsArgs
    assert getattr(lib, name)(None, None) == -2
    assert status(name, struct, **fwd, version=2) == -1
    assert status(name, struct, lse=4096) == -2
    assert status(name, struct, **fwd, targets=4096) == -2
    assert status(name, struct, **fwd, top_k=1) == -2
    assert status(name, struct, **fwd, logits=None) == -2
    assert status(name, struct, **fwd, vocab=0) == -3
    assert status(name, struct, **fwd, vocab=(1 << 20) + 1) == -3
    assert status(name, struct, **fwd, outer=1 << 20, inner=1 << 20) == -3
    assert status(name, struct, **fwd, top_k=65) == -3
    assert status(name, struct, **fwd, top_k=-1) == -3
    assert status(name, struct, **fwd, si=-64) == -4
    assert status(name, struct, **fwd, logits=4097) == -5
    assert status(name, struct, **fwd, dtype=3) == -6
    assert status(name, struct, **fwd, inv_temperature=0.0) == -9
    assert status(name, struct, **fwd, inv_temperature=math.nan) == -9
    assert status(name, struct, **fwd, inv_temperature=math.inf) == -9
    assert status(name, struct, inner=0, logits=None) == 0  # no rows: nothing to do
    name, struct = "dwarf_token_logprobs_bwd", _lib.TokenLogprobsBwdArgs
    bwd = dict(stats=4096, entropy=4096, grad=4096)
    assert status(name, struct, stats=4096, entropy=4096) == -2
    assert status(name, struct, **bwd, g_logprob=4096) == -2
    assert status(name, struct, **bwd, g_top=4096) == -2
    assert status(name, struct, **bwd, dtype=7) == -6


# ------------------------------------------------------------------ GPU

SHAPES = [(1, 1), (3, 2), (5, 31), (2, 129), (7, 1000), (4, 4097), (3, 32768), (1, 32768), (2, 50001), (9, 8192),
          (300, 515), (1, 131075), (2, 300000), (700, 2049), (1, 1 << 20), (2700, 601), (2700, 2049), (2700, 5), (2665, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,V", SHAPES)
def test_forward(R, V, dtype):
    from dwarf_v2_b200.logprobs import token_logprobs

    x = logits(R, V, dtype, R * 7 + V).cuda()
    g = torch.Generator().manual_seed(5)
    targets = torch.randint(0, V, (R,), generator=g).cuda()
    targets[R // 2] = -100 if R > 1 else 0
    for k in sorted({0, 1, min(5, V), min(20, V), min(128, V)}):
        for t in (1.0, 0.6):
            check_forward(token_logprobs(x, targets, top_k=k, temperature=t), x, targets, k, t)
    check_forward(token_logprobs(x, top_k=1), x, None, 1, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,V", [(6, 77), (3, 32768), (40, 8200), (2, 140001), (2700, 77), (2700, 2051)])
@pytest.mark.parametrize("kind", ["equal", "two_values", "rising", "falling", "front", "stripe", "zeros_signed"])
def test_top_order_of_hard_rows(R, V, dtype, kind):
    """Rows with many ties, and rows whose large values lie together: the ids are exact, ties to the lowest."""
    from dwarf_v2_b200.logprobs import token_logprobs

    i = torch.arange(V)
    row = {"equal": torch.zeros(V), "two_values": (i % 2).float(), "rising": i.float() / V * 20,
           "falling": -i.float() / V * 20, "front": torch.where(i < V // 3, 4.0 + i % 13, 0.0),
           "stripe": torch.where(i % 8 == 3, 5.0 + (i % 24) / 8, -1.0),
           "zeros_signed": torch.where(i % 3 == 0, 0.0, -0.0)}[kind]
    x = (row + torch.zeros(R, 1)).to(TYPES[dtype]).cuda()
    for r in range(min(R, 40)):
        x[r] = x[r].roll(r * 11)
    for k in sorted({1, min(7, V), min(32, V), min(64, V), min(128, V)}):
        check_forward(token_logprobs(x, top_k=k), x, None, k, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [50, 4096, 32768, 33001])
def test_masked_and_special_rows(V, dtype):
    """-inf, the type's lowest value, +inf and NaN: in places, and in whole rows."""
    from dwarf_v2_b200.logprobs import token_logprobs

    low = torch.finfo(TYPES[dtype]).min
    x = logits(14, V, dtype, 3)
    x[0] = -math.inf                      # nothing left
    x[1] = low                            # the lowest value everywhere: uniform
    x[2, 1:] = -math.inf                  # one left
    x[3, 5:] = low
    x[4, ::2] = -math.inf
    x[5] = -math.inf
    x[5, V - 1] = low                     # one finite value, the lowest
    x[6, 7] = math.inf
    x[7, 9] = math.nan
    x[8] = math.nan
    x[9] = math.inf
    x[10, 3], x[10, 8] = math.nan, math.inf
    x[11, :40] = -math.inf
    x[12] = torch.finfo(TYPES[dtype]).max
    x[13, 0] = torch.finfo(TYPES[dtype]).max
    x = torch.cat([x, torch.where(torch.arange(V) % 5 == 0, low, -math.inf).to(x.dtype)[None]]).cuda()  # the lowest or nothing
    targets = torch.full((15,), 1).cuda()
    targets[2], targets[4] = 0, 2
    for k in (1, 20, min(50, V)):
        check_forward(token_logprobs(x, targets, top_k=k), x, targets, k, 1.0)
    if V <= 4096:  # the same among many rows
        many, more = x.repeat(180, 1), targets.repeat(180)
        check_forward(token_logprobs(many, more, top_k=20), many, more, 20, 1.0)
    check_forward(token_logprobs(x[:6], targets[:6], top_k=3, temperature=4.0), x[:6], targets[:6], 3, 4.0)


@pytest.mark.gpu
def test_targets_outside_and_ignored():
    from dwarf_v2_b200.logprobs import token_logprobs

    x = logits(6, 100, "fp32", 0).cuda().requires_grad_()
    targets = torch.tensor([3, -100, -1, 100, 99, 7], dtype=torch.int32).cuda()
    out = token_logprobs(x, targets, ignore_index=7)
    lp = out.logprob.detach().cpu()
    assert torch.isnan(lp[[1, 2, 3]]).all() and lp[5] == 0 and torch.isfinite(lp[[0, 4]]).all()
    grad, = torch.autograd.grad(out.logprob, x, torch.ones_like(out.logprob))
    assert torch.isnan(grad[[1, 2, 3]]).all() and torch.equal(grad[5], torch.zeros_like(grad[5]))
    assert torch.isfinite(grad[[0, 4]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 2), (5, 31, 4), (2, 129, 128), (6, 1000, 0), (3, 32768, 20),
                                   (2, 50001, 3), (1, 131075, 8), (400, 519, 5), (1, 1 << 20, 2),
                                   (2700, 601, 5), (2700, 4000, 0)])
def test_gradient(R, V, k, dtype):
    from dwarf_v2_b200.logprobs import token_logprobs

    t = 1.3
    x = logits(R, V, dtype, R + V).cuda().requires_grad_()
    g = torch.Generator().manual_seed(11)
    targets = torch.randint(0, V, (R,), generator=g).cuda()
    if R > 2:
        targets[1] = -100
    # fp16 gradients of a large vocabulary would be subnormal: the upstream gradients are of a scaled loss
    gl, gh, gz = (torch.randn(R, generator=g).cuda() * 64 for _ in range(3))
    gt = torch.randn(R, k, generator=g).cuda() * 64 if k else None
    out = token_logprobs(x, targets, top_k=k, temperature=t)
    if k:
        targets[0] = int(out.top_ids[0, 0])  # the target among the alternatives: one id twice
        out = token_logprobs(x, targets, top_k=k, temperature=t)
    ends = {"g_logprob": (out.logprob, gl), "g_entropy": (out.entropy, gh), "g_lse": (out.lse, gz)}
    if k:
        ends["g_top"] = (out.top_logprobs, gt)
    for chosen in [list(ends), ["g_logprob"], ["g_entropy"], ["g_lse"]] + ([["g_top"]] if k else []):
        grad, = torch.autograd.grad([ends[c][0] for c in chosen], x, [ends[c][1] for c in chosen], retain_graph=True)
        assert grad.dtype == x.dtype and grad.shape == x.shape
        want, size = oracle.token_logprobs_grad(x.detach(), targets, top_ids=out.top_ids, temperature=t,
                                                **{c: ends[c][1] for c in chosen})
        close(grad, want, grad_tolerance(x.detach(), t, want, size), chosen)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_gradient_of_masked_rows(dtype):
    """-inf entries get gradient 0; a row without a finite logit and a row whose gradients are zero get zeros."""
    from dwarf_v2_b200.logprobs import token_logprobs

    V = 2500
    x = logits(6, V, dtype, 9)
    x[0] = -math.inf
    x[1, ::3] = -math.inf
    x[2, 5:] = -math.inf
    x[3] = math.nan                      # a padded row: its gradients are zero
    x[4] = torch.finfo(TYPES[dtype]).min
    x = x.cuda().requires_grad_()
    targets = torch.tensor([0, 1, 2, 3, 4, 5]).cuda()
    gl = torch.tensor([1.0, 2.0, -1.0, 0.0, 3.0, 1.0]).cuda()
    gh = torch.tensor([0.5, 1.0, 2.0, 0.0, 1.0, 0.0]).cuda()
    out = token_logprobs(x, targets, top_k=3)
    grad, = torch.autograd.grad([out.logprob, out.entropy], x, [gl, gh])
    want, size = oracle.token_logprobs_grad(torch.nan_to_num(x.detach(), nan=0.0, neginf=-math.inf), targets,
                                            g_logprob=gl, g_entropy=gh)
    want[3], size[3] = 0.0, 0.0
    close(grad, want, grad_tolerance(torch.nan_to_num(x.detach(), nan=0.0, neginf=-math.inf), 1.0, want, size))
    assert torch.equal(grad[3], torch.zeros_like(grad[3])) and torch.equal(grad[0], torch.zeros_like(grad[0]))


@pytest.mark.gpu
def test_gradient_against_differences():
    """The fp32 kernel's own outputs, differenced in a direction: 64-bit sums of fp32 outputs."""
    from dwarf_v2_b200.logprobs import token_logprobs

    g = torch.Generator().manual_seed(2)
    x = (torch.randn(4, 600, generator=g)).cuda().requires_grad_()
    targets = torch.randint(0, 600, (4,), generator=g).cuda()
    out = token_logprobs(x, targets)
    grad, = torch.autograd.grad(out.logprob.sum() + out.entropy.sum(), x)
    way = torch.randn(4, 600, generator=g).cuda()
    step = 2.0 ** -6
    with torch.no_grad():
        hi, lo = token_logprobs(x + step * way, targets), token_logprobs(x - step * way, targets)
    diff = ((hi.logprob - lo.logprob).double().sum() + (hi.entropy - lo.entropy).double().sum()) / (2 * step)
    # truncation step^2 |f'''| / 6 < 2^-12 at unit directions per entry; roundings 8 * 8 * 2^-24 / step < 2^-12
    assert abs(float(diff) - float((grad.double() * way.double()).sum())) < 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_strides_and_alignment(dtype):
    from dwarf_v2_b200.logprobs import token_logprobs

    g = torch.Generator().manual_seed(4)
    big = (torch.randn(3, 5, 6, 1031, generator=g) * 2).to(TYPES[dtype]).cuda()
    views = {"contiguous": big, "shifted": big[0, :, :-1], "last": big[0, :, -1], "columns": big[..., 3:1029],
             "three groups": big[:, :-1, :-1], "transposed": big[0, 0].t(), "row": big[1, 2, 3],
             "expanded": big[0, 0, :1].expand(4, 1031), "permuted": big[0].transpose(0, 1), "odd base": big[0, 0, 1:, 1:]}
    for name, view in views.items():
        lead, V = view.shape[:-1], view.shape[-1]
        targets = torch.randint(0, V, lead, generator=g).cuda()
        out = token_logprobs(view, targets, top_k=3)
        assert out.entropy.shape == lead and out.top_ids.shape == (*lead, 3)
        check_forward(out, view.contiguous(), targets, 3, 1.0)
        leaf = view.detach().requires_grad_()
        out = token_logprobs(leaf, targets)
        w = torch.randn(lead, generator=g).cuda() if lead else torch.tensor(1.5).cuda()
        grad, = torch.autograd.grad(out.logprob, leaf, w)
        flat = view.reshape(-1, V)
        want, size = oracle.token_logprobs_grad(flat, targets.reshape(-1), g_logprob=w.reshape(-1))
        close(grad.reshape(-1, V), want, grad_tolerance(flat, 1.0, want, size), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_without_targets_and_extreme_temperatures(dtype):
    """Entropy, lse and alternatives alone, with their gradients; temperatures far from 1."""
    from dwarf_v2_b200.logprobs import token_logprobs

    x = logits(5, 3001, dtype, 12).cuda().requires_grad_()
    for t in (1e-4, 0.02, 1e3):
        out = token_logprobs(x, top_k=4, temperature=t)
        check_forward(out, x.detach(), None, 4, t)
        gh, gt = torch.full((5,), 1.0 * t).cuda(), torch.full((5, 4), 0.5 * t).cuda()
        grad, = torch.autograd.grad([out.entropy, out.top_logprobs], x, [gh, gt])
        want, size = oracle.token_logprobs_grad(x.detach(), top_ids=out.top_ids, temperature=t, g_entropy=gh, g_top=gt)
        close(grad, want, grad_tolerance(x.detach(), t, want, size), t)
    out = token_logprobs(x)
    assert out.logprob is None and out.top_ids is None
    grad, = torch.autograd.grad(out.lse.sum(), x)
    want, size = oracle.token_logprobs_grad(x.detach(), g_lse=torch.ones(5).cuda())
    close(grad, want, grad_tolerance(x.detach(), 1.0, want, size))


@pytest.mark.gpu
def test_second_derivative_is_refused():
    from dwarf_v2_b200.distillation import topk_distillation_loss
    from dwarf_v2_b200.logprobs import token_logprobs

    x = logits(3, 64, "fp32", 0).cuda().requires_grad_()
    ids = torch.arange(4).repeat(3, 1).cuda()
    lp = torch.full((3, 4), -2.0).cuda()
    for value in (token_logprobs(x, torch.tensor([1, 2, 3]).cuda()).logprob.sum(), topk_distillation_loss(x, ids, lp)):
        plain, = torch.autograd.grad(value, x, retain_graph=True)
        grad, = torch.autograd.grad(value, x, create_graph=True)
        assert torch.equal(grad.detach(), plain)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grad.sum(), x)


@pytest.mark.gpu
def test_no_rows_and_neighbours_untouched():
    from dwarf_v2_b200 import _lib, _rows
    from dwarf_v2_b200.logprobs import token_logprobs

    x = torch.zeros(0, 7, device="cuda", requires_grad=True)
    out = token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), top_k=2)
    assert out.logprob.shape == (0,) and out.top_ids.shape == (0, 2)
    assert torch.autograd.grad(out.entropy.sum(), x)[0].shape == (0, 7)
    # one odd row in the middle of a buffer: nothing before or behind it is written
    V = 1003
    row = logits(1, V, "bf16", 1).cuda()
    buf = torch.full((3 * V,), 7.0, dtype=torch.bfloat16, device="cuda")
    out = token_logprobs(row.clone().requires_grad_(), torch.tensor([3]).cuda())
    stats = torch.tensor([[float(row.float().max()), 1.0]], device="cuda")
    one = torch.ones(1, device="cuda")
    targets = torch.tensor([3], device="cuda")
    args = _lib.TokenLogprobsBwdArgs(version=1, dtype=1, logits=row.data_ptr(), outer=1, inner=1, vocab=V, so=0, si=V,
                                     targets=targets.data_ptr(), ignore_index=-100, inv_temperature=1.0, top_k=0,
                                     stats=stats.data_ptr(), entropy=one.data_ptr(), g_logprob=one.data_ptr(),
                                     grad=buf.data_ptr() + 2 * V)
    _rows.launch("dwarf_token_logprobs_bwd", args, row.device)
    assert torch.equal(buf[:V], torch.full_like(buf[:V], 7.0)) and torch.equal(buf[2 * V:], buf[:V])
    assert not (buf[V:2 * V] == 7.0).all()


@pytest.mark.gpu
def test_repeatable_on_streams_and_in_graphs():
    """Bit-identical on a side stream, in a captured and replayed graph (forward and backward), and in two graphs."""
    from dwarf_v2_b200.logprobs import token_logprobs

    x = logits(37, 32768, "bf16", 8).cuda()
    targets = torch.arange(37).cuda()

    def both(v):
        leaf = v.detach().requires_grad_()
        out = token_logprobs(leaf, targets, top_k=20)
        grad, = torch.autograd.grad([out.logprob, out.entropy], leaf,
                                    [torch.ones_like(out.logprob), torch.ones_like(out.entropy)])
        return [out.logprob.detach(), out.entropy.detach(), out.top_logprobs.detach(), out.top_ids, grad]

    eager = both(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both(x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    static = torch.zeros_like(x)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both(static)
        graphs.append((graph, got))
    for shift in (0, 5):
        static.copy_(x.roll(shift, 1))
        want = both(static)
        for graph, got in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
def test_rows_past_32_bit_offsets():
    """A tensor of over 2^32 elements: its last rows are read and their gradient written in place."""
    from dwarf_v2_b200.logprobs import TokenLogprobs, token_logprobs

    V, R = 32768, (1 << 32) // 32768 + 3
    x = torch.empty(R, V, dtype=torch.bfloat16, device="cuda")
    x.zero_()
    tail = logits(3, V, "bf16", 6).cuda()
    x[-3:] = tail
    targets = torch.full((R,), 17, device="cuda")
    x.requires_grad_()
    out = token_logprobs(x, targets, top_k=2)
    check_forward(TokenLogprobs(*(t.detach()[-3:] for t in out)), tail, targets[-3:], 2, 1.0)
    up = torch.zeros(R, device="cuda")
    up[-3:] = 1.0
    grad, = torch.autograd.grad(out.logprob, x, up)
    want, size = oracle.token_logprobs_grad(tail, targets[-3:], g_logprob=up[-3:])
    close(grad[-3:], want, grad_tolerance(tail, 1.0, want, size))
    assert not bool((grad[:-3] != 0).any())


# ------------------------------------------------------------------ scaled maxima past the range of the packed form


def _near_ties(R, V, seed, low, high):
    """fp32 rows whose maxima are spread over [low, high], and whose best entries lie a few steps of the type apart:
    a step times 1 / temperature is from far below to far above 1."""
    g = torch.Generator().manual_seed(seed)
    top = low * (high / low) ** torch.rand(R, 1, generator=g)
    x = top * torch.rand(R, V, generator=g)
    at = torch.stack([torch.randperm(V, generator=g)[:12] for _ in range(R)])
    steps = torch.randint(0, 6, (R, 12), generator=g).float()
    steps[:, 0] = 0
    best = (top.view(torch.int32) - steps.int()).view(torch.float32)
    return x.scatter_(1, at, best), at[:, 3]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1e-12, 1e-10, 1e-9, 5e-9, 1e-8, 2e-8, 3e-8, 1e-7, 1e-6, 1e-5])
@pytest.mark.parametrize("R,V", [(2000, 300), (3000, 261), (6, 20000)])  # 128 threads, a warp for each row, clusters
def test_small_temperatures(R, V, t):
    """c m of up to 10^14: a float's step there is far above the range of an exponent, and d = c x - c m formed from
    the rounded c m would be as far off. The tolerances are those of every temperature: x - m is exact between
    neighbours, so d has its three roundings."""
    from dwarf_v2_b200.logprobs import token_logprobs

    x, targets = _near_ties(R, V, int(-math.log10(t) * 100) + V, 1.0, 130.0)
    x, targets = x.cuda(), targets.cuda()
    check_forward(token_logprobs(x, targets, temperature=t), x, targets, 0, t)
    leaf = x.clone().requires_grad_()
    out = token_logprobs(leaf, targets, top_k=4, temperature=t)
    check_forward(out, x, targets, 4, t)
    g = torch.Generator().manual_seed(3)
    gl, gh = torch.randn(R, generator=g).cuda() * t, torch.randn(R, generator=g).cuda() * t  # c g is of the order of 1
    gt = torch.randn(R, 4, generator=g).cuda() * t
    grad, = torch.autograd.grad([out.logprob, out.entropy, out.top_logprobs], leaf, [gl, gh, gt])
    want, size = oracle.token_logprobs_grad(x, targets, top_ids=out.top_ids, g_logprob=gl, g_entropy=gh, g_top=gt,
                                            temperature=t)
    # (c g is up to 5, and five such terms: the share of an exponential that counts as 0 is below 2^-119 still, by
    # 2^-126 (5 + 5 + 5 (88 + 6)) < 2^-117 at most)
    close(grad, want, grad_tolerance(x, t, want, size) + 2.0 ** -117, "grad")


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [3e7, 3e9, -3e9, 1e20])
@pytest.mark.parametrize("R,V", [(2000, 300), (3000, 261)])
def test_far_offsets(R, V, offset):
    """The same scaled maxima at temperature 1, from logits that lie far from 0 (steps of 2, 256 and more)."""
    from dwarf_v2_b200.logprobs import token_logprobs

    x, targets = _near_ties(R, V, 5, abs(offset), 1.3 * abs(offset))
    if offset < 0:
        x = x + 2 * offset
    x, targets = x.cuda(), targets.cuda()
    for t in (1.0, 150.0):
        check_forward(token_logprobs(x, targets, top_k=3, temperature=t), x, targets, 3, t)


@pytest.mark.gpu
def test_gradient_with_targets_outside():
    """A target outside [0, V) makes its row's gradient NaN exactly where its log probability's gradient is not 0."""
    from dwarf_v2_b200.logprobs import token_logprobs

    x = logits(4, 300, "fp32", 2).cuda()
    targets = torch.tensor([300, -1, 5, -100]).cuda()
    leaf = x.clone().requires_grad_()
    out = token_logprobs(leaf, targets)
    gl, gh = torch.tensor([0.5, 0.0, 0.0, 1.0]).cuda(), torch.ones(4).cuda()
    grad, = torch.autograd.grad([out.logprob, out.entropy], leaf, [gl, gh])
    assert torch.isnan(grad[0]).all()
    want, size = oracle.token_logprobs_grad(x[1:], g_entropy=gh[1:])
    close(grad[1:], want, grad_tolerance(x[1:], 1.0, want, size))


@pytest.mark.gpu
def test_host_threads_with_different_vocabularies():
    """Rows whose alternatives take more than 32 KB of shared memory, of different sizes, from several threads at
    once: the limit that one thread sets for the kernel must hold for another's launch."""
    import ctypes
    import threading

    from dwarf_v2_b200 import _lib

    lib, x, failed = _lib.load(), torch.zeros(1, 1 << 20, device="cuda"), []

    def work(rows, vocab, calls):
        with torch.cuda.stream(torch.cuda.Stream()):
            f, top = torch.zeros(rows, 2, device="cuda"), torch.zeros(rows, device="cuda")
            ids = torch.zeros(rows, dtype=torch.int64, device="cuda")
            args = _lib.TokenLogprobsArgs(version=_lib.ABI_VERSION, dtype=_lib.dtype_code(x.dtype), logits=x.data_ptr(),
                                          outer=1, inner=rows, vocab=vocab, so=0, si=0, inv_temperature=1.0, top_k=1,
                                          entropy=f.data_ptr(), lse=f.data_ptr() + 4 * rows,
                                          top_logprobs=top.data_ptr(), top_ids=ids.data_ptr())
            stream = torch.cuda.current_stream()
            status = {lib.dwarf_token_logprobs(ctypes.byref(args), stream.cuda_stream) for _ in range(calls)}
            stream.synchronize()
            if status != {0} or ids.any():
                failed.append((vocab, status))

    torch.cuda.synchronize()
    # one row: parts of 1 / 8; 80 rows: of 1 / 4
    threads = [threading.Thread(target=work, args=a) for a in ((80, 1 << 20, 1500), (1, 1 << 20, 6000), (1, 1 << 20, 6000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_forward_mode_and_transforms_are_refused():
    """A tangent or a batch dimension is refused before the tensors are looked at, not dropped."""
    from torch.autograd import forward_ad

    from dwarf_v2_b200.distillation import topk_distillation_loss
    from dwarf_v2_b200.logprobs import token_logprobs

    x, ids, lp = torch.randn(4, 10), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    losses = (lambda v: topk_distillation_loss(v, ids, lp), lambda v: topk_distillation_loss(x, ids, v[:, :3]))
    scores = (lambda v: token_logprobs(v).lse, lambda v: token_logprobs(v, ids[:, 0], top_k=2).logprob)
    with forward_ad.dual_level():
        for f in losses + scores:
            for leaf in (x, x.clone().requires_grad_()):
                with pytest.raises(NotImplementedError):
                    f(forward_ad.make_dual(leaf, torch.ones_like(x)))
            with torch.no_grad(), pytest.raises(NotImplementedError):  # no_grad does not stop a forward mode
                f(forward_ad.make_dual(x, torch.ones_like(x))[:, :5])
        with pytest.raises(RuntimeError, match="CUDA"):  # no tangent: as ever
            token_logprobs(x)
    for f in losses + scores:
        for transform in (lambda f: torch.func.vmap(f)(x.expand(2, 4, 10)), lambda f: torch.func.jvp(f, (x,), (x,)),
                          lambda f: torch.func.grad(lambda v: f(v).sum())(x),
                          lambda f: torch.func.functionalize(f)(x)):
            with pytest.raises(NotImplementedError):
                transform(f)
    for f in (lambda i: token_logprobs(x, i).logprob, lambda i: topk_distillation_loss(x, i[:, None], lp[:, :1])):
        with pytest.raises(NotImplementedError):
            torch.func.vmap(f)(ids[:, 0].expand(2, 4))


@pytest.mark.gpu
def test_lazily_negated_views():
    """Tensors whose sign is still to be applied (the imaginary part of a conjugate): logits, teacher, gradients."""
    from dwarf_v2_b200.distillation import topk_distillation_loss
    from dwarf_v2_b200.logprobs import token_logprobs

    def negated(t):
        z = torch.stack([torch.zeros_like(t), -t], -1)
        view = torch.view_as_complex(z).conj().imag
        assert view.is_neg() and torch.equal(view, t)
        return view, torch._neg_view(-t)  # strided, contiguous

    x = logits(5, 300, "fp32", 9).cuda()
    ids, lp = torch.arange(4).repeat(5, 1).cuda(), torch.full((5, 4), -2.0).cuda()
    g = torch.linspace(0.5, 1.5, 5).cuda()
    want = token_logprobs(x, ids[:, 0], top_k=3)
    kw = dict(reduction="none")
    loss = topk_distillation_loss(x, ids, lp, **kw)
    leaf = x.clone().requires_grad_()
    out, row_loss = token_logprobs(leaf, ids[:, 0], top_k=3), topk_distillation_loss(leaf, ids, lp, **kw)
    gx, = torch.autograd.grad(out.logprob, leaf, g, retain_graph=True)
    gd, = torch.autograd.grad(row_loss, leaf, g, retain_graph=True)
    for i in (0, 1):
        got = token_logprobs(negated(x)[i], ids[:, 0], top_k=3)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(topk_distillation_loss(negated(x)[i], ids, negated(lp)[i], **kw), loss)
        other = negated(x)[i].detach().requires_grad_()
        got, = torch.autograd.grad(token_logprobs(other, ids[:, 0]).logprob, other, negated(g)[i])
        assert torch.equal(got, gx)
        got, = torch.autograd.grad(topk_distillation_loss(other, ids, lp, **kw), other, negated(g)[i])
        assert torch.equal(got, gd)
        got, = torch.autograd.grad(out.logprob, leaf, negated(g)[i], retain_graph=True)
        assert torch.equal(got, gx)
