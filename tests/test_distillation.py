"""Distillation from a teacher's listed log probabilities against the 64-bit oracle (oracle/vocab.py).

Tolerances. ``rel`` bounds a sum of exponentials as in test_logprobs.py. A loss is a sum of at most k + 1 terms
p (log p - log q): p is off by 2^-22 + |log p| 2^-23 relative, log p and log q by rel and two roundings of
their size, so the loss by ``(4 rel + (k + 8) 2^-24)`` times the sum of the magnitudes of its terms, each taken
with 1 + |log p| <= 24, plus rel for the logarithms themselves (sum p <= 1). p_* = 1 - sum p is off by 2^-22
absolute, which its logarithm turns into 2^-22 (1 + |log p_* - log q_*|): p_* log p_* moves by that much.
Gradients are held entry by entry to that share of the magnitudes of their terms plus one rounding (eps / 2);
an entry below 2^-126 of the row's maximum may be left without its share of the rest, 2^-86 of it.
"""

import math

import pytest
import torch

from oracle import vocab as oracle
from test_logprobs import TYPES, close, logits, rel_of


def teacher(R, V, k, seed, mass=0.9):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(R)])
    raw = torch.randn(R, k, generator=g) * 1.5
    return ids.cuda(), (torch.log_softmax(raw, -1) + math.log(mass)).cuda()


def tolerances(x, ids, lp, t, loss_size, grad, size, tail):
    V, k = x.shape[-1], ids.shape[-1]
    rel = rel_of(V)
    share = 4 * rel + (k + 32) * 2.0 ** -24
    loss_tol = torch.nan_to_num(loss_size) * share + 2 * rel + (2.0 ** -18 if tail else 0.0)
    d = torch.nan_to_num((x.double() - x.double().amax(-1, keepdim=True)) / t, neginf=0.0).abs()
    tiny = 2.0 ** -24 if x.dtype == torch.float16 else 2.0 ** -86
    grad_tol = (torch.nan_to_num(size) * (2 * share + d * 2.0 ** -21)
                + torch.finfo(x.dtype).eps / 2 * torch.nan_to_num(grad).abs() * 1.01 + tiny)
    return loss_tol, grad_tol


def check(x, ids, lp, *, t=1.0, tail=True, row_mask=None, upstream=None):
    """The per-row loss and its gradient, the reduced losses and theirs."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    R, V = x.shape
    up = torch.ones(R, device=x.device) if upstream is None else upstream
    want, grad, size, loss_size = oracle.topk_distillation(x, ids, lp, temperature=t, tail=tail, row_mask=row_mask,
                                                           upstream=up)
    loss_tol, grad_tol = tolerances(x, ids, lp, t, loss_size, grad, size, tail)
    leaf = x.detach().clone().requires_grad_()
    kw = dict(temperature=t, tail=tail, row_mask=row_mask)
    loss = topk_distillation_loss(leaf, ids, lp, reduction="none", **kw)
    close(loss.detach(), want, loss_tol, "loss")
    got, = torch.autograd.grad(loss, leaf, up)
    close(got, grad, grad_tol, "grad of rows")
    with torch.no_grad():
        assert torch.equal(topk_distillation_loss(leaf, ids, lp, reduction="none", **kw).nan_to_num(), loss.nan_to_num())
    count = R if row_mask is None else max(1, int(row_mask.sum()))
    ones, g1, s1, _ = oracle.topk_distillation(x, ids, lp, temperature=t, tail=tail, row_mask=row_mask)
    for reduction, n in (("sum", 1), ("mean", count)):
        total = topk_distillation_loss(leaf, ids, lp, reduction=reduction, **kw)
        assert total.shape == ()
        close(total.detach(), ones.sum() / n, loss_tol.sum() / n + 2.0 ** -23 * torch.nan_to_num(ones).sum().abs() / n,
              reduction)
        for up1 in (1.0, 0.37):
            got, = torch.autograd.grad(total, leaf, torch.tensor(up1, device=x.device), retain_graph=True)
            f = up1 / n
            _, tol = tolerances(x, ids, lp, t, loss_size, g1 * f, s1 * f, tail)
            close(got, g1 * f, tol, (reduction, up1))


# ------------------------------------------------------------------ CPU


@pytest.mark.parametrize("tail", [True, False])
def test_oracle_gradient_against_differences(tail):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 9, generator=g, dtype=torch.float64)
    ids = torch.tensor([[0, 4, 4], [8, -1, 2], [-1, -1, -1]])
    lp = torch.log(torch.tensor([[0.2, 0.3, 0.1], [0.5, 0.9, 0.2], [0.1, 0.1, 0.1]], dtype=torch.float64))
    loss, grad, _, _ = oracle.topk_distillation(x, ids, lp, temperature=1.4, tail=tail)
    assert loss[2] == 0 and (loss[:2] > 0).all()
    for i in range(3):
        for v in range(9):
            step = torch.zeros_like(x)
            step[i, v] = 1e-5
            hi = oracle.topk_distillation(x + step, ids, lp, temperature=1.4, tail=tail)[0].sum()
            lo = oracle.topk_distillation(x - step, ids, lp, temperature=1.4, tail=tail)[0].sum()
            assert abs((hi - lo) / 2e-5 - grad[i, v]) < 1e-8


def test_oracle_full_list_is_the_divergence():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 7, generator=g, dtype=torch.float64)
    lp = torch.log_softmax(torch.randn(2, 7, generator=g, dtype=torch.float64), -1)
    ids = torch.arange(7).expand(2, 7)
    want = torch.nn.functional.kl_div(torch.log_softmax(x, -1), lp, log_target=True, reduction="none").sum(-1)
    for tail in (True, False):
        torch.testing.assert_close(oracle.topk_distillation(x, ids, lp, tail=tail)[0], want)


def test_refuses_what_it_does_not_take():
    from dwarf_v2_b200.distillation import TopKDistillationLoss, topk_distillation_loss

    x, ids, lp = torch.zeros(4, 10), torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    with pytest.raises(RuntimeError):
        topk_distillation_loss(x, ids, lp)
    with pytest.raises(RuntimeError):
        TopKDistillationLoss()(x, ids, lp)
    with pytest.raises(ValueError):
        topk_distillation_loss(x, ids, lp, reduction="avg")
    with pytest.raises(TypeError):
        topk_distillation_loss(x.double(), ids, lp)
    with pytest.raises(TypeError):
        topk_distillation_loss(x, ids.float(), lp)
    with pytest.raises(TypeError):
        topk_distillation_loss(x, ids, ids)
    with pytest.raises(ValueError):
        topk_distillation_loss(x, ids[:3], lp)
    with pytest.raises(ValueError):
        topk_distillation_loss(x, ids, lp[:, :2])
    with pytest.raises(ValueError):
        topk_distillation_loss(x, ids[:, :0], lp[:, :0])
    with pytest.raises(ValueError):
        topk_distillation_loss(x, torch.zeros(4, 129, dtype=torch.int64), torch.zeros(4, 129))
    with pytest.raises(TypeError):
        topk_distillation_loss(x, ids, lp, row_mask=torch.ones(4))
    with pytest.raises(ValueError):
        topk_distillation_loss(x, ids, lp, row_mask=torch.ones(3, dtype=torch.bool))
    with pytest.raises(NotImplementedError):
        topk_distillation_loss(x, ids, lp.requires_grad_())
    for bad in (0.0, -2.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            topk_distillation_loss(x, ids, lp.detach(), temperature=bad)
    for bad in (math.nan, math.inf):
        with pytest.raises(ValueError):
            topk_distillation_loss(x, ids, lp.detach(), weight=bad)


def test_c_entry_refuses_bad_arguments():
    import ctypes

    from dwarf_v2_b200 import _lib

    lib = _lib.load()

    def status(**fields):
        base = dict(version=_lib.ABI_VERSION, dtype=1, logits=4096, outer=1, inner=2, vocab=64, so=0, si=64,
                    inv_temperature=1.0, k=4, teacher_ids=4096, teacher_logprobs=4096, loss=4096, loss_scale=1.0,
                    scale=1.0)
        return lib.dwarf_topk_distill(ctypes.byref(_lib.TopkDistillArgs(**{**base, **fields})), None)

    assert lib.dwarf_topk_distill(None, None) == -2
    assert status(version=3) == -1
    assert status(teacher_ids=None) == -2 and status(teacher_logprobs=None) == -2 and status(loss=None) == -2
    assert status(k=0) == -3 and status(k=129) == -3 and status(vocab=0) == -3
    assert status(si=-1) == -4 and status(logits=4097) == -5 and status(dtype=9) == -6
    assert status(tail=2) == -9 and status(grad_rows_stride=2) == -9
    assert status(skip_if_one=1, loss=None, grad=4096) == -9
    assert status(skip_if_one=1, grad=4096, grad_rows=4096) == -9
    assert status(loss=None, grad=4096) == -2 and status(stats=4104) == -5
    assert status(inner=0) == 0
    reduce = lambda **f: lib.dwarf_row_reduce(ctypes.byref(_lib.RowReduceArgs(version=1, **f)), None)  # noqa: E731
    assert reduce(rows=-1, out=4096) == -3
    assert reduce(rows=3, out=4096) == -2 and reduce(rows=3, values=4096) == -2


# ------------------------------------------------------------------ GPU


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 1), (4, 33, 7), (2, 128, 128), (5, 1000, 100), (3, 32768, 64),
                                   (1, 32768, 20), (2, 50001, 33), (1, 131075, 128), (300, 515, 8), (2, 300001, 5),
                                   (600, 2052, 16), (2700, 700, 100), (2700, 4001, 9), (2700, 40, 40)])
def test_loss_and_gradient(R, V, k, tail, dtype):
    x = logits(R, V, dtype, R * 3 + V + k).cuda()
    # the whole vocabulary listed: the list is the teacher's whole distribution
    ids, lp = teacher(R, V, k, V + k, mass=1.0 if k == V else 0.9)
    g = torch.Generator().manual_seed(5)
    up = (torch.randn(R, generator=g) * (64 if dtype == "fp16" else 1)).cuda()
    check(x, ids, lp, t=1.5, tail=tail, upstream=up)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("V", [40, 4100, 33000])
def test_unused_slots_masks_and_repeated_ids(V, tail):
    x = logits(10, V, "bf16", 7)
    x[3] = math.nan                       # masked rows hold anything
    x[4] = math.inf
    x[5] = math.nan                       # a row without a used slot
    x = x.cuda()
    ids, lp = teacher(10, V, 12, 3)
    ids[0, 5:] = -1
    ids[1, ::2] = -7
    ids[2, 3] = ids[2, 8]                 # one id twice
    ids[6, :] = ids[6, 0]                 # one id in every slot
    ids[5] = -1
    lp[7, 4:] = -math.inf                 # a teacher that gives nothing to most of its list
    lp[0, 7] = math.nan                   # in an unused slot
    mask = torch.ones(10, dtype=torch.bool)
    mask[3:5] = False
    check(x, ids, lp, tail=tail, row_mask=mask.cuda(), upstream=torch.arange(1.0, 11.0).cuda())
    if V <= 4100:  # the same among many rows
        check(x.repeat(270, 1), ids.repeat(270, 1), lp.repeat(270, 1), tail=tail, row_mask=mask.cuda().repeat(270),
              upstream=torch.arange(1.0, 11.0).cuda().repeat(270))


@pytest.mark.gpu
def test_no_row_counts():
    from dwarf_v2_b200.distillation import topk_distillation_loss

    x = torch.full((3, 50), math.nan, device="cuda", requires_grad=True)
    ids, lp = teacher(3, 50, 4, 0)
    loss = topk_distillation_loss(x, ids, lp, row_mask=torch.zeros(3, dtype=torch.bool, device="cuda"))
    loss.backward()
    assert loss.item() == 0.0 and torch.equal(x.grad, torch.zeros_like(x))
    empty = torch.zeros(0, 50, device="cuda", requires_grad=True)
    for reduction in ("mean", "sum"):
        loss = topk_distillation_loss(empty, ids[:0], lp[:0], reduction=reduction)
        assert loss.item() == 0.0 and torch.autograd.grad(loss, empty)[0].shape == (0, 50)
    assert topk_distillation_loss(empty, ids[:0], lp[:0], reduction="none").shape == (0,)


@pytest.mark.gpu
def test_ids_past_the_vocabulary_are_nan():
    from dwarf_v2_b200.distillation import topk_distillation_loss

    x = logits(3, 50, "fp32", 1).cuda().requires_grad_()
    ids, lp = teacher(3, 50, 4, 0)
    ids[1, 2] = 50
    ids[2, 0] = 1 << 40
    loss = topk_distillation_loss(x, ids, lp, reduction="none")
    assert torch.isfinite(loss[0]) and torch.isnan(loss[1:]).all()
    grad, = torch.autograd.grad(loss, x, torch.ones(3, device="cuda"))
    assert torch.isfinite(grad[0]).all() and torch.isnan(grad[1:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_masked_student(dtype):
    """-inf and the lowest value among the student's logits; a list that holds all the student's mass; a student
    that gives a listed token nothing (the loss is inf, its gradient is not)."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    V = 3000
    x = logits(5, V, dtype, 2)
    ids, lp = teacher(5, V, 6, 1)
    host = ids.cpu()
    x[0] = -math.inf
    x[0, host[0]] = torch.arange(6.0).to(x.dtype)   # nothing outside the list: with a tail the loss is inf
    x[1] = torch.finfo(TYPES[dtype]).min
    x[1, host[1]] = torch.arange(6.0).to(x.dtype)
    x[2, ::2] = -math.inf
    x[2, host[2]] = 1.0
    x[3, host[3, 0]] = -math.inf                     # a listed token without mass
    x = x.cuda()
    check(x[2:3], ids[2:3], lp[2:3])
    check(x[4:], ids[4:], lp[4:])
    for row in (0, 1):  # without a tail both are ordinary rows
        check(x[row:row + 1], ids[row:row + 1], lp[row:row + 1], tail=False)
    leaf = x.clone().requires_grad_()
    loss = topk_distillation_loss(leaf, ids, lp, reduction="none")
    assert loss[0] == math.inf and loss[3] == math.inf
    want = oracle.topk_distillation(x[1:2], ids[1:2], lp[1:2])[0]  # a tenth of the lowest value: large, not inf
    assert float(want) > 1e37
    close(loss[1:2].detach(), want, 2.0 ** -20 * want.abs())
    grad, = torch.autograd.grad(loss, leaf, torch.ones(5, device="cuda"))
    assert torch.isfinite(grad[[2, 3, 4]]).all()
    close(grad[3, ids[3, 0]], -torch.exp(lp[3, 0]).double(), 2.0 ** -8 if dtype == "bf16" else 1e-6)


@pytest.mark.gpu
def test_student_that_has_learnt_the_list():
    """Nearly all mass on the list: the rest's share comes from its own sum, not from 1 - sum q."""
    V, k = 32768, 8
    x = torch.full((2, V), -30.0)
    g = torch.Generator().manual_seed(3)
    x += torch.randn(2, V, generator=g)
    ids, _ = teacher(2, V, k, 4)
    x[0, ids[0].cpu()] = torch.randn(k, generator=g)
    x[1, ids[1].cpu()] = torch.randn(k, generator=g) + 5
    lp = torch.log_softmax(torch.randn(2, k, generator=g), -1) + math.log(0.999)
    check(x.cuda(), ids, lp.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,k", [(3, 3000, 9), (2, 40000, 100), (2700, 300, 5), (1, 33001, 3)])
@pytest.mark.parametrize("gap", [40.0, 120.0, 400.0])
def test_rest_far_below_the_list(R, V, k, gap):
    """The list (and one of its ids twice) lies `gap` above all the rest, which exp(-gap) does not hold in
    fp32 from 104 on: the rest's sum has a maximum of its own, so the loss (about the rest's share times the gap) and
    the rest's gradients stay finite and right; a row whose list lies below the rest by as much, too."""
    g = torch.Generator().manual_seed(int(gap) + V)
    x = torch.randn(R, V, generator=g)
    ids, lp = teacher(R, V, k, V, mass=0.8)
    ids[0, 1] = ids[0, 0]
    x.scatter_add_(1, ids.cpu(), torch.full((R, k), gap))
    x[-1] = torch.randn(V, generator=g)
    x[-1, ids[-1].cpu()] -= gap
    for dtype in ("fp32", "bf16"):
        check(x.to(TYPES[dtype]).cuda(), ids, lp)
        check(x.to(TYPES[dtype]).cuda(), ids, lp, t=0.5)


@pytest.mark.gpu
def test_weight_and_second_backward():
    from dwarf_v2_b200.distillation import TopKDistillationLoss, topk_distillation_loss

    x = logits(40, 4096, "bf16", 1).cuda().requires_grad_()
    ids, lp = teacher(40, 4096, 16, 2)
    plain = topk_distillation_loss(x, ids, lp)
    half = TopKDistillationLoss(weight=0.5)(x, ids, lp)
    assert half.item() == plain.item() * 0.5
    g1, = torch.autograd.grad(plain, x, retain_graph=True)
    kept = g1.clone()
    g2, = torch.autograd.grad(plain, x)                      # computed anew, in a buffer of its own
    assert torch.equal(kept, g2) and g1.data_ptr() != g2.data_ptr()
    gh, = torch.autograd.grad(half, x)
    gs, = torch.autograd.grad(topk_distillation_loss(x, ids, lp) * 0.5, x)
    assert torch.equal(gh, gs)                               # one rounding either way
    rows = topk_distillation_loss(x, ids, lp, reduction="none", weight=2.0)
    torch.testing.assert_close(rows.mean(), 2 * plain, rtol=1e-6, atol=0)


@pytest.mark.gpu
def test_strides_types_and_accumulation():
    """logits[:, :-1], int32 ids, bf16 teacher values, two losses into one leaf's gradient."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 6, 1001, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    ids, lp = teacher(15, 1001, 9, 2)
    ids, lp = ids.view(3, 5, 9), lp.view(3, 5, 9).to(torch.bfloat16)
    loss = topk_distillation_loss(x[:, :-1], ids.int(), lp, reduction="none")
    want, grad, size, loss_size = oracle.topk_distillation(x.detach()[:, :-1].reshape(15, -1), ids.view(15, 9),
                                                           lp.view(15, 9).float())
    flat = x.detach()[:, :-1].reshape(15, -1)
    loss_tol, grad_tol = tolerances(flat, ids.view(15, 9), lp, 1.0, loss_size, grad, size, True)
    close(loss.detach().reshape(15), want, loss_tol)
    (loss.sum() + topk_distillation_loss(x[:, :-1], ids, lp, reduction="sum")).backward()
    got = x.grad[:, :-1].reshape(15, -1)
    close(got, 2 * grad, 2 * grad_tol + 2.0 ** -8 * 2 * grad.abs())  # two rounded gradients and their rounded sum
    assert torch.equal(x.grad[:, -1], torch.zeros_like(x.grad[:, -1]))


@pytest.mark.gpu
def test_streams_and_graphs():
    """The captured training step (forward and backward, upstream gradients 1 and 0.25) replays bit-identically."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    x = logits(33, 32768, "bf16", 8).cuda()
    ids, lp = teacher(33, 32768, 64, 2)
    mask = torch.ones(33, dtype=torch.bool, device="cuda")
    mask[4] = False

    def step(v, up):
        leaf = v.detach().requires_grad_()
        loss = topk_distillation_loss(leaf, ids, lp, temperature=2.0, row_mask=mask)
        grad, = torch.autograd.grad(loss * up, leaf)
        return [loss.detach(), grad]

    static = torch.zeros_like(x)
    side = torch.cuda.Stream()
    for up in (1.0, 0.25):
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = step(static, up)
            graphs.append((graph, got))
        for shift in (0, 3):
            static.copy_(x.roll(shift, 1))
            want = step(static, up)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = step(static, up)
            for graph, _ in graphs:
                graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, other))
            for _, got in graphs:
                assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_one_direction_captured(reduction):
    """A captured forward with eager backwards: a gradient handed out stays as it is through later replays. An eager
    forward with a captured backward: each replay writes the gradient, whatever was done to the last one."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    x = logits(33, 4096, "bf16", 8).cuda()
    moved = x.roll(3, 1)
    ids, lp = teacher(33, 4096, 16, 2)
    up = torch.ones(33 if reduction == "none" else (), device="cuda")

    def forward(leaf):
        return topk_distillation_loss(leaf, ids, lp, reduction=reduction)

    def right(got, v):
        f = 1 / 33 if reduction == "mean" else 1.0
        _, want, size, loss_size = oracle.topk_distillation(v, ids, lp)
        close(got, want * f, tolerances(v, ids, lp, 1.0, loss_size, want * f, size * f, True)[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        static = x.clone().requires_grad_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = forward(static)
        graph.replay()
        g1, = torch.autograd.grad(loss, static, up, retain_graph=True)
        right(g1, x)
        kept = g1.clone()
        static.data.copy_(moved)
        graph.replay()
        g2, = torch.autograd.grad(loss, static, up, retain_graph=True)
        right(g2, moved)
        assert torch.equal(g1, kept)

        leaf = x.clone().requires_grad_()
        loss = forward(leaf)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            g3, = torch.autograd.grad(loss, leaf, up, retain_graph=True)  # replays read what forward saved
        for _ in range(2):
            g3.zero_()
            graph.replay()
            right(g3, x)


@pytest.mark.gpu
def test_teacher_to_student():
    """As used: a teacher's top alternatives at a temperature feed the student's loss; equal models give a
    divergence of zero and a gradient of zero, up to the roundings."""
    from dwarf_v2_b200.distillation import topk_distillation_loss
    from dwarf_v2_b200.logprobs import token_logprobs

    t_logits = logits(64, 32768, "bf16", 21).cuda()
    with torch.no_grad():
        top = token_logprobs(t_logits, top_k=64, temperature=2.0)
    student = logits(64, 32768, "bf16", 22).cuda().requires_grad_()
    loss = topk_distillation_loss(student, top.top_ids, top.top_logprobs, temperature=2.0, reduction="none")
    want, grad, size, loss_size = oracle.topk_distillation(student.detach(), top.top_ids, top.top_logprobs,
                                                           temperature=2.0)
    loss_tol, grad_tol = tolerances(student.detach(), top.top_ids, top.top_logprobs, 2.0, loss_size, grad, size, True)
    close(loss.detach(), want, loss_tol)
    got, = torch.autograd.grad(loss, student, torch.ones(64, device="cuda"))
    close(got, grad, grad_tol)
    same = topk_distillation_loss(t_logits, top.top_ids, top.top_logprobs, temperature=2.0, reduction="none")
    assert same.abs().max() < 2.0 ** -16


# ------------------------------------------------------------------ rows whose masks leave nothing to a part of the teacher


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("R,V,k", [(3, 300, 6), (2, 40000, 20), (1, 33001, 3), (2700, 261, 5)])
@pytest.mark.parametrize("shift", [-2000.0, -200.0, 0.0, 200.0])
def test_nothing_outside_the_list(R, V, k, shift, dtype):
    """Every logit outside the list is -inf and the teacher leaves a rest: the loss is inf; the listed entries have
    their gradient and the others exact zeros, wherever the listed values lie."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    ids, lp = teacher(R, V, k, V + k)
    g = torch.Generator().manual_seed(k)
    x = torch.full((R, V), -math.inf).scatter_(1, ids.cpu(), torch.randn(R, k, generator=g) + shift)
    x = x.to(TYPES[dtype]).cuda()
    check(x, ids, lp)
    leaf = x.clone().requires_grad_()
    rows = topk_distillation_loss(leaf, ids, lp, reduction="none")
    assert (rows == math.inf).all()
    for loss in (rows.sum(), topk_distillation_loss(leaf, ids, lp, reduction="sum")):
        for up in (1.0, 0.25):
            grad, = torch.autograd.grad(loss, leaf, torch.tensor(up).cuda(), retain_graph=True)
            assert torch.isfinite(grad).all()
            assert not grad.scatter(1, ids, 0.0).any()


def test_oracle_row_without_a_finite_logit():
    x = torch.full((4, 6), -math.inf)
    x[3] = 0.0
    ids = torch.tensor([[1, 3], [1, -1], [-1, -1], [0, 1]])
    lp = torch.log(torch.tensor([[0.5, 0.2], [0.9, 0.1], [0.3, 0.3], [0.5, 0.25]]))
    for tail in (True, False):
        loss, grad, size, _ = oracle.topk_distillation(x, ids, lp, tail=tail)
        assert loss[:3].tolist() == [math.inf, math.inf, 0.0] and 0 < loss[3] < math.log(6)  # against an even q
        assert not grad[:3].any() and grad[3].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("tail", [True, False])
@pytest.mark.parametrize("R,V,k", [(5, 7, 2), (5, 1000, 6), (5, 40000, 20), (2700, 261, 5), (5, 4, 4)])
def test_rows_without_a_finite_logit(R, V, k, tail, dtype):
    """A counted row whose mask leaves nothing: loss inf, gradient 0; its neighbours are what they are without it,
    and so is the gradient of a reduced loss. An id past the vocabulary or a NaN of the teacher still makes it NaN."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    ids, lp = teacher(R, V, k, V + k, mass=1.0 if k == V else 0.9)
    x = logits(R, V, dtype, V)
    x[1:-1] = -math.inf
    x = x.cuda()
    ids[2, 1:] = -1
    if R > 4:
        ids[3, 0] = V
        lp[R - 2, 1] = math.nan
    check(x, ids, lp, tail=tail, upstream=torch.linspace(0.5, 2.0, R).cuda())
    mask = torch.ones(R, dtype=torch.bool).cuda()
    mask[1:3] = False
    check(x, ids, lp, tail=tail, row_mask=mask)
    leaf = x.clone().requires_grad_()
    good = [0, 1, 2, R - 1]
    loss = topk_distillation_loss(leaf, ids, lp, tail=tail, reduction="none")
    assert (loss[1:3] == math.inf).all() and torch.isfinite(loss[[0, R - 1]]).all()
    assert torch.isnan(loss[3]) and torch.isnan(loss[R - 2])
    grad, = torch.autograd.grad(topk_distillation_loss(leaf, ids, lp, tail=tail, reduction="sum"), leaf)
    assert torch.isfinite(grad[good]).all() and not grad[1:3].any()
    if k < V:  # (with every id listed and learnt there may be nothing to learn)
        assert grad[0].any() and grad[R - 1].any()


def test_oracle_teacher_without_a_value():
    x, ids, lp = torch.zeros(1, 4), torch.tensor([[0, 1]]), torch.full((1, 2), -math.inf)
    loss, grad, _, _ = oracle.topk_distillation(x, ids, lp, tail=False)
    assert torch.isnan(loss).all() and torch.isnan(grad).all()
    loss, grad, _, _ = oracle.topk_distillation(x, ids, lp)  # all of the mass is the rest's
    assert abs(loss.item() - math.log(2)) < 1e-12 and torch.isfinite(grad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 1000, 40000])
def test_teacher_without_a_value(V):
    """A list of -inf alone: all mass is the rest's with a tail, NaN without one; unused slots do not count."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    x = logits(4, V, "fp32", V).cuda()
    ids, lp = torch.arange(2).repeat(4, 1).cuda(), torch.full((4, 2), -1.0).cuda()
    lp[1] = -math.inf
    lp[2, 1] = -math.inf
    ids[2, 0], ids[3, 0] = -1, -1
    check(x, ids, lp, tail=True)
    check(x, ids, lp, tail=False)
    rows = topk_distillation_loss(x, ids, lp, tail=False, reduction="none")
    assert torch.isnan(rows).tolist() == [False, True, True, False]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("V", [13, 1001, 4097])
def test_views_of_logits(V, dtype):
    """Rows of larger tensors, at every offset from the 16-byte boundary: the listed ids' bits, the ends and the
    gradient's rows go by the row's own start."""
    from dwarf_v2_b200.distillation import topk_distillation_loss

    g = torch.Generator().manual_seed(V)
    big = (torch.randn(3, 6, V + 9, generator=g) * 3).to(TYPES[dtype]).cuda()
    views = [big[:, :-1, :V], big[:, 1:, 9:], big[1, :, 1:V + 1], big[:, 2, 3:V + 3], big.transpose(0, 1)[:, :, 5:V + 5],
             big[:, ::2, 7:V + 7], big[:1, :1, 2:V + 2], big[0, 0, :V].expand(5, V), big[:, :, ::2]]
    for view in views:
        n, lead = view.shape[-1], view.shape[:-1]
        flat = view.reshape(-1, n)
        k = min(7, n)
        ids, lp = teacher(len(flat), n, k, V)
        ids[0, :3] = torch.tensor([0, n - 1, n // 2]).cuda()[:3]  # the ends
        up = torch.linspace(0.5, 2.0, len(flat)).cuda()
        want, grad, size, loss_size = oracle.topk_distillation(flat, ids, lp, upstream=up)
        loss_tol, grad_tol = tolerances(flat, ids, lp, 1.0, loss_size, grad, size, True)
        leaf = big.clone().requires_grad_()
        rows = leaf.as_strided(view.shape, view.stride(), view.storage_offset())
        loss = topk_distillation_loss(rows, ids.reshape(*lead, k), lp.reshape(*lead, k), reduction="none")
        close(loss.detach().reshape(-1), want, loss_tol, view.shape)
        got, = torch.autograd.grad(loss, rows, up.reshape(lead))
        close(got.reshape(-1, n), grad, grad_tol, view.shape)
        total = topk_distillation_loss(rows, ids.reshape(*lead, k), lp.reshape(*lead, k), reduction="sum")
        _, grad, size, _ = oracle.topk_distillation(flat, ids, lp)
        _, grad_tol = tolerances(flat, ids, lp, 1.0, loss_size, grad, size, True)
        got, = torch.autograd.grad(total, rows)
        close(got.reshape(-1, n), grad, grad_tol, view.shape)


def test_c_entries_refuse_a_gradient_off_its_elements():
    import ctypes

    from dwarf_v2_b200 import _lib

    lib = _lib.load()
    base = dict(version=_lib.ABI_VERSION, logits=4096, outer=1, inner=2, vocab=64, so=0, si=64, inv_temperature=1.0,
                stats=4096)
    for dtype, off in ((0, 2), (0, 1), (1, 1), (2, 1)):
        args = _lib.TokenLogprobsBwdArgs(**base, dtype=dtype, entropy=4096, grad=4096 + off)
        assert lib.dwarf_token_logprobs_bwd(ctypes.byref(args), None) == -5
        for loss in (None, 4096):
            args = _lib.TopkDistillArgs(**base, dtype=dtype, k=4, teacher_ids=4096, teacher_logprobs=4096, loss=loss,
                                        loss_scale=1.0, scale=1.0, grad=4096 + off)
            assert lib.dwarf_topk_distill(ctypes.byref(args), None) == -5
