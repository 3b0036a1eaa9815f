"""The vocabulary-row operators on the model, as they are used: scoring a batch, the alternatives of a
decoding step, and a distillation step from a teacher's scores."""

import math

import pytest
import torch

from oracle import vocab as oracle
from test_distillation import tolerances
from test_logprobs import check_forward, close, rel_of


def _model(**kw):
    from dwarf_v2_b200.model import DwarfForCausalLM

    return DwarfForCausalLM(**kw).to(torch.bfloat16)


def test_forward_logprobs_refuses_cpu_ids():
    with pytest.raises(RuntimeError):
        _model().eval().forward_logprobs(torch.zeros(1, 4, dtype=torch.int64))


@pytest.mark.gpu
@torch.no_grad()
def test_forward_logprobs_matches_logits():
    """1400 rows: two pieces, the second not whole."""
    from dwarf_v2_b200.logprobs import TokenLogprobs

    model = _model(kv_cache="q6").eval().cuda()
    g = torch.Generator().manual_seed(5)
    batch = torch.randint(57, 32768, (2, 701), generator=g).cuda()
    ids, labels = batch[:, :-1], batch[:, 1:].clone()
    labels[0, :7] = -100
    out = model.forward_logprobs(ids, labels, top_k=20, temperature=0.8)
    assert out.logprob.shape == (2, 700) and out.top_ids.shape == (2, 700, 20)
    logits = model(ids)
    check_forward(out, logits, labels, 20, 0.8)
    none = model.forward_logprobs(ids)
    assert none.logprob is None and none.top_ids is None
    lse, argmax, loss = model.forward_lse(ids, labels)
    close(none.lse, lse, rel_of(32768) * 2 + 2.0 ** -22 * lse.abs().double().cpu())  # two kernels' sums
    one = model.forward_logprobs(ids, labels, top_k=1)
    assert torch.equal(one.top_ids[..., 0], argmax)
    close(-one.logprob, loss, rel_of(32768) * 2 + 2.0 ** -21 * loss.abs().double().cpu())
    assert isinstance(out, TokenLogprobs)
    with pytest.raises(ValueError):
        model.forward_logprobs(ids, labels[:, 1:])
    with pytest.raises(ValueError):
        model.forward_logprobs(ids, labels, top_k=129)
    model.train()
    with pytest.raises(NotImplementedError):
        model.forward_logprobs(ids, labels)


@pytest.mark.gpu
@torch.no_grad()
def test_alternatives_of_decoding_steps():
    """Greedy decoding reads its token and the reported alternatives from one call, eager and inside the graph."""
    from dwarf_v2_b200.logprobs import token_logprobs

    model = _model(kv_cache="q6").eval().cuda()
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(57, 32768, (3, 90), generator=g).cuda()
    logits, state = model.prefill(ids, max_len=128)
    graph = model.capture_decode(state)
    static = torch.zeros(3, 32768, dtype=torch.bfloat16, device="cuda")
    capture = torch.cuda.CUDAGraph()
    token_logprobs(static, top_k=5)
    with torch.cuda.graph(capture):
        captured = token_logprobs(static, top_k=5)
    for _ in range(4):
        out = token_logprobs(logits, top_k=5)
        check_forward(out, logits, None, 5, 1.0)
        assert torch.equal(out.top_ids[:, 0], logits.float().argmax(-1))
        static.copy_(logits)
        capture.replay()
        assert torch.equal(captured.top_ids, out.top_ids) and torch.equal(captured.top_logprobs, out.top_logprobs)
        logits = graph.step(out.top_ids[:, 0])


@pytest.mark.gpu
def test_distillation_step():
    """A teacher's scores (no logits kept) train a student: the gradient that reaches the student's logits is the
    formula's, and the parameters get theirs."""
    from dwarf_v2_b200.distillation import topk_distillation_loss
    from dwarf_v2_b200.model import DwarfConfig

    g = torch.Generator().manual_seed(7)
    ids = torch.randint(57, 32768, (2, 256), generator=g).cuda()
    mask = torch.ones(2, 256, dtype=torch.bool)
    mask[1, 200:] = False
    teacher = _model(config=DwarfConfig(init_seed=7)).eval().cuda()
    with torch.no_grad():
        top = teacher.forward_logprobs(ids, top_k=32, temperature=2.0)
    student = _model(config=DwarfConfig(dropout=0.0)).cuda().train()
    logits, aux = student(ids, return_auxiliary=True)
    logits.retain_grad()
    loss = topk_distillation_loss(logits, top.top_ids, top.top_logprobs, temperature=2.0, row_mask=mask.cuda())
    (loss + aux).backward()
    R, V = 512, 32768
    x, up = logits.detach().reshape(R, V), torch.full((R,), 1.0 / int(mask.sum())).cuda()
    flat = (top.top_ids.reshape(R, 32), top.top_logprobs.reshape(R, 32))
    rows, grad, size, loss_size = oracle.topk_distillation(x, *flat, temperature=2.0,
                                                           row_mask=mask.reshape(-1).cuda(), upstream=up)
    loss_tol, grad_tol = tolerances(x, *flat, 2.0, loss_size, grad, size, True)
    close(loss.detach(), rows.sum() * up[0].double(), (loss_tol.sum() * up[0].double()).cpu() + 2.0 ** -23)
    close(logits.grad.reshape(R, V), grad, grad_tol)
    assert math.isfinite(float(loss.detach()))
    grads = [p.grad for p in student.parameters() if p.requires_grad]
    # the DSQG blocks' NPCI angles (two in each of nine) are not reached by any loss
    assert sum(v is None for v in grads) == 18 and all(torch.isfinite(v).all() for v in grads if v is not None)
