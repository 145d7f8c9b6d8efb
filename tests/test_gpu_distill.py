"""Distillation of a teacher's top entries against 64-bit arithmetic and against differences.

Bounds, with z the scores over tau, c_k the teacher's logits over tau, Z and C their largest distances from the maximum among
what carries weight: a shifted logit rounds by 3 roundings of its size, an exponential by 2^-20 of itself, sums over n
by n 2^-24 at most in 32 lanes' order, logarithms and differences by 2^-22 of their size.
"""
import math

import pytest
import torch

from spruce_research_b200 import _lib, native
from spruce_research_b200.selector.loss import teacher_top_blocks, topk_distill_loss

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def want(scores, ids, teacher, visible, tau, weight):
    """Losses and gradients in 64 bits."""
    R, n = scores.shape
    z = scores.double() / tau
    seen = torch.arange(n, device="cuda") < (n if visible is None else visible[:, None])
    z = z.masked_fill(~seen, -math.inf)
    limit = seen.sum(-1, keepdim=True) if visible is not None else torch.full((R, 1), n, device="cuda")
    use = (ids >= 0) & (ids < limit)
    t = (teacher.double() / tau).masked_fill(~use, -math.inf)
    empty = (z.amax(-1) == -math.inf) if n else torch.ones(R, device="cuda", dtype=torch.bool)
    empty = empty | ((t.amax(-1) == -math.inf) if t.shape[1] else True)
    p = torch.softmax(t, -1).nan_to_num(0.0)
    log_q = torch.log_softmax(z, -1)
    at = ids.long().clamp(0, max(n - 1, 0))
    terms = p * (torch.log(p) - log_q.gather(-1, at)) if n else torch.zeros_like(p)
    loss = torch.where(use & (p > 0), terms, 0.0).sum(-1)
    target = torch.zeros_like(z).scatter_add_(-1, at, torch.where(use, p, 0.0)) if n else z
    grad = (log_q.exp() - target) * (weight.double() / tau)[:, None]
    return torch.where(empty, 0.0, loss), torch.where(empty[:, None], 0.0, grad), log_q, p


def make(R, n, K, dtype, causal=False, seed=0, ids_type=torch.int32, teacher_type=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    scores = (2 * torch.randn(R, n, generator=g, device="cuda")).to(dtype)
    visible = torch.randint(0, n + 1, (R,), generator=g, device="cuda", dtype=torch.int32) if causal else None
    t = 0.7 * scores.float() + torch.randn(R, n, generator=g, device="cuda")
    if causal:
        t = t.masked_fill(torch.arange(n, device="cuda") >= visible[:, None], -math.inf)
    best, ids = t.topk(min(K, n), -1)
    ids = ids.masked_fill(best == -math.inf, -1).to(ids_type)
    best = best.masked_fill(best == -math.inf, 0.0).to(teacher_type)
    return scores, ids, best, visible, 0.5 + torch.rand(R, generator=g, device="cuda")


def check(scores, ids, teacher, visible, weight, tau=1.0):
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    kw = dict(visible=visible, temperature=tau, status=status)
    loss, grad = native.topk_distill(scores, ids, teacher, grad_weight=weight, **kw)
    alone = native.topk_distill(scores, ids, teacher, **kw)
    x = scores.detach().clone().requires_grad_()
    recorded = topk_distill_loss(x, ids, teacher, **kw)
    by_autograd, = torch.autograd.grad(recorded, x, weight)
    assert status.item() == 0
    wl, wg, log_q, p = want(scores, ids, teacher, visible, tau, weight)
    u, n = torch.finfo(scores.dtype).eps / 2, scores.shape[1]
    size = (scores.double().abs().nan_to_num(posinf=0, neginf=0).amax() if n else 0) / tau
    far = 16 * 2.0 ** -24 * (2 * size + 2 * teacher.double().abs().nan_to_num(posinf=0).amax().item() / tau + 40) + 2.0 ** -19 + n * 2.0 ** -24 / 32
    for got in (loss, alone, recorded):
        assert got.dtype == torch.float32 and ((got - wl).abs() <= far).all(), (got - wl).abs().max()
    q = log_q.exp().nan_to_num(0.0)
    mass = torch.zeros_like(q).scatter_add_(-1, ids.long().clamp(0, max(n - 1, 0)), torch.where(ids >= 0, p, 0.0))
    bound = u * wg.abs() + (1 + u) * far * (q + mass) * (weight.double() / tau)[:, None] + 2.0 ** -126 + (
        2.0 ** -25 if scores.dtype == torch.float16 else 0.0)
    for got in (grad, by_autograd):
        assert got.dtype == scores.dtype and ((got.double() - wg).abs() <= bound).all(), (
            (got.double() - wg).abs() / bound).max()
    return loss, grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, K", [(1, 1), (2, 2), (7, 3), (31, 8), (64, 64), (129, 16), (512, 27), (2048, 200), (2049, 5),
                                  (5003, 33), (40001, 1)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("tau", [1.0, 0.5, 3.0])
def test_losses_and_gradients(dtype, n, K, causal, tau):
    check(*make(37, n, K, dtype, causal, seed=n), tau=tau)


@pytest.mark.parametrize("ids_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("teacher_type", DTYPES)
def test_types_of_the_teacher(ids_type, teacher_type):
    check(*make(9, 300, 20, torch.bfloat16, True, ids_type=ids_type, teacher_type=teacher_type))


@pytest.mark.parametrize("R, n", [(1, 131072), (3, 100003), (5000, 40), (300, 1030)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_from_few_long_to_many_short(R, n, dtype):
    check(*make(R, n, 64, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [50, 700])
def test_strided_rows_and_more_dimensions(dtype, n):
    scores, ids, teacher, visible, weight = make(24, n, 6, dtype, True)
    loss, grad = check(scores, ids, teacher, visible, weight)
    wide = torch.full((24, n + 11), math.nan, device="cuda", dtype=dtype)
    wide[:, 5:5 + n] = scores
    w = weight.view(4, 6).T.contiguous().T
    got = native.topk_distill(wide[:, 5:5 + n].view(4, 6, n), ids.view(4, 6, -1), teacher.view(4, 6, -1),
                              visible=visible.view(4, 6), grad_weight=w)
    assert got[0].shape == (4, 6) and torch.equal(got[0].flatten(), loss)
    # Columns of another alignment may be summed in another order.
    assert got[1].shape == (4, 6, n) and (got[1].flatten(0, 1).float() - grad.float()).abs().max() <= 2e-2 * grad.float().abs().max()
    one = native.topk_distill(scores[0], ids[0], teacher[0], visible=visible[0])
    assert one.shape == () and torch.equal(one, loss[0])
    same = native.topk_distill(scores[:1].expand(5, -1), ids[:1].expand(5, -1), teacher[:1].expand(5, -1),
                               visible=visible[:1].expand(5), grad_weight=weight[:1].expand(5))
    assert torch.equal(same[0], loss[:1].expand(5)) and torch.equal(same[1], grad[:1].expand(5, -1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [20, 900])
def test_rows_that_teach_nothing(dtype, n):
    """No teacher entry, none above -inf, no visible column, none above -inf: loss and gradient 0."""
    scores, ids, teacher, _, weight = make(6, n, 4, dtype)
    visible = torch.full((6,), n, device="cuda", dtype=torch.int32)
    ids[0] = -1
    teacher[1] = -math.inf
    visible[2], ids[2] = 0, -1
    scores[3] = -math.inf
    teacher[4, 1:] = -math.inf
    loss, grad = check(scores, ids, teacher, visible, weight)
    assert (loss[:4] == 0).all() and (grad[:4] == 0).all() and loss[4] > 0
    loss, grad = native.topk_distill(scores, ids[:, :0], teacher[:, :0], grad_weight=weight)
    assert (loss == 0).all() and (grad == 0).all()
    assert native.topk_distill(scores[:, :0], ids, teacher.zero_()).shape == (6,)
    assert native.topk_distill(scores[:0], ids[:0], teacher[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [40, 3000])
def test_masked_and_lowest_scores(dtype, n):
    """-inf and the type's lowest value as masks within the visible columns; a row of lowest values alone is flat."""
    scores, ids, teacher, _, weight = make(5, n, 3, dtype)
    low = torch.finfo(dtype).min
    masked = torch.ones(n, device="cuda", dtype=torch.bool)
    masked[ids.long().flatten()] = False
    scores[0, masked] = -math.inf
    scores[1, masked] = low
    scores[2] = low
    loss, grad = native.topk_distill(scores, ids, teacher, grad_weight=weight)
    wl, wg, _, _ = want(scores, ids, teacher, None, 1.0, weight)
    assert torch.allclose(loss.double(), wl, rtol=1e-5, atol=1e-5)
    assert torch.allclose(grad.double(), wg, rtol=2.0 ** -7, atol=1e-6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [40, 3000])
def test_values_that_are_not_numbers_stay_in_their_row(dtype, n):
    scores, ids, teacher, _, weight = make(6, n, 3, dtype)
    clean = native.topk_distill(scores, ids, teacher, grad_weight=weight)
    scores[1, 7], scores[2, 5] = math.nan, math.inf
    teacher[3, 1] = math.nan
    loss, grad = native.topk_distill(scores, ids, teacher, grad_weight=weight)
    assert loss[1:4].isnan().all() and grad[1:3].isnan().all()
    for r in (0, 4, 5):
        assert torch.equal(loss[r], clean[0][r]) and torch.equal(grad[r], clean[1][r])
    visible = torch.full((6,), 5, device="cuda", dtype=torch.int32)      # past the visible columns nothing is read
    ids = ids.clamp(max=4)
    a = native.topk_distill(scores, ids, teacher, visible=visible, grad_weight=weight)
    scores[:, 5:] = math.nan
    b = native.topk_distill(scores, ids, teacher, visible=visible, grad_weight=weight)
    rows = [0, 1, 2, 4, 5]
    assert torch.equal(a[0][rows], b[0][rows]) and torch.equal(a[1][rows], b[1][rows]) and (b[1][:, 5:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [30, 5000])
def test_a_column_named_twice_counts_twice_and_one_outside_not_at_all(dtype, n):
    scores, ids, teacher, _, weight = make(5, n, 6, dtype)
    ids[:, 3] = ids[:, 1]
    ids[:, 4] = ids[:, 1]
    check(scores, ids, teacher, None, weight)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    visible = torch.tensor([n, n, 10, 10, n], device="cuda", dtype=torch.int32)
    ids[:] = torch.arange(6, device="cuda")
    ids[1, 0], ids[2, 2] = n, 10
    kw = dict(visible=visible, grad_weight=weight)
    got = native.topk_distill(scores, ids, teacher, status=status, **kw)
    assert status.item() == _lib.STATUS_BAD_INDEX
    ids[1, 0] = ids[2, 2] = -1
    for a, b in zip(got, native.topk_distill(scores, ids, teacher, **kw)):
        assert torch.equal(a, b)
    status.zero_()
    visible[0], visible[4] = n + 3, -2
    ids[4] = -1
    got = native.topk_distill(scores, ids, teacher, status=status, **kw)
    assert status.item() == _lib.STATUS_BAD_LENGTH
    visible[0], visible[4] = n, 0
    for a, b in zip(got, native.topk_distill(scores, ids, teacher, **kw)):
        assert torch.equal(a, b)


def test_the_most_entries_that_a_teacher_may_have():
    check(*make(3, 4000, 2048, torch.float32))
    scores, ids, teacher, _, weight = make(3, 4000, 2049, torch.float32)
    with pytest.raises(ValueError, match="at most 2048"):
        native.topk_distill(scores, ids, teacher)


def test_the_gradient_against_differences():
    """Central differences of the losses, taken in 64 bits by the plain form: a loss is smooth in its scores."""
    scores, ids, teacher, visible, weight = make(4, 33, 5, torch.float32, True, seed=3)
    _, grad = native.topk_distill(scores, ids, teacher, visible=visible, grad_weight=weight)
    h = 1e-5
    for j in range(33):
        up, down = scores.double(), scores.double()
        up, down = up.clone(), down.clone()
        up[:, j] += h
        down[:, j] -= h
        a = want(up, ids, teacher, visible, 1.0, weight)[0]
        b = want(down, ids, teacher, visible, 1.0, weight)[0]
        slope = (a - b) / (2 * h) * weight
        assert (slope - grad[:, j]).abs().max() <= 1e-6       # h^2 of the third derivative, 1e-16 / h of the difference


def test_backward_in_a_graph_and_on_another_stream():
    scores, ids, teacher, visible, weight = make(50, 900, 9, torch.bfloat16, True)
    want_loss, want_grad = native.topk_distill(scores, ids, teacher, visible=visible, grad_weight=weight)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x = scores.detach().requires_grad_()
    with torch.cuda.stream(side):
        loss = topk_distill_loss(x, ids, teacher, visible=visible)
        grad, = torch.autograd.grad(loss, x, weight)
    side.synchronize()
    assert torch.equal(loss, want_loss) and torch.equal(grad, want_grad)
    loss = grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, stats = native.topk_distill_forward(scores, ids, teacher, visible=visible)
        grad = native.topk_distill_backward(scores, ids, teacher, stats, weight, visible=visible)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, want_loss) and torch.equal(grad, want_grad)


def test_a_second_backward_is_refused():
    scores, ids, teacher, _, _ = make(3, 50, 4, torch.float32)
    x = scores.requires_grad_()
    grad, = torch.autograd.grad(topk_distill_loss(x, ids, teacher).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()


def test_the_top_blocks_of_a_teacher():
    mass = torch.tensor([[1.0, 0.0, 0.0], [0.25, 0.75, 0.0], [0.5, 0.125, 0.375]], device="cuda")
    ids, logits = teacher_top_blocks(mass, 2)
    assert ids.tolist() == [[0, -1], [1, 0], [0, 2]] and ids.dtype == torch.int32
    p = torch.softmax(logits.masked_fill(ids < 0, -math.inf), -1)
    assert torch.allclose(p, torch.tensor([[1.0, 0.0], [0.75, 0.25], [4 / 7, 3 / 7]], device="cuda"))


@pytest.mark.parametrize("n", [131072, 1000])
def test_rows_past_the_32_bit_offset(n):
    """The last rows of more than 2^32 scores give what they give by themselves."""
    R = (1 << 32) // n + 20
    few = make(12, n, 8, torch.bfloat16, seed=4)
    scores = torch.zeros(R, n, device="cuda", dtype=torch.bfloat16)
    ids = torch.full((R, 8), -1, device="cuda", dtype=torch.int32)
    teacher, weight = torch.zeros(R, 8, device="cuda"), torch.ones(R, device="cuda")
    scores[-12:], ids[-12:], teacher[-12:], weight[-12:] = few[0], few[1], few[2], few[4]
    loss, grad = native.topk_distill(scores, ids, teacher, grad_weight=weight)
    alone, alone_grad = native.topk_distill(*few[:3], grad_weight=few[4])
    assert (loss[:-12] == 0).all() and (grad[-20:-12] == 0).all()
    assert (loss[-12:] - alone).abs().max() <= 1e-5 and (grad[-12:].float() - alone_grad.float()).abs().max() <= 2.0 ** -8 * alone_grad.abs().max()


@pytest.mark.parametrize("lead", [(3,), (2, 3), (0,)])
def test_rows_without_columns_have_an_empty_gradient(lead):
    scores = torch.zeros(*lead, 0, device="cuda", requires_grad=True)
    ids, teacher = torch.zeros(*lead, 2, device="cuda", dtype=torch.int32), torch.zeros(*lead, 2, device="cuda")
    loss = topk_distill_loss(scores, ids, teacher)
    loss.sum().backward()
    assert loss.shape == lead and (loss == 0).all() and scores.grad.shape == scores.shape
    loss, grad = native.topk_distill(scores.detach(), ids, teacher, grad_weight=torch.ones(lead, device="cuda"))
    assert (loss == 0).all() and grad.shape == scores.shape
