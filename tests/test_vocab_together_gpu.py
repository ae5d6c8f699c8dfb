"""The vocabulary operators as a program uses them: lookup, a tied projection, distillation loss and gradient, the
gradient of the lookup added to the projection's, an update, and tokens drawn from the result and looked up again.

The projections between the operators are computed in 64 bits and rounded once to fp32 (u = 2^-24 of the value), and
the lookup's scale is a power of two, so that its rows are exact. What is left to count, for a gradient g of a logit
with f = |T weight|: the operator's own error and that of the logits' rounding (2 u |z| of a softmax probability q),
together at most f (q + p) C with C below; from there on the errors pass through sums of absolute values, each
rounding adding u of its value and each sum of n terms n u of theirs."""
import math

import pytest
import torch

from raft_b200 import linalg
from test_sample_tokens_gpu import check as check_sample
from test_topk_distill_gpu import U, reference, sum_error

pytestmark = pytest.mark.gpu

VOCAB, COLS, K, T, SCALE = 1003, 72, 12, 2.0, 8.0


def program(device, n, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    table = torch.randn((VOCAB, COLS), generator=gen, device=device) * 0.05
    tokens = torch.randint(-1, VOCAB, (n,), generator=gen, device=device)
    tokens[n // 2:] = tokens[: n - n // 2].clone()  # every token of the first half again
    ids = torch.randint(-1, VOCAB, (n, K), generator=gen, device=device)
    teacher = torch.randn((n, K), generator=gen, device=device) * 2.0
    weight = torch.rand(n, generator=gen, device=device) / n
    return table, tokens, ids, teacher, weight


def project(a, b):
    return (a.double() @ b.double()).float()


def step(table, tokens, ids, teacher, weight):
    h = linalg.embedding_lookup(table, tokens, scale=SCALE)
    logits = project(h, table.T)
    loss, lse, g = linalg.topk_distill_step(logits, ids, teacher, weight, temperature=T)
    grad_table = project(g.T, h)
    linalg.embedding_grad(project(g, table), tokens, VOCAB, scale=SCALE, grad_table=grad_table, accumulate=True)
    return h, logits, loss, lse, g, grad_table


def rows_of(values, tokens):
    """Sums of the rows of `values` by token, 64 bits."""
    out = torch.zeros((VOCAB + 1, values.shape[1]), dtype=torch.float64, device=values.device)
    return out.index_add_(0, torch.where(tokens >= 0, tokens, VOCAB), values)[:VOCAB]


@pytest.mark.parametrize("n", [1, 2, 64, 1500])
def test_a_training_step_has_the_gradient_of_its_loss(cuda, n):
    table, tokens, ids, teacher, weight = program(cuda, n, n)
    h, logits, loss, lse, g, got = step(table, tokens, ids, teacher, weight)
    # the same in 64 bits, by differentiation
    leaf = table.double().requires_grad_()
    hd = torch.where(tokens[:, None] >= 0, SCALE * leaf[tokens.clamp(min=0)], 0.0)
    z = hd @ leaf.T / T
    logq = torch.log_softmax(z, 1)
    y = torch.where(ids >= 0, teacher.double() / T, -math.inf)
    some = (ids >= 0).any(1)
    logp = torch.log_softmax(torch.where(some[:, None], y, 0.0), 1)
    p = torch.where(some[:, None] & (ids >= 0), logp.exp(), 0.0)
    each = torch.where(p > 0, p * (torch.where(p > 0, logp, 0.0) - logq.gather(1, ids.clamp(min=0))), 0.0)
    exp_loss = T * T * each.sum(1)
    (exp_loss * weight.double()).sum().backward()
    # errors
    r = reference(logits, ids, teacher, weight, T)
    f = (T * weight.double()).abs()[:, None]
    z_max, lse_max = float(r["z"].abs().max()), float(r["lse"].abs().max())
    span = float(teacher.abs().max()) * 2 / T + 8
    c = sum_error(VOCAB) + U * (4 * (z_max + lse_max) + 4 * lse_max + 8) + U * (3 * span + 12 + K) + 2 * U * z_max * T
    eg = f * (r["q"] + r["spread"]) * (c + 4 * U)
    assert torch.all((g.double() - r["grad"]).abs() <= eg)
    t64, h64 = table.double().abs(), h.double().abs()
    dh = (g.double().abs() + eg) @ t64
    eh = eg @ t64 + U * dh
    base = (g.double().abs() + eg).T @ h64
    tol = eg.T @ h64 + U * base + SCALE * rows_of(eh, tokens) + (n + 4) * U * (base + SCALE * rows_of(dh, tokens))
    err = (got.double() - leaf.grad).abs()
    assert torch.all(err <= tol + 1e-37), float((err - tol).max())
    # loss: its own error and the logits' (at most u |z| T / T each, in the listed tokens and in the lse)
    el = T * T * (p * (c + 4 * U * (logp.abs().nan_to_num(posinf=0.0) + logq.gather(1, ids.clamp(min=0)).abs() + 1))).sum(1)
    el = el + T * T * U * (3 * span + 8 + K) * (p * (logp.abs().nan_to_num(posinf=0.0) + z_max + lse_max + 1)).sum(1)
    assert torch.all((loss.double() - exp_loss).abs() <= el + 4 * U * exp_loss.abs() + 1e-30)


@pytest.mark.parametrize("n", [3, 1500])
def test_a_step_and_the_tokens_behind_it_in_one_graph(cuda, n):
    table, tokens, ids, teacher, weight = program(cuda, n, 7)
    gen = torch.Generator(device=cuda).manual_seed(8)
    uniform = torch.rand(n, generator=gen, device=cuda)
    top_p = torch.full((n,), 0.9, device=cuda)

    def whole():
        grad = step(table, tokens, ids, teacher, weight)[-1]
        new = table - 3.0 * grad
        drawn = tokens
        out = []
        for _ in range(3):  # decode: what was drawn is looked up
            logits = project(linalg.embedding_lookup(new, drawn, scale=SCALE), new.T)
            drawn, lp = linalg.sample_tokens(logits, uniform, 0.7, 50, top_p, 0.01)
            out += [logits, drawn, lp]
        return out
    eager = whole()
    for logits, drawn, lp in zip(eager[::3], eager[1::3], eager[2::3]):
        got, got_lp = check_sample(logits, uniform, 0.7, 50, top_p, 0.01)
        assert torch.equal(got, drawn) and torch.equal(got_lp, lp)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        whole()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = whole()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(eager, captured):
        assert torch.equal(a, b)
    # other inputs in the same places
    tokens.copy_(tokens.flip(0))
    ids.copy_(ids.roll(1, 1))
    again = whole()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(again, captured):
        assert torch.equal(a, b)


def test_calls_at_once_on_two_streams_from_two_threads(cuda):
    """Scratch, status words and launch records are shared: each thread's results have to be those it gets alone."""
    import threading
    sets = [program(cuda, n, n) for n in (900, 1500)]
    uniforms = [torch.rand(s[1].numel(), device=cuda) for s in sets]

    def once(s, u):
        out = step(*s)
        return [*out, *linalg.sample_tokens(out[1], u, 0.9, 0, 0.95, 0.0)]
    alone = [once(s, u) for s, u in zip(sets, uniforms)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = once(sets[i], uniforms[i])
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, alone[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    assert linalg.last_kernel_status(cuda) == 0


def test_outputs_over_inputs_are_refused(cuda):
    logits = torch.randn((6, 50), device=cuda)
    ids = torch.zeros((6, 6), dtype=torch.int64, device=cuda)
    teacher, weight = torch.zeros((6, 6), device=cuda), torch.ones(6, device=cuda)
    lse, both = torch.zeros(6, device=cuda), torch.zeros(6, device=cuda)
    for kw in (dict(loss=weight), dict(lse=weight), dict(loss=both, lse=both), dict(loss=logits[0, :6]),
               dict(lse=teacher[0]), dict(loss=logits[0, :6], grad=logits)):
        with pytest.raises(ValueError):
            linalg.topk_distill_step(logits, ids, teacher, weight, **kw)
    square = torch.randn((6, 6), device=cuda)
    with pytest.raises(ValueError):
        linalg.topk_distill_step(square, ids, teacher, weight, grad=teacher)
    with pytest.raises(ValueError):
        linalg.topk_distill_grad(square, ids, teacher, lse, weight, grad=teacher)
    uniform = torch.rand(6, device=cuda)
    for kw in (dict(logprobs=uniform), dict(logprobs=logits[0, :6]), dict(temperature=both, logprobs=both),
               dict(out=both.view(torch.int32), logprobs=both)):
        with pytest.raises(ValueError):
            linalg.sample_tokens(logits, uniform, **kw)
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight, loss=both, lse=lse, grad=logits)
    assert grad is logits and loss is both
