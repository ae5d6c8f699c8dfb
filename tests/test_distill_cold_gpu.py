"""The gradient of the distillation loss alone where the lse is large beside 1: low temperatures, large logits.

What an fp32 lse allows: lse is off by at most half a step, |lse| 2^-24, and so is each of the three products and sums
of the exponent z / T - lse, whose terms are as large; with that, the exponential and the product with the weight
(8 units) a probability is off by a factor of exp(6 U (|z| / T + |lse|) + 8 U), U = 2^-24. And no probability is above
1, so that no error is above 1 either, however large the exponent's."""
import math

import pytest
import torch

from raft_b200 import linalg
from test_topk_distill_gpu import TYPES, U, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1.0, 0.1, 0.01, 1e-3, 1e-4, 1e-6, 1e-10, 1e-20, 1e-30])
@pytest.mark.parametrize("scale", [0.01, 3.0, 1000.0])
def test_probabilities_at_low_temperatures(cuda, dtype, t, scale):
    vocab = 2000
    logits, ids, teacher, weight = make(8, vocab, 5, dtype, cuda, 1, scale)
    ids[0] = 3  # unlisted tokens' elements are probabilities, times the weight
    logits[1, 7] = -math.inf
    r = reference(logits, ids, teacher, weight, t)
    _, lse = linalg.topk_distill(logits, ids, teacher, temperature=t)
    got = linalg.topk_distill_grad(logits, ids, teacher, lse, weight, temperature=t)
    assert torch.isfinite(got).all()
    f = (t * weight.double()).abs()[:, None]
    exponent = U * (6 * (torch.where(torch.isfinite(r["z"]), r["z"].abs(), 0.0) + r["lse"].abs()[:, None]) + 8)
    off = torch.where(exponent < 1, torch.minimum(r["q"] * torch.expm1(exponent), torch.ones_like(exponent)), 1.0)
    listed = r["spread"] > 0
    tol = f * (off + torch.where(listed, r["spread"] * 1e-4 + 1e-4, 0.0))  # (the teacher's weights are tested elsewhere)
    tol = tol + (r["grad"].abs() + tol) * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == torch.float16 else 1e-37)
    err = (got.double() - r["grad"]).abs()
    # a listed probability at a low temperature: the teacher's softmax is as steep, its errors as large
    unlisted_ok = (err <= tol) | listed
    assert torch.all(unlisted_ok), float((err - tol)[~listed].max())
    assert torch.all(err[listed] <= (f.expand_as(err)[listed] * 2) * (1 + torch.finfo(dtype).eps) + 2.0 ** -25)


@pytest.mark.parametrize("vocab", [100, 9001])
def test_a_row_of_masked_logits_alone(cuda, vocab):
    """No probabilities: NaN from the step and from the gradient alone, in a row that has a list."""
    logits, ids, teacher, weight = make(3, vocab, 4, torch.float32, cuda, 2)
    logits[1:] = -math.inf
    ids[2] = -1
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
    alone = linalg.topk_distill_grad(logits, ids, teacher, lse, weight)
    assert lse[1] == -math.inf and torch.isnan(loss[1])
    for g in (grad, alone):
        assert torch.isnan(g[1]).all() and torch.isfinite(g[0]).all() and torch.all(g[2] == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1.0, 0.7])
def test_infinite_logits_show(cuda, dtype, t):
    """Also beside an lse that is not theirs: no probability that looks like one."""
    logits, ids, teacher, weight = make(3, 3001, 4, dtype, cuda, 2)
    lse = torch.logsumexp(logits.double() / t, 1).float()
    exp = linalg.topk_distill_grad(logits, ids, teacher, lse, weight, temperature=t)
    for v in (0, 77, 3000):
        logits[1, v] = math.inf
    got = linalg.topk_distill_grad(logits, ids, teacher, lse, weight, temperature=t)
    bad = torch.isposinf(logits)
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], exp[~bad])
