"""Distillation lists with entries that weigh nothing in fp32: a valid entry far below the list's largest has a finite
log weight and a weight of 0, and adds nothing - as if it were not listed - whatever the student's logit is."""
import math

import pytest
import torch

from raft_b200 import linalg
from test_topk_distill_gpu import TYPES, assert_all, make

pytestmark = pytest.mark.gpu


# loss: one CTA of either size, rows split over a cluster; step: CTAs of each size, clusters, rows read twice (long rows,
# long lists)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k", [(3, 400, 8), (3, 3000, 8), (5, 20000, 40), (3, 131072, 64), (2, 300007, 20),
                                          (2, 5000, 900)])
def test_entries_without_weight_on_masked_logits(cuda, dtype, rows, vocab, k):
    logits, _, teacher, weight = make(rows, vocab, k, dtype, cuda, vocab)
    ids = torch.arange(k, device=cuda).repeat(rows, 1) * (vocab // k) + torch.arange(rows, device=cuda)[:, None] % 7
    far = torch.arange(k, device=cuda) % 3 == 1  # exp(-1e4 / 1.3) is 0 in 32 and in 64 bits
    teacher[:, far] = -1e4
    logits.scatter_(1, ids[:, far], -math.inf)
    unlisted = torch.where(far, -1, ids)
    exp = linalg.topk_distill_step(logits, unlisted, teacher, weight, temperature=1.3)
    got = linalg.topk_distill_step(logits, ids, teacher, weight, temperature=1.3)
    alone = linalg.topk_distill(logits, ids, teacher, temperature=1.3)
    grad = linalg.topk_distill_grad(logits, ids, teacher, alone[1], weight, temperature=1.3)
    assert torch.isfinite(exp[0]).all()
    for a, b in zip(got, exp):
        assert torch.equal(a, b)
    assert torch.isfinite(alone[0]).all() and torch.isfinite(grad).all()
    for loss, lse in (got[:2], alone):
        assert_all(logits, ids, teacher, weight, 1.3, loss, lse)


@pytest.mark.parametrize("vocab", [400, 20000, 300007])
def test_entries_without_weight_keep_nan_and_infinite_losses(cuda, vocab):
    """A weight that is not 0 on a masked logit still makes the loss infinite, a NaN still shows."""
    logits, _, teacher, weight = make(3, vocab, 6, torch.float32, cuda, 1)
    ids = torch.arange(6, device=cuda).repeat(3, 1) * 50
    teacher[:, 5] = -1e4
    logits[:, ids[0, 5]] = -math.inf
    logits[0, ids[0, 2]] = -math.inf
    teacher[1, 1] = math.nan
    for loss, *_ in (linalg.topk_distill_step(logits, ids, teacher, weight), linalg.topk_distill(logits, ids, teacher)):
        assert loss[0] == math.inf and torch.isnan(loss[1]) and torch.isfinite(loss[2])
