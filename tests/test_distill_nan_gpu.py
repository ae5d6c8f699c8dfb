"""The gradient of the distillation loss alone: NaN logits show in it, whatever the lse that it is given."""
import math

import pytest
import torch

from raft_b200 import linalg
from test_topk_distill_gpu import TYPES, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [33, 5000, 9001])
def test_gradient_alone_shows_nan_logits(cuda, dtype, vocab):
    logits, ids, teacher, weight = make(5, vocab, 4, dtype, cuda, vocab)
    ids[3] = -1
    logits[0, 1] = -math.inf
    lse = torch.logsumexp(logits.double(), 1).float()
    exp = linalg.topk_distill_grad(logits, ids, teacher, lse, weight)
    assert torch.isfinite(exp).all() and exp[0, 1] <= 0
    bad = torch.zeros((5, vocab), dtype=torch.bool, device=cuda)
    for r, v in ((0, vocab - 1), (1, 0), (1, vocab // 2), (2, int(ids[2, 1])), (3, 5)):
        logits[r, v] = math.nan
        bad[r, v] = True
    got = linalg.topk_distill_grad(logits, ids, teacher, lse, weight)
    bad[3] = False  # a row without a list: 0, whatever it holds
    assert torch.equal(torch.isnan(got), bad)
    assert torch.equal(got[~bad], exp[~bad])
