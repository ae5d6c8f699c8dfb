"""Logits whose rows are far apart: the gradient that is allocated takes the memory of its rows."""
import pytest
import torch

from raft_b200 import linalg
from test_topk_distill_gpu import TYPES, assert_all, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1003, 20003])
@pytest.mark.parametrize("length", [3, 100])
def test_last_positions_of_sequences(cuda, dtype, vocab, length):
    logits, ids, teacher, weight = make(6, vocab, 9, dtype, cuda, 5)
    every = torch.full((6, length, vocab), 50.0, device=cuda).to(dtype)
    every[:, -1] = logits
    last = every[:, -1]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss, lse, grad = linalg.topk_distill_step(last, ids, teacher, weight)
    assert torch.cuda.max_memory_allocated() - before < 2 * 6 * vocab * grad.element_size() + 4096
    assert_all(logits, ids, teacher, weight, 1.0, loss, lse, grad)
    grad = linalg.topk_distill_grad(last, ids, teacher, lse, weight)
    assert_all(logits, ids, teacher, weight, 1.0, grad=grad)
    assert torch.equal(every[:, -1], logits)
