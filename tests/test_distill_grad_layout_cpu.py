"""The gradient that the distillation calls allocate: rows at the alignment of the logits' rows, no more memory than
that takes. Host code alone, no GPU needed."""
import pytest
import torch

from raft_b200 import linalg


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 7, 96, 1003])
@pytest.mark.parametrize("pad", [0, 1, 5, 8, 64, 100003])
def test_memory_and_alignment_of_a_new_gradient(dtype, vocab, pad):
    logits = torch.empty_strided((5, vocab), (vocab + pad, 1), dtype=dtype)
    grad, ldg = linalg._grad_like(None, logits, vocab + pad)
    assert grad.shape == logits.shape and grad.dtype == dtype and grad.stride() == (ldg, 1) and ldg >= vocab
    # the rows' phases are the logits' (relative to the first row), with less than 16 bytes between rows
    assert (ldg - (vocab + pad)) * grad.element_size() % 16 == 0
    assert (ldg - vocab) * grad.element_size() < 16
    assert grad.untyped_storage().nbytes() <= 5 * ldg * grad.element_size()


def test_last_positions_of_sequences():
    """The logits of the last position of each sequence of a batch: a row stride of a whole sequence."""
    logits = torch.empty((4, 50, 1000))[:, -1]
    grad, ldg = linalg._grad_like(None, logits, logits.stride(0))
    assert grad.untyped_storage().nbytes() <= 4 * 1004 * 4


def test_one_row_and_none():
    for rows, vocab in ((1, 1000), (0, 1000), (3, 0), (0, 0)):
        grad, ldg = linalg._grad_like(None, torch.empty((rows, vocab)), vocab)
        assert grad.shape == (rows, vocab) and ldg == vocab
