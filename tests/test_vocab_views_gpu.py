"""Outputs of the vocabulary operators between the rows of their inputs: column blocks of one buffer share no element."""
import pytest
import torch

from raft_b200 import linalg
from test_embedding_gpu import assert_grad, assert_lookup, tokens_of
from test_topk_distill_gpu import TYPES, assert_all, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 37])
def test_lookup_beside_its_table(cuda, dtype, cols):
    wide = torch.randn((300, 2 * cols + 1), device=cuda).to(dtype)
    tokens = tokens_of(300, 300, torch.int64, cuda, "skew")
    before = wide.clone()
    out = linalg.embedding_lookup(wide[:, :cols], tokens, scale=1.7, out=wide[:, cols:2 * cols])
    assert_lookup(out, before[:, :cols], tokens, 1.7)
    assert torch.equal(wide[:, :cols], before[:, :cols]) and torch.equal(wide[:, 2 * cols:], before[:, 2 * cols:])
    with pytest.raises(ValueError):
        linalg.embedding_lookup(wide[:, :cols], tokens, out=wide[:, cols - 1:2 * cols - 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [64, 37])
@pytest.mark.parametrize("n", [300, 3000])
def test_gradient_beside_its_input(cuda, dtype, cols, n):
    wide = torch.randn((n, 2 * cols + 1), device=cuda).to(dtype)
    tokens = tokens_of(n, n, torch.int64, cuda, "skew")
    before = wide.clone()
    table = linalg.embedding_grad(wide[:, cols + 1:], tokens, n, grad_table=wide[:, 1:cols + 1])
    assert_grad(table, before[:, cols + 1:], tokens, n, 1.0)
    assert torch.equal(wide[:, cols + 1:], before[:, cols + 1:]) and torch.equal(wide[:, :1], before[:, :1])
    with pytest.raises(ValueError):
        linalg.embedding_grad(wide[:, cols:2 * cols], tokens, n, grad_table=wide[:, 1:cols + 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1000, 20003, 140001, 300007])
def test_distillation_gradient_beside_the_logits(cuda, dtype, vocab):
    logits, ids, teacher, weight = make(6, vocab, 9, dtype, cuda, 3)
    wide = torch.full((6, 2 * vocab + 3), 7.0, device=cuda).to(dtype)
    wide[:, 1:vocab + 1] = logits
    z, g = wide[:, 1:vocab + 1], wide[:, vocab + 2:2 * vocab + 2]
    edges = [0, vocab + 1, 2 * vocab + 2]
    loss, lse, got = linalg.topk_distill_step(z, ids, teacher, weight, grad=g)
    assert torch.equal(z, logits) and torch.all(wide[:, edges] == 7.0)
    assert_all(logits, ids, teacher, weight, 1.0, loss, lse, got)
    g.fill_(7.0)
    got = linalg.topk_distill_grad(z, ids, teacher, lse, weight, grad=g)
    assert torch.equal(z, logits) and torch.all(wide[:, edges] == 7.0)
    assert_all(logits, ids, teacher, weight, 1.0, grad=got)
    with pytest.raises(ValueError):
        linalg.topk_distill_step(z, ids, teacher, weight, grad=wide[:, 2:vocab + 2])


def test_odd_layouts_are_refused_as_before(cuda):
    logits, ids, teacher, weight = make(6, 100, 4, torch.float32, cuda)
    for kw in (dict(loss=torch.zeros(12, device=cuda)[::2]), dict(lse=torch.zeros((2, 3), device=cuda).t()),
               dict(grad=torch.zeros((1, 100), device=cuda).expand(6, 100)), dict(grad=torch.zeros((100, 6), device=cuda).t())):
        with pytest.raises(ValueError):
            linalg.topk_distill_step(logits, ids, teacher, weight, **kw)
