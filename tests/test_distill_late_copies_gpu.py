"""A warp of the distillation step whose wait for a row's copy runs out: whichever warp it is, the status says so, and
what was not finished is NaN. A test hook tells one warp of the first CTA that one row has not arrived in time; the copy
itself lands as ever, so that nothing else in the CTA notices - the case in which a report is easily lost."""
import pytest
import torch

from raft_b200 import _lib, linalg
from test_topk_distill_gpu import make

pytestmark = pytest.mark.gpu

# bf16 vocabularies that take CTAs of 64, 256 and 512 workers, and a cluster of four of the last
FORMS = [(400, 2), (10000, 8), (20000, 16), (70000, 16)]


def late_step(device, knobs, row, warp, *args):
    assert linalg.last_kernel_status(device) in (_lib.OK, _lib.ERR_TIMEOUT)
    linalg.set_wait_limit_ms(50)
    knobs(B2R_TEST_SKIP_TILE=row + 1, B2R_TEST_LATE_WARP=warp + 1)
    try:
        out = linalg.topk_distill_step(*args)
        status = linalg.last_kernel_status(device)
    finally:
        knobs(B2R_TEST_SKIP_TILE=None, B2R_TEST_LATE_WARP=None)
        linalg.set_wait_limit_ms(0)
    assert linalg.last_kernel_status(device) == _lib.OK
    return status, out


@pytest.mark.parametrize("vocab,warps", FORMS)
@pytest.mark.parametrize("who", ["first worker", "last worker", "list"])
def test_the_last_row_of_a_cluster(cuda, knobs, vocab, warps, who):
    args = make(3, vocab, 8, torch.bfloat16, cuda)
    args[1][0] %= 390  # in the first CTA's part of the row
    exp = linalg.topk_distill_step(*args)
    warp = {"first worker": 0, "last worker": warps - 1, "list": warps + 1}[who]
    status, (loss, lse, grad) = late_step(cuda, knobs, 0, warp, *args)  # a cluster per row: its first row and its last
    assert status == _lib.ERR_TIMEOUT
    assert torch.isnan(loss[0])
    if who == "list":
        assert lse[0] == exp[1][0] and torch.all(torch.isnan(grad[0, :400]))
        assert torch.all(torch.isnan(grad[0]) | (grad[0] == exp[2][0]))
    else:
        assert torch.isnan(lse[0]) and torch.all(torch.isnan(grad[0]))
    for a, b in zip((loss, lse, grad), exp):
        assert torch.equal(a[1:], b[1:])
    for a, b in zip(linalg.topk_distill_step(*args), exp):
        assert torch.equal(a, b)
    assert linalg.last_kernel_status(cuda) == _lib.OK


@pytest.mark.parametrize("vocab,warps", FORMS)
@pytest.mark.parametrize("who", ["first worker", "last worker", "list"])
def test_a_row_in_the_middle(cuda, knobs, vocab, warps, who):
    """Later rows of the cluster are not finished either; every element is right or NaN."""
    args = make(3000, vocab, 8, torch.bfloat16, cuda)
    exp = linalg.topk_distill_step(*args)
    warp = {"first worker": 0, "last worker": warps - 1, "list": warps + 1}[who]
    status, out = late_step(cuda, knobs, 2, warp, *args)
    assert status == _lib.ERR_TIMEOUT
    for a, b in zip(out, exp):
        assert torch.all(torch.isnan(a) | (a == b))
    assert 0 < int(torch.isnan(out[0]).sum()) < 300
    for a, b in zip(linalg.topk_distill_step(*args), exp):
        assert torch.equal(a, b)
