"""topk_distill, topk_distill_step and topk_distill_grad against a plain 64-bit implementation.

Tolerances, in units of u = 2^-24 (half a step of fp32). A term of the sum S of exponentials carries the error of
the exponential (4u), of its exponent d = (z - max) / (T ln 2) (three roundings: 3u |d| ln 2, and |d| 2^-|d| summed
over a distribution is at most its entropy, log2 V), and of the additions (elements per thread, and 20 levels of
partial sums). log S is off by the relative error of S. A teacher weight is off by its exponent's roundings and
those of the exponential and the sum."""
import math

import pytest
import torch

from raft_b200 import _lib, linalg

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def make(rows, vocab, k, dtype, device, seed=0, scale=3.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    logits = (torch.randn((rows, vocab), generator=gen, device=device) * scale).to(dtype)
    ids = torch.randint(0, max(vocab, 1), (rows, k), generator=gen, device=device)
    teacher = torch.randn((rows, k), generator=gen, device=device) * 2.0
    weight = torch.rand(rows, generator=gen, device=device) - 0.3
    return logits, ids, teacher, weight


def reference(logits, ids, teacher, weight, t):
    z = logits.double() / t
    vocab = z.shape[1]
    valid = (ids >= 0) & (ids < vocab)
    y = torch.where(valid, teacher.double() / t, -math.inf)
    some = y.amax(1, keepdim=True) > -math.inf if y.shape[1] else torch.zeros((z.shape[0], 1), dtype=torch.bool,
                                                                              device=z.device)
    logp = torch.where(some, torch.log_softmax(torch.where(some, y, 0.0), 1), -math.inf)
    p = logp.exp()
    lse = torch.logsumexp(z, 1) if vocab else torch.full((z.shape[0],), -math.inf, device=z.device).double()
    logq = z.gather(1, torch.where(valid, ids, 0).long()) - lse[:, None] if vocab and ids.shape[1] else torch.zeros_like(p)
    loss = t * t * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    spread = torch.zeros((z.shape[0], vocab + 1), dtype=torch.float64, device=z.device)
    spread.scatter_add_(1, torch.where(valid, ids, vocab).long(), p)
    q = (z - lse[:, None]).exp()
    grad = torch.where(some, t * weight.double()[:, None] * (q - spread[:, :vocab]), 0.0)
    return dict(loss=loss, lse=lse, grad=grad, p=p, logp=logp, logq=logq, q=q, spread=spread[:, :vocab], z=z)


def sum_error(vocab):
    per_thread = 64 if vocab <= 8 * 512 * 64 else math.ceil(vocab / (8 * 512)) + 64
    return U * (4 + 2.1 * math.log2(max(vocab, 2)) + per_thread + 20)


def assert_all(logits, ids, teacher, weight, t, loss=None, lse=None, grad=None):
    r = reference(logits, ids, teacher, weight, t)
    vocab, k = logits.shape[1], ids.shape[1]
    es = sum_error(vocab)
    logp = torch.where(r["p"] > 0, r["logp"].abs(), 0.0)
    # weights: exponent (y - max) / T - log sum, each with three roundings of their magnitude; k additions; expf 4u
    finite = torch.where(torch.isfinite(teacher), teacher.double(), 0.0)  # entries at -inf weigh exactly 0
    span = finite.abs().amax(1, keepdim=True) * 2 / t + 8 if k else torch.zeros_like(logp)
    ep_abs = U * (3 * span + 4 + k)          # of log p
    ep = ep_abs + 4 * U                      # of p, relative
    if lse is not None:
        err = (lse.double() - r["lse"]).abs()
        tol = es + 4 * U * r["lse"].abs()
        assert torch.all(err <= tol), (float(err.max()), float(tol.min()))
    if loss is not None:
        elq = es + 4 * U * (r["logq"].abs() + 1)
        term = torch.where(r["p"] > 0, r["p"] * (ep * (logp + r["logq"].abs()) + ep_abs + elq), 0.0)
        tol = t * t * term.sum(1) + 4 * U * r["loss"].abs() + 1e-30
        err = (loss.double() - r["loss"]).abs()
        assert torch.all(err <= tol), (float(err.max()), float(tol.min()))
    if grad is not None:
        assert grad.dtype == logits.dtype and grad.shape == logits.shape
        top = r["lse"][:, None]
        eq = es + U * (4 * (r["z"] - top).abs() + 4 * top.abs() + 8)  # roundings of the exponent; lse of a call
        f = (t * weight.double()).abs()[:, None]
        tol = f * (r["q"] * eq + r["spread"] * (ep.amax(1, keepdim=True) if k else 0.0)) + 3 * U * r["grad"].abs()
        tol = tol + (r["grad"].abs() + tol) * torch.finfo(grad.dtype).eps / 2 + 1e-37
        if grad.dtype == torch.float16:
            tol = tol + 2.0 ** -25
        if grad.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -133
        err = (grad.double() - r["grad"]).abs()
        assert torch.all(err <= tol), float((err - tol).max())


def run_all(logits, ids, teacher, weight, t):
    loss, lse = linalg.topk_distill(logits, ids, teacher, temperature=t)
    assert_all(logits, ids, teacher, weight, t, loss, lse)
    loss2, lse2, grad = linalg.topk_distill_step(logits, ids, teacher, weight, temperature=t)
    assert_all(logits, ids, teacher, weight, t, loss2, lse2, grad)
    grad2 = linalg.topk_distill_grad(logits, ids, teacher, lse, weight, temperature=t)
    assert_all(logits, ids, teacher, weight, t, grad=grad2)


# sizes at and around the borders between the forms (16-bit types: one CTA of 128 threads up to 4096 tokens, of 512 up
# to 16384, clusters of 1, 2, 4, 8 CTAs of 1024 threads up to 262144, beyond that the row is read twice; fp32: half)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 4), (5, 31, 3), (200, 1000, 17), (7, 4082, 5), (7, 4090, 5),
                                          (7, 4096, 8), (5, 4097, 9), (4, 16384, 33), (4, 20001, 1), (3, 50001, 64),
                                          (3, 65535, 40), (2, 131072, 64), (2, 131073, 100), (2, 200003, 7),
                                          (1, 262144, 16), (2, 300007, 50), (600, 2048, 5), (400, 8192, 3),
                                          (300, 40000, 40)])
@pytest.mark.parametrize("t", [1.0, 2.5])
def test_sizes(cuda, dtype, rows, vocab, k, t):
    run_all(*make(rows, vocab, k, dtype, cuda, rows + vocab), t)


@pytest.mark.parametrize("k", [0, 1, 31, 32, 33, 300, 1024])
def test_list_lengths(cuda, k):
    logits, ids, teacher, weight = make(6, 5000, k, torch.float32, cuda, k)
    run_all(logits, ids, teacher, weight, 1.5)


@pytest.mark.parametrize("id_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("teacher_dtype", TYPES)
def test_list_types(cuda, id_dtype, teacher_dtype):
    logits, ids, teacher, weight = make(9, 3000, 20, torch.bfloat16, cuda)
    run_all(logits, ids.to(id_dtype), teacher.to(teacher_dtype), weight, 1.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [3000, 40000])
def test_padded_lists_and_rows_without_one(cuda, dtype, vocab):
    logits, ids, teacher, weight = make(40, vocab, 12, dtype, cuda)
    length = torch.arange(40, device=cuda)[:, None] % 13
    ids = torch.where(torch.arange(12, device=cuda) < length, ids, -1)
    ids[5, 2] = vocab       # just outside
    ids[6, :] = 2 ** 40     # far outside
    teacher[7, :3] = -math.inf
    teacher[8, :] = -math.inf
    run_all(logits, ids, teacher, weight, 2.0)
    loss, _, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
    for r in (0, 6, 8, 13, 26, 39):
        assert loss[r] == 0 and torch.all(grad[r] == 0), r


@pytest.mark.parametrize("vocab", [700, 40000])
def test_a_token_named_twice_counts_twice(cuda, vocab):
    logits, ids, teacher, weight = make(8, vocab, 40, torch.float32, cuda)
    ids = ids % 5 * 7
    ids[3] = 11
    run_all(logits, ids, teacher, weight, 1.0)


def test_masked_rows_may_hold_anything(cuda):
    """Rows without a list: NaN and infinities in their logits reach nothing; other rows are not disturbed."""
    logits, ids, teacher, weight = make(6, 20000, 8, torch.float32, cuda)
    ids[[1, 3, 4]] = -1
    logits[1, 5] = math.nan
    logits[3, 7] = math.inf
    logits[4] = -math.inf
    teacher[1] = math.nan
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
    grad2 = linalg.topk_distill_grad(logits, ids, teacher, lse, weight)
    for r in (1, 3, 4):
        assert loss[r] == 0 and torch.all(grad[r] == 0) and torch.all(grad2[r] == 0)
    keep = [0, 2, 5]
    assert_all(logits[keep], ids[keep], teacher[keep], weight[keep], 1.0, loss[keep], lse[keep], grad[keep])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1.0, 0.7, 2.3, 3.0])
def test_masked_logits(cuda, dtype, t):
    """Logits at -inf and at the type's lowest value have probability 0 and gradient 0 (where no target is)."""
    logits, ids, teacher, weight = make(4, 9000, 8, dtype, cuda)
    ids = ids % 4000 + 5000
    logits[:, :2500] = -math.inf
    logits[:, 2500:5000] = torch.finfo(dtype).min
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight, temperature=t)
    assert torch.all(grad[:, :5000] == 0)
    grad2 = linalg.topk_distill_grad(logits, ids, teacher, lse, weight, temperature=t)
    assert torch.all(grad2[:, :5000] == 0)
    assert_all(logits[:, 5000:], ids - 5000, teacher, weight, t, loss, lse, grad[:, 5000:])
    # a target on a masked logit: infinite loss, finite gradient
    ids[0, 0] = 3
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight, temperature=t)
    assert loss[0] == math.inf and torch.isfinite(grad).all() and torch.isfinite(loss[1:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1000, 40000])
def test_a_row_at_the_lowest_value_is_flat(cuda, dtype, vocab):
    """All logits at the type's lowest finite value: no overflow of their products, a flat distribution."""
    logits, ids, teacher, weight = make(2, vocab, 4, dtype, cuda)
    logits[1] = torch.finfo(dtype).min
    _, _, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
    free = torch.ones(vocab, dtype=torch.bool, device=cuda)
    free[ids[1]] = False
    exp = float(weight[1]) / vocab
    # q = 2^-log2(vocab): the logarithm's half step (log2 vocab * 2^-24) and ex2's 4u; one rounding of the output
    tol = abs(exp) * (40 * U + torch.finfo(dtype).eps / 2) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert torch.all((grad[1, free].double() - exp).abs() <= tol)


def test_nan_logits_show(cuda):
    logits, ids, teacher, weight = make(3, 9000, 8, torch.float32, cuda)
    logits[1, 8999] = math.nan
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
    assert torch.isnan(loss[1]) and torch.isnan(lse[1]) and torch.isnan(grad[1]).all()
    assert torch.isfinite(loss[[0, 2]]).all() and torch.isfinite(grad[[0, 2]]).all()


@pytest.mark.parametrize("scale", [0.0, 1e-3, 40.0, 2000.0])
def test_flat_and_peaked_rows(cuda, scale):
    logits, ids, teacher, weight = make(5, 12000, 6, torch.float32, cuda, scale=scale)
    run_all(logits, ids, teacher, weight, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad_l,pad_g,off_l,off_g", [(0, 0, 0, 0), (8, 8, 0, 0), (3, 3, 1, 1), (3, 5, 0, 0),
                                                     (0, 0, 1, 2), (1, 0, 3, 0)])
@pytest.mark.parametrize("vocab", [1003, 33000])
def test_strides_and_alignment(cuda, dtype, pad_l, pad_g, off_l, off_g, vocab):
    rows, k = 6, 10
    base = (torch.randn(rows * (vocab + pad_l) + off_l, device=cuda) * 3).to(dtype)
    logits = base[off_l:].as_strided((rows, vocab), (vocab + pad_l, 1))
    _, ids, teacher, weight = make(rows, vocab, k + 3, dtype, cuda)
    ids, teacher = ids[:, :k], teacher[:, 2:k + 2]  # strided lists
    gbase = torch.full((rows * (vocab + pad_g) + off_g,), 7.0, device=cuda).to(dtype)
    grad = gbase[off_g:].as_strided((rows, vocab), (vocab + pad_g, 1))
    mask = torch.ones_like(gbase, dtype=torch.bool)
    mask[off_g:].as_strided((rows, vocab), (vocab + pad_g, 1)).fill_(False)
    loss, lse, out = linalg.topk_distill_step(logits, ids, teacher, weight, grad=grad)
    assert out is grad
    assert_all(logits, ids, teacher, weight, 1.0, loss, lse, grad)
    assert torch.all(gbase[mask] == 7.0)
    grad.fill_(7.0)
    linalg.topk_distill_grad(logits, ids, teacher, lse, weight, grad=grad)
    assert_all(logits, ids, teacher, weight, 1.0, grad=grad)
    assert torch.all(gbase[mask] == 7.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1001, 20003, 140001, 530001])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_padding_entries_write_nothing(cuda, dtype, vocab, off):
    """Rows off 16-byte boundaries with -1 in their lists: the element before the row, the last one of the row before
    and the one behind the matrix stay what they are."""
    rows, k = 5, 9
    base = torch.full((rows * vocab + off + 1,), 7.0, device=cuda).to(dtype)
    grad = base[off:-1].view(rows, vocab)
    logits, ids, teacher, weight = make(rows, vocab, k, dtype, cuda, seed=vocab)
    ids[:, 4:] = -1
    src = torch.zeros_like(base)
    src[off:-1] = logits.reshape(-1)
    src = src[off:-1].view(rows, vocab)
    loss, lse, _ = linalg.topk_distill_step(src, ids, teacher, weight, grad=grad)
    assert torch.all(base[:off] == 7.0) and base[-1] == 7.0
    assert_all(logits, ids, teacher, weight, 1.0, loss, lse, grad)
    grad.fill_(7.0)
    linalg.topk_distill_grad(src, ids, teacher, lse, weight, grad=grad)
    assert torch.all(base[:off] == 7.0) and base[-1] == 7.0
    assert_all(logits, ids, teacher, weight, 1.0, grad=grad)


@pytest.mark.parametrize("vocab", [3000, 40000])
def test_threads_that_see_only_masked_logits(cuda, vocab):
    """Most of the row at -inf, the rest far below zero: no product of a zero and an overflowed factor."""
    logits, ids, teacher, weight = make(3, vocab, 4, torch.float32, cuda)
    logits[:, 50:] = -math.inf
    logits[:, :50] -= 1000.0
    ids = ids % 50
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
    assert torch.isfinite(loss).all() and torch.all(grad[:, 50:] == 0)
    grad2 = linalg.topk_distill_grad(logits, ids, teacher, lse, weight)
    for g in (grad, grad2):
        assert_all(logits[:, :50].contiguous(), ids, teacher, weight, 1.0, loss, lse, g[:, :50])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [999, 30000, 131072, 300000])
def test_in_place(cuda, dtype, vocab):
    logits, ids, teacher, weight = make(5, vocab, 20, dtype, cuda)
    loss, lse, exp = linalg.topk_distill_step(logits, ids, teacher, weight)
    work = logits.clone()
    loss2, lse2, grad = linalg.topk_distill_step(work, ids, teacher, weight, grad=work)
    assert grad is work and torch.equal(work, exp) and torch.equal(loss, loss2) and torch.equal(lse, lse2)
    exp = linalg.topk_distill_grad(logits, ids, teacher, lse, weight)
    work = logits.clone()
    assert torch.equal(linalg.topk_distill_grad(work, ids, teacher, lse, weight, grad=work), exp)


@pytest.mark.parametrize("vocab", [50, 5000])
def test_gradient_is_the_difference_quotient_of_the_loss(cuda, vocab):
    """In 64 bits the reference's loss is differenced at h = 1e-5 (error h^2 of the third derivative, under 1e-9, and
    1e-16 |loss| / h = 1e-10); the kernel's gradient is held to that plus its own fp32 error (1e-5 of the weight)."""
    logits, ids, teacher, weight = make(4, vocab, 6, torch.float32, cuda, seed=9)
    weight = torch.ones_like(weight)
    _, _, grad = linalg.topk_distill_step(logits, ids, teacher, weight, temperature=1.7)
    h = 1e-5
    for v in [0, 1, vocab - 1] + ids[0, :3].tolist():
        step = torch.zeros((4, vocab), dtype=torch.float64, device=cuda)
        step[:, v] = h
        up = reference(logits.double() + step, ids, teacher, weight, 1.7)["loss"]
        down = reference(logits.double() - step, ids, teacher, weight, 1.7)["loss"]
        assert torch.allclose((up - down) / (2 * h), grad[:, v].double(), rtol=0, atol=2e-5)


@pytest.mark.parametrize("rows,vocab", [(700, 4000), (300, 40000)])
def test_repeats_bit_for_bit_and_captures(cuda, rows, vocab):
    logits, ids, teacher, weight = make(rows, vocab, 16, torch.bfloat16, cuda)
    exp = linalg.topk_distill_step(logits, ids, teacher, weight)
    out = [torch.empty_like(x) for x in exp]
    for _ in range(3):
        for a, b in zip(linalg.topk_distill_step(logits, ids, teacher, weight), exp):
            assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        linalg.topk_distill_step(logits, ids, teacher, weight, loss=out[0], lse=out[1], grad=out[2])
    graph.replay()
    for a, b in zip(out, exp):
        assert torch.equal(a, b)


def test_on_another_stream(cuda):
    logits, ids, teacher, weight = make(300, 20000, 16, torch.float16, cuda)
    exp = linalg.topk_distill_step(logits, ids, teacher, weight)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linalg.topk_distill_step(logits, ids, teacher, weight)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, exp):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,vocab,k", [(0, 10, 3), (3, 0, 2), (0, 0, 0), (2, 10, 0)])
def test_empty(cuda, rows, vocab, k):
    logits, ids, teacher, weight = make(rows, vocab, k, torch.float32, cuda)
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
    assert grad.shape == (rows, vocab) and torch.all(loss == 0)
    if vocab == 0:
        assert torch.all(lse == -math.inf)
    grad = linalg.topk_distill_grad(logits, ids, teacher, lse, weight)
    assert grad.shape == (rows, vocab) and torch.all(grad == 0)


def test_offsets_beyond_32_bits(cuda):
    rows, vocab = 33000, 131072  # 4.3e9 elements
    logits = torch.zeros((rows, vocab), dtype=torch.float16, device=cuda)
    logits[-1, 5] = 4.0
    ids = torch.full((rows, 2), 5, dtype=torch.int32, device=cuda)
    teacher = torch.zeros((rows, 2), device=cuda)
    weight = torch.ones(rows, device=cuda)
    loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight, grad=logits)
    lse0 = math.log(vocab - 1 + math.exp(4.0))
    assert abs(float(lse[-1]) - lse0) < 1e-5 and abs(float(lse[0]) - math.log(vocab)) < 1e-5
    # two entries of weight 1/2 each: log p = -log 2 for both
    assert abs(float(loss[-1]) - (lse0 - 4.0 - math.log(2.0))) < 1e-4
    assert abs(float(grad[-1, 5]) - (math.exp(4.0 - lse0) - 1.0)) < 1e-3


def test_refusals(cuda):
    logits, ids, teacher, weight = make(4, 100, 3, torch.float32, cuda)
    lse = torch.zeros(4, device=cuda)
    with pytest.raises(ValueError):
        linalg.topk_distill(logits.cpu(), ids, teacher)
    with pytest.raises(ValueError):
        linalg.topk_distill(logits, ids.cpu(), teacher)
    with pytest.raises(ValueError):
        linalg.topk_distill(logits, ids[:3], teacher)
    with pytest.raises(ValueError):
        linalg.topk_distill(logits, ids[:, :2], teacher)
    with pytest.raises(ValueError):
        linalg.topk_distill(logits.t(), ids, teacher)
    with pytest.raises(ValueError):
        linalg.topk_distill(logits[:1].expand(4, 100), ids, teacher)
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            linalg.topk_distill(logits, ids, teacher, temperature=t)
    with pytest.raises(_lib.B2RError):
        linalg.topk_distill(logits.double(), ids, teacher)
    with pytest.raises(_lib.B2RError):
        linalg.topk_distill(logits, ids.short(), teacher)
    with pytest.raises(_lib.B2RError):
        linalg.topk_distill(logits, ids, teacher.double())
    with pytest.raises(_lib.B2RError):  # more than 1024 entries
        linalg.topk_distill(logits, ids.repeat(1, 400), teacher.repeat(1, 400))
    with pytest.raises(ValueError):
        linalg.topk_distill_step(logits, ids, teacher, weight[:3])
    with pytest.raises(ValueError):
        linalg.topk_distill_step(logits, ids, teacher, weight.double())
    with pytest.raises(ValueError):
        linalg.topk_distill_step(logits, ids, teacher, weight, grad=torch.empty((4, 99), device=cuda))
    big = torch.randn((5, 100), device=cuda)
    with pytest.raises(ValueError):
        linalg.topk_distill_step(big[:4], ids, teacher, weight, grad=big[1:])
    with pytest.raises(ValueError):
        linalg.topk_distill_grad(logits, ids, teacher, lse[:2], weight)


def test_a_record_that_never_arrives_ends_in_nan_and_a_status(cuda, knobs):
    """The exchange between the CTAs of a row waits with a limit: the first CTA's record for the third row of its
    cluster is withheld, so that its cluster gives up on that row, its later rows are NaN, and all others are right."""
    logits, ids, teacher, weight = make(300, 70000, 8, torch.bfloat16, cuda)
    exp = linalg.topk_distill_step(logits, ids, teacher, weight)
    assert linalg.last_kernel_status(cuda) == _lib.OK
    linalg.set_wait_limit_ms(50)
    knobs(B2R_TEST_SKIP_TILE=3)
    try:
        loss, lse, grad = linalg.topk_distill_step(logits, ids, teacher, weight)
        assert linalg.last_kernel_status(cuda) == _lib.ERR_TIMEOUT
    finally:
        knobs(B2R_TEST_SKIP_TILE=None)
        linalg.set_wait_limit_ms(0)
    bad = torch.isnan(grad).any(1)
    assert 0 < int(bad.sum()) < 150
    assert torch.equal(grad[~bad], exp[2][~bad])
    again = linalg.topk_distill_step(logits, ids, teacher, weight)
    assert linalg.last_kernel_status(cuda) == _lib.OK
    for a, b in zip(again, exp):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [799, 800, 801, 1024])
@pytest.mark.parametrize("vocab", [32768, 131072, 262144])
def test_long_lists_beside_full_rows(cuda, dtype, k, vocab):
    """The list takes its place beside the row's buffers in shared memory, or the row is streamed."""
    run_all(*make(3, vocab, k, dtype, cuda, k), 1.5)
