"""sample_tokens against a plain implementation in 64 bits. Tokens have to be EQUAL: the kernel's weights carry a
relative error of 2^-50 and are rounded to 2^-45 of the largest or finer, so a border or a draw could only fall on the
other side where it lies within about 1e-11 of it; the inputs are fixed by their seeds. Log-probabilities: fp64,
rounded once to fp32 (2^-24), weights as above (1e-12)."""
import math

import pytest
import torch

from raft_b200 import _lib, linalg

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference(logits, uniform, temperature, top_k, top_p, min_p):
    n, vocab = logits.shape
    dev = logits.device

    def per_row(v):
        # (numbers are taken as fp32, as the vectors are)
        return (v if isinstance(v, torch.Tensor) else torch.full((n,), v, device=dev, dtype=torch.float32)).double()[:, None]
    t, k, p, m = (per_row(v) for v in (temperature, top_k, top_p, min_p))
    x = torch.where(torch.isnan(logits), -math.inf, logits.double())
    x = torch.where(x == 0, 0.0, x)  # -0 equals +0
    order = torch.argsort(x, dim=1, descending=True, stable=True)
    top = x.gather(1, order[:, :1])
    greedy = ~(t > 0)
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, t)))
    w = torch.where(x > -math.inf, w, 0.0)
    sw = w.gather(1, order)
    rank = torch.arange(vocab, device=dev)
    keep = (sw > 0) & ((k <= 0) | (rank < k)) & (sw >= m.clamp(max=1.0))
    sw = torch.where(keep, sw, 0.0)
    upto = sw.cumsum(1)
    whole = upto[:, -1:]
    keep &= (p >= 1) | (rank == 0) | (upto - sw < p * whole)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    w = torch.where(kept, w, 0.0)
    upto = w.cumsum(1)
    total = upto[:, -1:]
    token = (upto <= uniform.double()[:, None] * total).sum(1)
    last = vocab - 1 - kept.flip(1).to(torch.int8).argmax(1)
    token = torch.minimum(token, last)
    token = torch.where(greedy[:, 0], order[:, 0], token)
    logp = torch.where(greedy[:, 0], 0.0, torch.log(w.gather(1, token[:, None])[:, 0] / total[:, 0]))
    alive = top[:, 0] > -math.inf
    return torch.where(alive, token, -1), torch.where(alive, logp, -math.inf)


def check(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, **kw):
    exp, exp_lp = reference(logits, uniform, temperature, top_k, top_p, min_p)
    got, lp = linalg.sample_tokens(logits, uniform, temperature, top_k, top_p, min_p, **kw)
    assert torch.equal(got.long(), exp), (got.long() != exp).nonzero()[:5].tolist()
    alive = torch.isfinite(exp_lp)
    assert torch.equal(torch.isfinite(lp), alive)
    err = (lp.double() - exp_lp)[alive].abs()
    assert torch.all(err <= exp_lp[alive].abs() * 2.0 ** -24 + 1e-11), float(err.max())
    return got, lp


def make(rows, vocab, dtype, device, seed=0, scale=2.5):
    gen = torch.Generator(device=device).manual_seed(seed)
    logits = (torch.randn((rows, vocab), generator=gen, device=device) * scale).to(dtype)
    return logits, torch.rand(rows, generator=gen, device=device), gen


def mixed(rows, gen, device):
    def some(values, dtype):
        at = torch.randint(0, len(values), (rows,), generator=gen, device=device)
        return torch.tensor(values, device=device, dtype=dtype)[at]
    return dict(temperature=some([0.0, 0.3, 0.7, 1.0, 1.5], torch.float32),
                top_k=some([-1, 0, 1, 2, 20, 50, 1000, 10 ** 9], torch.int32),
                top_p=some([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 1.0, 2.0], torch.float32),
                min_p=some([0.0, 0.0, 0.01, 0.3, 1.0, 5.0], torch.float32))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(40, 1), (40, 2), (40, 7), (64, 33), (200, 1000), (64, 4097), (30, 20001),
                                        (20, 32768), (12, 50001), (8, 131072), (4, 262144), (2, 1400003)])
def test_every_mix_of_filters(cuda, dtype, rows, vocab):
    logits, uniform, gen = make(rows, vocab, dtype, cuda, rows + vocab)
    check(logits, uniform, **mixed(rows, gen, cuda))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("filters", [dict(), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05),
                                     dict(top_k=3000, top_p=0.95), dict(top_k=50, top_p=0.8, min_p=0.02),
                                     dict(temperature=0.0), dict(temperature=0.01), dict(temperature=50.0, top_p=0.7)])
def test_numbers_for_all_rows(cuda, dtype, filters):
    logits, uniform, _ = make(50, 30011, dtype, cuda, 3)
    check(logits, uniform, **filters)


@pytest.mark.parametrize("rows", [1, 100, 700])
def test_number_of_rows_changes_nothing(cuda, rows):
    logits, uniform, gen = make(700, 9001, torch.float32, cuda, 5)
    kw = mixed(700, gen, cuda)
    whole, lp = linalg.sample_tokens(logits, uniform, **kw)
    part, lq = linalg.sample_tokens(logits[:rows], uniform[:rows], **{k: v[:rows] for k, v in kw.items()})
    assert torch.equal(part, whole[:rows]) and torch.equal(lq, lp[:rows])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [100, 20000])
@pytest.mark.parametrize("filters", [dict(), dict(top_k=7), dict(top_k=60, top_p=0.5), dict(top_p=0.25),
                                     dict(min_p=1.0), dict(top_k=5000)])
def test_equal_logits(cuda, dtype, vocab, filters):
    """Ties everywhere: equal logits are kept in the order of their tokens."""
    _, uniform, gen = make(60, vocab, dtype, cuda, 7)
    flat = torch.full((60, vocab), 1.25, device=cuda, dtype=dtype)
    check(flat, uniform, **filters)
    few = torch.randint(0, 4, (60, vocab), generator=gen, device=cuda).to(dtype)
    few[few == 0] = -0.0
    few[:, ::3] = 0.0  # -0 and +0 are equal
    check(few, uniform, **filters)


@pytest.mark.parametrize("scale", [1e-6, 1e-2, 30.0, 1e4, 1e12, 1e30])
@pytest.mark.parametrize("shift", [0.0, -5.0, 5.0])
def test_flat_peaked_and_distant_logits(cuda, scale, shift):
    """Distributions from flat to one token; logits so large that neighbouring floats are whole units apart."""
    logits, uniform, gen = make(40, 6001, torch.float32, cuda, 31, scale=scale)
    logits += shift * scale
    check(logits, uniform, **mixed(40, gen, cuda))
    check(logits, uniform)
    check(logits, uniform, top_p=0.7)


@pytest.mark.parametrize("k", [400, 511, 512, 513, 900, 1500, 2047, 2048, 2049, 5000])
@pytest.mark.parametrize("top_p", [1.0, 0.9, 0.3])
def test_long_lists(cuda, k, top_p):
    """Beginnings of the order around the lengths at which the way of sorting and of drawing changes."""
    logits, uniform, _ = make(30, 20011, torch.float32, cuda, k, scale=0.7)
    check(logits, uniform, top_k=k, top_p=top_p)
    few = (logits * 8).round() / 8  # many equal logits
    check(few, uniform, top_k=k, top_p=top_p)


def test_every_token_gets_its_share(cuda):
    """The same row for a fine grid of uniform numbers: a token is drawn for the grid points of its interval."""
    n, vocab = 20000, 50
    logits, _, _ = make(1, vocab, torch.float32, cuda, 11, scale=1.5)
    grid = (torch.arange(n, device=cuda).double() + 0.5) / n
    got, lp = linalg.sample_tokens(logits.expand(n, vocab).contiguous(), grid.float(), temperature=0.8)
    t = float(torch.tensor(0.8, dtype=torch.float32))
    p = torch.softmax(logits[0].double() / t, 0)
    count = torch.bincount(got.long(), minlength=vocab)
    # an interval of length p holds p * n points of the grid, give or take one at either end; fp32 moves points by 2^-25
    assert torch.all((count - p * n).abs() <= 2.001)
    # p of each draw, as an fp32 logarithm above -16 (half a step there: 2^-21, and as much relative to p)
    assert torch.all(lp > -16) and torch.allclose(lp.double().exp(), p[got.long()], rtol=2.0 ** -21 * 1.001, atol=0)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_and_special_logits(cuda, dtype):
    logits, uniform, gen = make(16, 5000, dtype, cuda, 13)
    low = torch.finfo(dtype).min
    logits[0] = -math.inf
    logits[1, :4990] = -math.inf
    logits[2] = math.nan
    logits[3, ::2] = math.nan
    logits[4, 17] = math.inf
    logits[5, [3, 99, 4000]] = math.inf
    logits[6] = low
    logits[7, :4999] = low
    logits[8, 1:] = -math.inf
    logits[9, ::7] = low
    logits[10] = -math.inf
    logits[10, 4999] = low
    for kw in (dict(), dict(top_k=10), dict(top_p=0.9), dict(top_k=4000, top_p=0.99, min_p=0.001),
               dict(temperature=0.0)):
        got, lp = check(logits, uniform, **kw)
        assert got[0] == -1 and got[2] == -1 and lp[0] == -math.inf
        assert got[4] == 17 and got[8] == 0 and got[10] == 4999


@pytest.mark.parametrize("u", [0.0, 1e-30, 0.5, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan])
def test_ends_of_the_uniform_range(cuda, u):
    """0 takes the first kept token, anything from 1 on the last; below 0 and NaN count as 0."""
    logits, _, _ = make(9, 3001, torch.float32, cuda, 17)
    uniform = torch.full((9,), u, device=cuda)
    clean = 0.0 if not u >= 0 else u
    exp, _ = reference(logits, torch.full((9,), clean, device=cuda), 1.0, 100, 1.0, 0.0)
    got, _ = linalg.sample_tokens(logits, uniform, top_k=100)
    assert torch.equal(got.long(), exp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,off", [(0, 0), (8, 0), (3, 1), (0, 3), (5, 2)])
@pytest.mark.parametrize("vocab", [1001, 40003])
def test_strides_and_alignment(cuda, dtype, pad, off, vocab):
    rows = 12
    base = torch.full((rows * (vocab + pad) + off + 8,), 50.0, device=cuda).to(dtype)  # large where it must not be read
    view = base[off:].as_strided((rows, vocab), (vocab + pad, 1))
    logits, uniform, gen = make(rows, vocab, dtype, cuda, 19)
    view.copy_(logits)
    check(view, uniform, **mixed(rows, gen, cuda))


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_outputs_streams_and_capture(cuda, index_dtype):
    logits, uniform, gen = make(300, 20011, torch.bfloat16, cuda, 23)
    kw = mixed(300, gen, cuda)
    exp, exp_lp = check(logits, uniform, index_dtype=index_dtype, **kw)
    assert exp.dtype == index_dtype
    out, lp = torch.empty_like(exp), torch.empty_like(exp_lp)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        linalg.sample_tokens(logits, uniform, out=out, logprobs=lp, **kw)
    graph.replay()
    assert torch.equal(out, exp) and torch.equal(lp, exp_lp)
    uniform.uniform_()  # the graph reads its inputs when it is replayed
    graph.replay()
    assert torch.equal(out, linalg.sample_tokens(logits, uniform, index_dtype=index_dtype, **kw)[0])
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = linalg.sample_tokens(logits, uniform, index_dtype=index_dtype, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, out)


@pytest.mark.parametrize("rows,vocab", [(0, 10), (3, 0), (0, 0)])
def test_empty(cuda, rows, vocab):
    got, lp = linalg.sample_tokens(torch.empty((rows, vocab), device=cuda), torch.rand(rows, device=cuda))
    assert got.shape == (rows,) and torch.all(got == -1) and torch.all(lp == -math.inf)


def test_offsets_beyond_32_bits(cuda):
    rows, vocab = 16500, 262144  # 4.3e9 elements
    logits = torch.zeros((rows, vocab), dtype=torch.bfloat16, device=cuda)
    logits[-1, 77] = 50.0
    logits[-2, vocab - 1] = 50.0
    uniform = torch.full((rows,), 0.5, device=cuda)
    got, _ = linalg.sample_tokens(logits, uniform)
    assert int(got[-1]) == 77 and int(got[-2]) == vocab - 1 and torch.all(got[:-2] == vocab // 2)


def test_refusals(cuda):
    logits, uniform, _ = make(4, 100, torch.float32, cuda)
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits.cpu(), uniform)
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits, uniform.cpu())
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits, uniform[:3])
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits, uniform.double())
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits.t(), uniform)
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits[0], uniform)
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits, uniform, top_k=torch.ones(4, device=cuda))
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits, uniform, top_p=torch.ones(3, device=cuda))
    with pytest.raises(ValueError):
        linalg.sample_tokens(logits, uniform, out=torch.empty(3, dtype=torch.int32, device=cuda))
    with pytest.raises(_lib.B2RError):
        linalg.sample_tokens(logits, uniform, out=torch.empty(4, dtype=torch.int16, device=cuda))
    with pytest.raises(_lib.B2RError):
        linalg.sample_tokens(logits.double(), uniform)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_vocabulary(cuda, dtype):
    logits, uniform, _ = make(3, 1 << 24, dtype, cuda, 5)
    temperature = torch.tensor([0.0, 0.7, 1.3], device=cuda)
    check(logits, uniform, temperature, top_k=40)
    check(logits[1:], uniform[1:].contiguous(), 1.0)
    with pytest.raises(_lib.B2RError):
        linalg.sample_tokens(torch.empty((1, (1 << 24) + 1), dtype=dtype, device=cuda), uniform[:1].contiguous())


@pytest.mark.parametrize("k", [-1, -2 ** 31, -2 ** 32 + 5, 2 ** 40])
def test_numbers_of_kept_tokens_beyond_32_bits_keep_all(cuda, k):
    logits, uniform, _ = make(64, 1000, torch.float32, cuda, 6)
    got = linalg.sample_tokens(logits, uniform, 1.0, k)
    exp = linalg.sample_tokens(logits, uniform, 1.0, 0)
    assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
