"""embedding_lookup and embedding_grad against plain 64-bit implementations: every type, odd sizes, strides,
padding tokens, repeated and missing tokens, every path of the sort, accumulation, capture and streams.

Tolerances. lookup: one product in fp32 and one rounding to the output's type: relative error at most
eps(fp32) for the scale and the product (2^-24 each) plus eps / 2 of the type. Gradient: a sum of m terms in fp32 is
off by at most (m - 1) * 2^-24 * sum|x| (any order), the product with the scale by 2 * 2^-24 of it, and the output's
rounding by eps / 2 of the value."""
import numpy as np
import pytest
import torch

from raft_b200 import _lib, linalg

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
U32 = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def tokens_of(n, vocab, dtype, device, kind, seed=0):
    rng = np.random.default_rng(seed)
    if kind == "one":          # a single token everywhere
        t = np.full(n, vocab // 2)
    elif kind == "none":       # nothing but padding
        t = np.full(n, -1)
    elif kind == "ends":       # first and last token, and values just outside
        t = rng.choice([0, vocab - 1, -1, vocab], n)
    elif kind == "skew":       # text-like, with padding
        t = np.floor(np.exp(rng.random(n) * np.log(vocab + 1)) - 1)
        t[rng.random(n) < 0.05] = -1
    else:
        t = rng.integers(0, vocab, n)
    return torch.tensor(t.astype(np.int64), device=device).to(dtype)


def ref_lookup(table, tokens, scale):
    flat = tokens.reshape(-1).long()
    ok = (flat >= 0) & (flat < table.shape[0])
    out = torch.zeros((flat.numel(), table.shape[1]), dtype=torch.float64, device=table.device)
    if table.shape[0]:
        out = torch.where(ok[:, None], table.double()[torch.where(ok, flat, 0)] * scale, out)
    return out


def ref_grad(g, tokens, vocab, scale):
    flat = tokens.reshape(-1).long()
    ok = (flat >= 0) & (flat < vocab)
    at = torch.where(ok, flat, vocab)
    out = torch.zeros((vocab + 1, g.shape[1]), dtype=torch.float64, device=g.device)
    mag, cnt = torch.zeros_like(out), torch.zeros(vocab + 1, dtype=torch.float64, device=g.device)
    out.index_add_(0, at, g.double())
    mag.index_add_(0, at, g.double().abs())
    cnt.index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    return out[:vocab] * scale, mag[:vocab] * abs(scale), cnt[:vocab]


def assert_lookup(got, table, tokens, scale):
    exp = ref_lookup(table, tokens, scale)
    tol = exp.abs() * (half_step(table.dtype) * (1 + 4 * U32) + 2 * U32) + 1e-300
    if table.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step of the subnormal range
    err = (got.reshape(exp.shape).double() - exp).abs()
    assert torch.all(err <= tol), float((err - tol).max())


def assert_grad(got, g, tokens, vocab, scale, old=None):
    exp, mag, cnt = ref_grad(g, tokens, vocab, scale)
    tol = mag * ((cnt[:, None] + 2) * U32)
    if old is not None:
        tol = tol + (exp + old.double()).abs() * U32
        exp = exp + old.double()
    tol = tol + (exp.abs() + tol) * half_step(got.dtype) + 1e-300
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = (got.double() - exp).abs()
    assert torch.all(err <= tol), float((err - tol).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,cols", [(1, 1, 1), (1, 7, 8), (5, 3, 1000), (64, 32000, 2048), (333, 50001, 777),
                                          (1000, 1000, 64), (257, 999, 2), (3, 100, 70001), (100, 5, 12)])
@pytest.mark.parametrize("token_dtype,kind", [(torch.int64, "skew"), (torch.int32, "ends"), (torch.int64, "none")])
def test_lookup(cuda, dtype, n, vocab, cols, token_dtype, kind):
    g = torch.Generator(device=cuda).manual_seed(n + cols)
    table = torch.randn((vocab, cols), generator=g, device=cuda).to(dtype)
    tokens = tokens_of(n, vocab, token_dtype, cuda, kind, n)
    got = linalg.embedding_lookup(table, tokens, scale=1.7)
    assert got.shape == (n, cols) and got.dtype == dtype
    assert_lookup(got, table, tokens, 1.7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad_t,pad_o,off", [(8, 16, 0), (3, 5, 0), (0, 0, 1), (2, 4, 2), (1, 0, 3)])
def test_lookup_strides_and_alignment(cuda, dtype, pad_t, pad_o, off):
    n, vocab, cols = 77, 123, 96
    base = torch.randn(vocab * (cols + pad_t) + off, device=cuda).to(dtype)
    table = base[off:].as_strided((vocab, cols), (cols + pad_t, 1))
    obase = torch.full((n * (cols + pad_o) + off,), 7.0, device=cuda).to(dtype)
    out = obase[off:].as_strided((n, cols), (cols + pad_o, 1))
    tokens = tokens_of(n, vocab, torch.int64, cuda, "skew")
    assert linalg.embedding_lookup(table, tokens, out=out) is out
    assert_lookup(out, table, tokens, 1.0)
    mask = torch.ones_like(obase, dtype=torch.bool)
    mask[off:].as_strided((n, cols), (cols + pad_o, 1)).fill_(False)
    assert torch.all(obase[mask] == 7.0)  # nothing between or around the rows is written


def test_lookup_keeps_the_shape_of_the_tokens(cuda):
    table = torch.randn((50, 24), device=cuda)
    tokens = torch.randint(0, 50, (3, 4, 5), device=cuda)
    got = linalg.embedding_lookup(table, tokens)
    assert got.shape == (3, 4, 5, 24)
    assert torch.equal(got, table[tokens])


def test_lookup_special_values_are_copied(cuda):
    table = torch.tensor([[float("inf"), -float("inf"), float("nan"), 1.0]] * 2, device=cuda)
    got = linalg.embedding_lookup(table, torch.tensor([1, -1], device=cuda))
    assert torch.equal(torch.nan_to_num(got[0], nan=5.0), torch.nan_to_num(table[1], nan=5.0))
    assert torch.all(got[1] == 0)  # padding: zeros, not 0 * inf


@pytest.mark.parametrize("n,vocab,cols", [(0, 5, 8), (4, 5, 0), (3, 0, 8), (0, 0, 0)])
def test_empty(cuda, n, vocab, cols):
    table = torch.randn((vocab, cols), device=cuda)
    tokens = torch.zeros(n, dtype=torch.int64, device=cuda)
    got = linalg.embedding_lookup(table, tokens)
    assert got.shape == (n, cols)
    if vocab == 0:
        assert torch.all(got == 0)
    grad = linalg.embedding_grad(torch.randn((n, cols), device=cuda), tokens, vocab)
    assert grad.shape == (vocab, cols)
    if n == 0:
        assert torch.all(grad == 0)


# one launch up to 1024 positions; above, counting ranks up to 8192, then radix passes: one up to 511 tokens, two up to
# 2^18 - 1, three above
@pytest.mark.parametrize("in_dtype,out_dtype", [(torch.float32, torch.float32), (torch.float16, torch.float16),
                                                (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("n,vocab,cols", [(1, 1, 1), (1, 300, 8), (2, 2, 33), (100, 1000, 64), (1000, 50, 777),
                                          (4096, 32000, 24), (8192, 100, 16), (8193, 511, 8), (9001, 512, 40),
                                          (20011, 50001, 72), (40000, 300000, 9), (3000, 20, 1032), (1023, 5000, 520),
                                          (1024, 130, 1032), (1025, 130, 1031), (2000, 131072, 8)])
@pytest.mark.parametrize("kind", ["skew", "ends", "uniform"])
def test_grad(cuda, in_dtype, out_dtype, n, vocab, cols, kind):
    gen = torch.Generator(device=cuda).manual_seed(n + cols)
    g = torch.randn((n, cols), generator=gen, device=cuda).to(in_dtype)
    tokens = tokens_of(n, vocab, torch.int64 if n % 2 else torch.int32, cuda, kind, n)
    got = linalg.embedding_grad(g, tokens, vocab, scale=0.6, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    assert_grad(got, g, tokens, vocab, 0.6)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 1000, 1024, 1025, 5000, 20000])
@pytest.mark.parametrize("kind", ["one", "none"])
@pytest.mark.parametrize("cols", [8, 13, 2056])
def test_grad_of_one_token_everywhere_or_none(cuda, n, kind, cols):
    g = torch.randn((n, cols), device=cuda)
    tokens = tokens_of(n, 1001, torch.int64, cuda, kind)
    got = linalg.embedding_grad(g, tokens, 1001)
    assert_grad(got, g, tokens, 1001, 1.0)
    if kind == "none":
        assert torch.all(got == 0)


@pytest.mark.parametrize("n", [100, 10000])
@pytest.mark.parametrize("in_dtype,out_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                                (torch.float32, torch.float32)])
@pytest.mark.parametrize("cols", [64, 37])
def test_grad_accumulates(cuda, n, in_dtype, out_dtype, cols):
    vocab = 3000
    g = torch.randn((n, cols), device=cuda).to(in_dtype)
    tokens = tokens_of(n, vocab, torch.int64, cuda, "skew")
    old = torch.randn((vocab, cols), device=cuda).to(out_dtype)
    got = old.clone()
    linalg.embedding_grad(g, tokens, vocab, scale=2.0, grad_table=got, accumulate=True)
    assert_grad(got, g, tokens, vocab, 2.0, old)
    named = torch.zeros(vocab + 1, dtype=torch.bool, device=cuda)
    named[torch.where(tokens < 0, vocab, tokens)] = True
    assert torch.equal(got[~named[:vocab]], old[~named[:vocab]])  # rows that no token names are left alone


@pytest.mark.parametrize("pad_g,pad_t,off", [(8, 8, 0), (3, 5, 0), (0, 1, 0), (0, 0, 1), (4, 0, 2)])
@pytest.mark.parametrize("dtype", TYPES)
def test_grad_strides_and_alignment(cuda, dtype, pad_g, pad_t, off):
    n, vocab, cols = 500, 211, 48
    base = torch.randn(n * (cols + pad_g) + off, device=cuda).to(dtype)
    g = base[off:].as_strided((n, cols), (cols + pad_g, 1))
    tbase = torch.full((vocab * (cols + pad_t) + off,), 7.0, device=cuda)
    table = tbase[off:].as_strided((vocab, cols), (cols + pad_t, 1))
    tokens = tokens_of(n, vocab, torch.int64, cuda, "skew")
    linalg.embedding_grad(g, tokens, vocab, grad_table=table)
    assert_grad(table, g, tokens, vocab, 1.0)
    mask = torch.ones_like(tbase, dtype=torch.bool)
    mask[off:].as_strided((vocab, cols), (cols + pad_t, 1)).fill_(False)
    assert torch.all(tbase[mask] == 7.0)


@pytest.mark.parametrize("n,vocab,cols", [(3000, 500, 264), (30000, 70000, 40)])
def test_grad_repeats_bit_for_bit(cuda, n, vocab, cols):
    g = torch.randn((n, cols), device=cuda)
    tokens = tokens_of(n, vocab, torch.int64, cuda, "skew")
    first = linalg.embedding_grad(g, tokens, vocab)
    for _ in range(3):
        assert torch.equal(linalg.embedding_grad(g, tokens, vocab), first)


def test_grad_poisoned_rows_of_padding_are_not_read_into_sums(cuda):
    n, vocab, cols = 3000, 100, 40
    g = torch.randn((n, cols), device=cuda)
    tokens = tokens_of(n, vocab, torch.int64, cuda, "skew")
    g[tokens < 0] = float("nan")
    got = linalg.embedding_grad(g, tokens, vocab)
    assert torch.isfinite(got).all()
    assert_grad(got, torch.nan_to_num(g), tokens, vocab, 1.0)


def test_grad_is_the_difference_quotient_of_the_lookup(cuda):
    """d/dtable of sum(w * lookup(table)): the lookup is linear, so a difference of two exactly representable
    tables gives the gradient up to the rounding of the products: 64-bit sums of fp32 outputs, small integers."""
    vocab, cols, n = 40, 12, 300
    gen = torch.Generator(device=cuda).manual_seed(3)
    w = torch.randint(-4, 5, (n, cols), generator=gen, device=cuda).float()
    tokens = tokens_of(n, vocab, torch.int64, cuda, "skew")
    table = torch.randint(-8, 9, (vocab, cols), generator=gen, device=cuda).float()
    grad = linalg.embedding_grad(w, tokens, vocab, scale=0.5)

    def f(t):
        return (linalg.embedding_lookup(t, tokens, scale=0.5).double() * w.double()).sum()
    for v, c in [(0, 0), (1, 5), (39, 11), (7, 3)]:
        up, down = table.clone(), table.clone()
        up[v, c] += 1
        down[v, c] -= 1
        assert float((f(up) - f(down)) / 2) == float(grad[v, c])  # all values are small multiples of 1/4: exact


@pytest.mark.parametrize("n", [700, 20000])
def test_grad_workspace_and_capture(cuda, n):
    vocab, cols = 5000, 64
    g = torch.randn((n, cols), device=cuda)
    tokens = tokens_of(n, vocab, torch.int64, cuda, "skew")
    need = linalg.embedding_grad_workspace_bytes(g, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    exp = linalg.embedding_grad(g, tokens, vocab)
    assert torch.equal(linalg.embedding_grad(g, tokens, vocab, workspace=ws), exp)
    table = torch.empty((vocab, cols), device=cuda)
    for w in (ws, None):  # both graphs use the workspace, one after the other; the second takes the library's pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            linalg.embedding_grad(g, tokens, vocab, grad_table=table, workspace=w)
        for _ in range(3):
            table.fill_(5.0)
            graph.replay()
            assert torch.equal(table, exp)
    g.mul_(2.0)
    graph.replay()
    assert torch.equal(table, exp * 2)


def test_on_another_stream(cuda):
    side = torch.cuda.Stream(cuda)
    table = torch.randn((1000, 128), device=cuda)
    tokens = tokens_of(5000, 1000, torch.int64, cuda, "skew")
    g = torch.randn((5000, 128), device=cuda)
    exp, exp_g = linalg.embedding_lookup(table, tokens), linalg.embedding_grad(g, tokens, 1000)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_g = linalg.embedding_lookup(table, tokens), linalg.embedding_grad(g, tokens, 1000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, exp) and torch.equal(got_g, exp_g)


def test_offsets_beyond_32_bits(cuda):
    """A table of more than 2^32 bytes and elements: the last rows."""
    vocab, cols = 2100000, 2056
    table = torch.zeros((vocab, cols), dtype=torch.float16, device=cuda)
    table[-1] = 3.0
    table[-2] = 4.0
    tokens = torch.tensor([vocab - 1, 0, vocab - 2, vocab], device=cuda)
    got = linalg.embedding_lookup(table, tokens)
    assert got[:, 0].tolist() == [3.0, 0.0, 4.0, 0.0] and got[:, -1].tolist() == [3.0, 0.0, 4.0, 0.0]
    table.fill_(9.0)
    linalg.embedding_grad(got, tokens, vocab, grad_table=table)
    assert torch.all(table[-1] == 3.0) and torch.all(table[-2] == 4.0) and torch.all(table[:-2] == 0)


def test_refusals(cuda):
    table = torch.randn((10, 8), device=cuda)
    tokens = torch.zeros(4, dtype=torch.int64, device=cuda)
    g = torch.randn((4, 8), device=cuda)
    with pytest.raises(ValueError):
        linalg.embedding_lookup(table.cpu(), tokens)
    with pytest.raises(ValueError):
        linalg.embedding_lookup(table, tokens.cpu())
    with pytest.raises(ValueError):
        linalg.embedding_lookup(table.t(), tokens)
    with pytest.raises(ValueError):
        linalg.embedding_lookup(table, torch.zeros((4, 2), dtype=torch.int64, device=cuda).t())
    with pytest.raises(ValueError):
        linalg.embedding_lookup(table, tokens, out=torch.empty((4, 7), device=cuda))
    with pytest.raises(ValueError):
        linalg.embedding_lookup(table, tokens, out=torch.empty((4, 8), device=cuda, dtype=torch.float16))
    with pytest.raises(ValueError):
        linalg.embedding_lookup(table, tokens, out=table[2:6])
    with pytest.raises(_lib.B2RError):
        linalg.embedding_lookup(table.double(), tokens)
    with pytest.raises(_lib.B2RError):
        linalg.embedding_lookup(table, tokens.to(torch.int16))
    with pytest.raises(ValueError):
        linalg.embedding_grad(g[:3], tokens, 10)
    with pytest.raises(ValueError):
        linalg.embedding_grad(g[:1].expand(4, 8), tokens, 10)
    with pytest.raises(ValueError):
        linalg.embedding_grad(g, tokens, -1)
    with pytest.raises(ValueError):
        linalg.embedding_grad(g, tokens, 10, accumulate=True)
    with pytest.raises(ValueError):
        linalg.embedding_grad(g, tokens, 10, grad_table=torch.empty((9, 8), device=cuda))
    with pytest.raises(ValueError):
        linalg.embedding_grad(g, tokens, 4, grad_table=g)
    with pytest.raises(_lib.B2RError):
        linalg.embedding_grad(g, tokens, 10, out_dtype=torch.float16)
    with pytest.raises(_lib.B2RError):
        linalg.embedding_grad(g.half(), tokens, 10, out_dtype=torch.bfloat16)


def test_refuses_a_broadcast_gradient(cuda):
    """What a sum's backward pass hands on: every row at the same address."""
    g = torch.ones(1, 8, device=cuda).expand(4, 8)
    with pytest.raises(ValueError):
        linalg.embedding_grad(g, torch.arange(4, device=cuda), 10)
    assert_grad(linalg.embedding_grad(g.contiguous(), torch.arange(4, device=cuda), 10), g.contiguous(),
                torch.arange(4, device=cuda), 10, 1.0)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 8191, 8192, 8193])
def test_grad_at_the_borders_between_the_forms(cuda, n):
    tokens = tokens_of(n, 700, torch.int64, cuda, "skew", n)
    g = torch.randn((n, 36), generator=torch.Generator(device=cuda).manual_seed(n), device=cuda)
    assert_grad(linalg.embedding_grad(g, tokens, 700, scale=0.5), g, tokens, 700, 0.5)
