"""What the vocabulary entry points of the C ABI refuse: every call returns its status before it touches a device, so
no GPU is needed. The pointers are never dereferenced."""
import ctypes

import pytest

from raft_b200 import _lib as L

P = 4096  # any non-null, 256-byte aligned "pointer"


@pytest.fixture(scope="module")
def lib():
    return L.load()


def lookup(lib, out=P, ldo=8, table=P, ldt=8, tokens=P, dt=L.F32, tt=L.I64, n=4, c=8, v=10, scale=1.0):
    return lib.b2r_embedding_lookup(out, ldo, table, ldt, tokens, dt, tt, n, c, v, scale, None)


def grad(lib, out=P, ldg=8, odt=L.F32, g=P, ldo=8, dt=L.F32, tokens=P, tt=L.I64, n=4, c=8, v=10, ws=None, wb=0):
    return lib.b2r_embedding_grad(out, ldg, odt, g, ldo, dt, tokens, tt, n, c, v, 1.0, 0, ws, wb, None)


def distill(lib, loss=P, lse=P, grad=None, ldg=0, gl=None, z=P, ldl=100, dt=L.F32, ids=P, ldi=4, it=L.I64, y=P, ldt=4,
            tt=L.F32, n=3, v=100, k=4, t=1.0):
    return lib.b2r_topk_distill(loss, lse, grad, ldg, gl, z, ldl, dt, ids, ldi, it, y, ldt, tt, n, v, k, t, None)


def distill_grad(lib, grad=P, ldg=100, lse=P, gl=P, z=P, ldl=100, dt=L.F32, ids=P, ldi=4, it=L.I64, y=P, ldt=4,
                 tt=L.F32, n=3, v=100, k=4, t=1.0):
    return lib.b2r_topk_distill_grad(grad, ldg, lse, gl, z, ldl, dt, ids, ldi, it, y, ldt, tt, n, v, k, t, None)


def sample(lib, out=P, lp=P, z=P, u=P, **kw):
    d = dict(dtype=L.F32, out_dtype=L.I32, n_rows=3, vocab=100, ld=100, temperature_all=1.0, top_p_all=1.0)
    d.update(kw)
    return lib.b2r_sample_tokens(ctypes.byref(L.SampleDesc(**d)), out, lp, z, u, None)


BIG = 2 ** 31

@pytest.mark.parametrize("kw,status", [
    (dict(out=None), 1), (dict(table=None), 1), (dict(tokens=None), 1), (dict(n=-1), 1), (dict(c=-1), 1),
    (dict(v=-1), 1), (dict(ldo=7), 1), (dict(ldt=7), 1), (dict(dt=L.F64), 2), (dict(dt=L.I32), 2),
    (dict(tt=L.I16), 2), (dict(tt=L.U32), 2), (dict(n=BIG), 4), (dict(v=BIG), 4),
    (dict(c=BIG, ldo=BIG, ldt=BIG), 4)])
def test_lookup(lib, kw, status):
    assert lookup(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(out=None), 1), (dict(g=None), 1), (dict(tokens=None), 1), (dict(n=-1), 1), (dict(c=-1), 1), (dict(v=-1), 1),
    (dict(ldg=7), 1), (dict(ldo=7), 1), (dict(ws=P + 8, wb=1 << 30), 1), (dict(dt=L.F64, odt=L.F64), 2),
    (dict(odt=L.F16), 2), (dict(dt=L.BF16, odt=L.F16), 2), (dict(tt=L.I16), 2), (dict(n=BIG), 4), (dict(v=BIG), 4),
    (dict(c=BIG, ldg=BIG, ldo=BIG), 4)])
def test_grad(lib, kw, status):
    assert grad(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(z=None), 1), (dict(ids=None), 1), (dict(y=None), 1), (dict(n=-1), 1), (dict(v=-1), 1), (dict(k=-1), 1),
    (dict(ldl=99), 1), (dict(ldi=3), 1), (dict(ldt=3), 1), (dict(t=0.0), 1), (dict(t=-1.0), 1), (dict(t=1e-31), 1),
    (dict(t=1e31), 1), (dict(t=float("inf")), 1), (dict(t=float("nan")), 1), (dict(dt=L.F64), 2), (dict(it=L.I16), 2),
    (dict(tt=L.F64), 2), (dict(k=1025, ldi=1025, ldt=1025), 4), (dict(n=BIG), 4), (dict(v=BIG, ldl=BIG), 4)])
def test_distill(lib, kw, status):
    assert distill(lib, **kw) == status
    assert distill(lib, grad=P, ldg=kw.get("ldl", 100), gl=P, **kw) == status
    assert distill_grad(lib, ldg=max(kw.get("ldl", 100), 100), **kw) == status


def test_distill_gradient_arguments(lib):
    assert distill(lib, grad=P, ldg=100, gl=None) == 1
    assert distill(lib, grad=P, ldg=99, gl=P) == 1
    for kw in (dict(grad=None), dict(lse=None), dict(gl=None), dict(ldg=99)):
        assert distill_grad(lib, **kw) == 1


@pytest.mark.parametrize("kw,status", [
    (dict(out=None), 1), (dict(z=None), 1), (dict(u=None), 1), (dict(n_rows=-1), 1), (dict(vocab=-1), 1),
    (dict(ld=99), 1), (dict(dtype=L.F64), 2), (dict(dtype=L.I32), 2), (dict(out_dtype=L.I16), 2),
    (dict(n_rows=BIG), 4), (dict(vocab=BIG, ld=BIG), 4)])
def test_sample(lib, kw, status):
    assert sample(lib, **kw) == status
    assert lib.b2r_sample_tokens(None, P, P, P, P, None) == 1


def test_nothing_to_do_is_fine_without_a_device(lib):
    assert lookup(lib, n=0, tokens=None, out=None) == 0
    assert lookup(lib, c=0, ldo=0, ldt=0) == 0
    assert distill(lib, n=0) == 0
    assert distill_grad(lib, n=0) == 0
    assert sample(lib, n_rows=0) == 0


def test_workspace_sizes(lib):
    size = lib.b2r_embedding_grad_workspace_bytes
    assert size(0, 8, 10) == 0 and size(4, 0, 10) == 0 and size(4, 8, 0) == 0 and size(BIG, 8, 10) == 0
    assert size(1024, 8, 10) == 0  # one launch, without scratch
    assert size(5000, 8, 10) >= 5000 * 8 and size(100000, 64, 50000) > size(5000, 64, 50000)


def test_sample_descriptor_layout_matches_the_header():
    # 2 x int32, 3 x int64, 4 pointers, float, int32, 2 x float = 80 bytes
    assert ctypes.sizeof(L.SampleDesc) == 80
    assert L.SampleDesc.temperature.offset == 32 and L.SampleDesc.temperature_all.offset == 64


@pytest.mark.parametrize("vocab,status", [(1 << 24, 1), ((1 << 24) + 1, 4), (0x7fffffff, 4)])
def test_sample_vocabulary_limit(lib, vocab, status):
    # (a null `uniform` is refused behind the sizes, so that no call is launched here)
    assert sample(lib, u=None, vocab=vocab, ld=vocab) == status
