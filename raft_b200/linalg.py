"""Host-side mirror of the raft::linalg reduction entry points, on torch CUDA tensors.

Every function forwards to the C ABI (include/raft_b200.h) on the current torch CUDA stream
and is asynchronous, like the reference. Names, argument meaning and error behaviour follow
the reference:

  reduce               linalg/reduce.cuh:140-180  (mdspan form: matrix view, vector view, init,
                       inplace, main_op, reduce_op, final_op)
  coalesced_reduction  linalg/coalesced_reduction.cuh:104-149
  strided_reduction    linalg/strided_reduction.cuh:115-160
  norm                 linalg/norm.cuh:112-148
  reduce_rows_by_key   linalg/reduce_rows_by_key.cuh:140-181
  reduce_cols_by_key   linalg/reduce_cols_by_key.cuh:76-102

Beside them, without a counterpart in the reference, the vocabulary operators: embedding_lookup, embedding_grad,
topk_distill, topk_distill_grad, topk_distill_step and sample_tokens.

No function here takes part in autograd: results have no graph, also where an input requires a gradient.
embedding_grad and topk_distill_grad are the backward passes of embedding_lookup and topk_distill.

Shape errors raise ValueError where the reference's RAFT_EXPECTS raises raft::logic_error;
unsupported type / operator combinations raise B2RError (raft::exception in the reference).
Functors are named by strings because a C ABI cannot carry a device lambda; the C++ headers
under include/raft/ accept arbitrary functors.
"""
import contextlib

import torch

from . import _lib as L

_DTYPES = {
    torch.float32: L.F32,
    torch.float64: L.F64,
    torch.float16: L.F16,
    torch.int32: L.I32,
    torch.int64: L.I64,
    torch.int16: L.I16,
}
_MAIN = {"identity": L.MAIN_IDENTITY, "sq": L.MAIN_SQ, "abs": L.MAIN_ABS, "nz": L.MAIN_NZ, "to_kvp": L.MAIN_TO_KVP}
_REDUCE = {"add": L.REDUCE_ADD, "min": L.REDUCE_MIN, "max": L.REDUCE_MAX, "argmin": L.REDUCE_ARGMIN,
           "argmax": L.REDUCE_ARGMAX}
_FINAL = {"identity": L.FINAL_IDENTITY, "sqrt": L.FINAL_SQRT, "mul_const": L.FINAL_MUL_CONST,
          "div_const": L.FINAL_DIV_CONST, "abs": L.FINAL_ABS}
_NORM = {"L1": L.NORM_L1, "L2": L.NORM_L2, "Linf": L.NORM_LINF, "L0": L.NORM_L0}
_KVP_OF = {L.F32: L.KVP_I32_F32, L.F64: L.KVP_I32_F64, L.I16: L.KVP_I32_I16, L.I32: L.KVP_I32_I32}

ALONG_ROWS = L.ALONG_ROWS
ALONG_COLUMNS = L.ALONG_COLUMNS


def _as_int(v):
    try:
        return int(v)
    except (OverflowError, ValueError):  # inf / nan initial values of floating outputs
        return 0


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_NO_SWITCH = contextlib.nullcontext()


def _stream_ptr(device):
    """cudaStream_t of torch's current stream on `device`."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _on(device):
    """Context that makes `device` current - a no-op object when it already is (the usual case; switching
    costs microseconds that small reductions notice)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _NO_SWITCH
    return torch.cuda.device(device)


def _layout_of(data):
    """Row- or column-major contiguous 2-D tensor -> (layout, n_rows, n_cols); else ValueError,
    like RAFT_EXPECTS(is_row_or_column_major(data)) in linalg/reduce.cuh:157."""
    if data.dim() != 2:
        raise ValueError("Input must be a matrix")
    n_rows, n_cols = data.shape
    if data.is_contiguous():
        return L.ROW_MAJOR, n_rows, n_cols
    if data.t().is_contiguous():
        return L.COL_MAJOR, n_rows, n_cols
    raise ValueError("Input must be contiguous")


def _require_cuda(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")


class KeyValueVector:
    """Device array of {int32 key, value} pairs with the memory layout of
    raft::KeyValuePair<int, V> (core/kvp.hpp:20-27)."""

    def __init__(self, n, value_dtype, device):
        self.value_dtype = value_dtype
        self.n = n
        wide = value_dtype == torch.float64
        self.raw = torch.empty((n, 2), dtype=torch.int64 if wide else torch.int32, device=device)

    def data_ptr(self):
        return self.raw.data_ptr()

    @property
    def keys(self):
        if self.value_dtype == torch.float64:
            return self.raw.view(torch.int32)[:, 0]
        return self.raw[:, 0]

    @property
    def values(self):
        if self.value_dtype == torch.float64:
            return self.raw[:, 1].view(torch.float64)
        if self.value_dtype == torch.float32:
            return self.raw[:, 1].view(torch.float32)
        if self.value_dtype == torch.int16:
            return self.raw.view(torch.int16)[:, 2]
        return self.raw[:, 1]

    def fill(self, key, value):
        self.keys.fill_(key)
        self.values.fill_(value)


def reduce(data, apply=ALONG_ROWS, dots=None, init=0.0, inplace=False, main_op="identity", reduce_op="add",
           final_op="identity", final_scalar=1.0, out_dtype=None, init_key=0, workspace=None):
    """dots[k] = final_op(reduce_op over the reduced axis of main_op(data[..], index)).

    `apply` = ALONG_ROWS gives one output per row, ALONG_COLUMNS one per column. With
    reduce_op "argmin"/"argmax" (and main_op "to_kvp") `dots` is a KeyValueVector.
    Returns `dots`.
    """
    _require_cuda(data, "data")
    layout, n_rows, n_cols = _layout_of(data)
    n_out = n_rows if apply == ALONG_ROWS else n_cols
    in_dt = _DTYPES.get(data.dtype)
    if in_dt is None:
        raise L.B2RError(L.ERR_UNSUPPORTED, "reduce")
    kvp = reduce_op in ("argmin", "argmax")
    if kvp:
        if dots is None:
            dots = KeyValueVector(n_out, data.dtype, data.device)
        if not isinstance(dots, KeyValueVector) or dots.value_dtype != data.dtype:
            raise ValueError("argmin/argmax need a KeyValueVector of the input's value type")
        out_dt = _KVP_OF.get(in_dt)
        if out_dt is None:
            raise L.B2RError(L.ERR_UNSUPPORTED, "reduce")
        n_dots = dots.n
    else:
        if dots is None:
            dots = torch.empty(n_out, dtype=out_dtype or (torch.float32 if data.dtype == torch.float16
                                                          else data.dtype), device=data.device)
        _require_cuda(dots, "dots")
        out_dt = _DTYPES.get(dots.dtype)
        n_dots = dots.numel()
        if not dots.is_contiguous():
            raise ValueError("Output must be contiguous")
    if n_dots != n_out:
        raise ValueError("Output should be equal to number of %s in Input" %
                         ("rows" if apply == ALONG_ROWS else "columns"))
    desc = L.ReduceDesc(in_dtype=in_dt, out_dtype=out_dt, layout=layout, apply=apply, n_rows=n_rows, n_cols=n_cols,
                        main_op=_MAIN[main_op], reduce_op=_REDUCE[reduce_op], final_op=_FINAL[final_op],
                        inplace=1 if inplace else 0, init=float(init), init_i=_as_int(init), init_key=int(init_key),
                        final_scalar=float(final_scalar))
    ws_ptr, ws_bytes = (workspace.data_ptr(), workspace.numel() * workspace.element_size()) if workspace is not None \
        else (None, 0)
    lib = L.load()
    with _on(data.device):
        st = lib.b2r_reduce(desc, dots.data_ptr(), data.data_ptr(), ws_ptr, ws_bytes, _stream_ptr(data.device))
    L.check(st, "b2r_reduce")
    return dots


def reduce_workspace_bytes(data, apply=ALONG_ROWS, reduce_op="add", out_dtype=None):
    layout, n_rows, n_cols = _layout_of(data)
    in_dt = _DTYPES[data.dtype]
    out_dt = _KVP_OF[in_dt] if reduce_op in ("argmin", "argmax") else _DTYPES[out_dtype or data.dtype]
    desc = L.ReduceDesc(in_dtype=in_dt, out_dtype=out_dt, layout=layout, apply=apply, n_rows=n_rows, n_cols=n_cols,
                        reduce_op=_REDUCE[reduce_op])
    with _on(data.device):
        return L.load().b2r_reduce_workspace_bytes(desc, data.data_ptr())


def coalesced_reduction(data, dots=None, init=0.0, inplace=False, main_op="identity", reduce_op="add",
                        final_op="identity", final_scalar=1.0, **kw):
    """Reduction along the contiguous dimension: rows of a row-major matrix, columns of a
    column-major one (linalg/coalesced_reduction.cuh:104-149)."""
    layout, _, _ = _layout_of(data)
    apply = ALONG_ROWS if layout == L.ROW_MAJOR else ALONG_COLUMNS
    return reduce(data, apply, dots, init, inplace, main_op, reduce_op, final_op, final_scalar, **kw)


def strided_reduction(data, dots=None, init=0.0, inplace=False, main_op="identity", reduce_op="add",
                      final_op="identity", final_scalar=1.0, **kw):
    """Reduction along the strided dimension: columns of a row-major matrix, rows of a
    column-major one (linalg/strided_reduction.cuh:115-160)."""
    layout, _, _ = _layout_of(data)
    apply = ALONG_COLUMNS if layout == L.ROW_MAJOR else ALONG_ROWS
    return reduce(data, apply, dots, init, inplace, main_op, reduce_op, final_op, final_scalar, **kw)


def norm(data, norm_type="L2", apply=ALONG_ROWS, out=None, fin_op="identity", final_scalar=1.0, out_dtype=None,
         workspace=None):
    """L1 / L2 / Linf norm of every row or column (linalg/norm.cuh:112-148). As in the
    reference L2 is the SQUARED norm unless fin_op is "sqrt"; "L0" is refused."""
    _require_cuda(data, "data")
    layout, n_rows, n_cols = _layout_of(data)
    n_out = n_rows if apply == ALONG_ROWS else n_cols
    if out is None:
        out = torch.empty(n_out, dtype=out_dtype or (torch.float32 if data.dtype == torch.float16 else data.dtype),
                          device=data.device)
    if out.numel() != n_out:
        raise ValueError("Output should be equal to number of %s in Input" %
                         ("rows" if apply == ALONG_ROWS else "columns"))
    ws_ptr, ws_bytes = (workspace.data_ptr(), workspace.numel() * workspace.element_size()) if workspace is not None \
        else (None, 0)
    with _on(data.device):
        st = L.load().b2r_norm(_NORM[norm_type], apply, layout, _DTYPES[data.dtype], _DTYPES[out.dtype], n_rows,
                               n_cols, _FINAL[fin_op], float(final_scalar), out.data_ptr(), data.data_ptr(), ws_ptr,
                               ws_bytes, _stream_ptr(data.device))
    L.check(st, "b2r_norm")
    return out


_KEY_DTYPES = {torch.int32: L.I32, torch.int64: L.I64, torch.uint32: L.U32} if hasattr(torch, "uint32") else \
    {torch.int32: L.I32, torch.int64: L.I64}


def reduce_rows_by_key(d_A, d_keys, n_unique_keys, d_sums=None, d_weights=None, reset_sums=True, counts=None,
                       lda=None, workspace=None):
    """d_sums[d_keys[i], :] += d_weights[i] * d_A[i, :] (linalg/reduce_rows_by_key.cuh:140-181).

    d_A is [nrows x ncols] row-major (row stride `lda`, default ncols); d_sums is
    [n_unique_keys x ncols]. `counts` (int64 [n_unique_keys], optional) receives the rows per
    key - an extension the reference does not have. Returns d_sums.
    """
    _require_cuda(d_A, "d_A")
    _require_cuda(d_keys, "d_keys")
    if d_A.dim() != 2:
        raise ValueError("d_A must be a matrix")
    nrows, ncols = d_A.shape
    if lda is None:
        if d_A.stride(1) != 1 and ncols > 1:
            raise ValueError("d_A must be row-major")
        lda = d_A.stride(0) if nrows > 1 else ncols
    if d_keys.numel() != nrows:
        raise ValueError("Keys is not of size nrows")
    if d_weights is not None and d_weights.numel() != nrows:
        raise ValueError("Weights is not of size nrows")
    if d_sums is None:
        d_sums = torch.zeros((n_unique_keys, ncols), dtype=d_A.dtype, device=d_A.device)
    if tuple(d_sums.shape) != (n_unique_keys, ncols) or not d_sums.is_contiguous():
        raise ValueError("Output is not of size ncols * n_unique_keys")
    if d_sums.dtype != d_A.dtype or (d_weights is not None and d_weights.dtype != d_A.dtype):
        raise L.B2RError(L.ERR_UNSUPPORTED, "reduce_rows_by_key")
    if counts is not None and (counts.dtype != torch.int64 or counts.numel() != n_unique_keys):
        raise ValueError("counts must be int64 of size n_unique_keys")
    key_dt = _KEY_DTYPES.get(d_keys.dtype)
    if key_dt is None or d_A.dtype not in (torch.float32, torch.float64):
        raise L.B2RError(L.ERR_UNSUPPORTED, "reduce_rows_by_key")
    ws_ptr, ws_bytes = (workspace.data_ptr(), workspace.numel() * workspace.element_size()) if workspace is not None \
        else (None, 0)
    with _on(d_A.device):
        st = L.load().b2r_reduce_rows_by_key(
            d_sums.data_ptr(), counts.data_ptr() if counts is not None else None, d_A.data_ptr(), lda,
            d_keys.data_ptr(), d_weights.data_ptr() if d_weights is not None else None, _DTYPES[d_A.dtype], key_dt,
            nrows, ncols, n_unique_keys, 1 if reset_sums else 0, ws_ptr, ws_bytes, _stream_ptr(d_A.device))
    L.check(st, "b2r_reduce_rows_by_key")
    return d_sums


def reduce_rows_by_key_workspace_bytes(d_A, n_unique_keys, lda=None):
    nrows, ncols = d_A.shape
    with _on(d_A.device):
        return L.load().b2r_reduce_rows_by_key_workspace_bytes(d_A.data_ptr(), lda or ncols, _DTYPES[d_A.dtype],
                                                               nrows, ncols, n_unique_keys)


def reduce_cols_by_key(data, keys, out=None, nkeys=0, reset_sums=True, workspace=None):
    """out[r, keys[c]] += data[r, c] (linalg/reduce_cols_by_key.cuh:76-102). nkeys = 0 infers
    the number of keys from out.shape[1], as the reference does. `workspace` (uint8, see
    reduce_cols_by_key_workspace_bytes) keeps the call allocation-free."""
    _require_cuda(data, "data")
    _require_cuda(keys, "keys")
    if data.dim() != 2 or not data.is_contiguous():
        raise ValueError("data must be a row-major matrix")
    nrows, ncols = data.shape
    if out is None:
        if nkeys <= 0:
            raise ValueError("nkeys or out is required")
        out = torch.zeros((nrows, nkeys), dtype=data.dtype, device=data.device)
    if nkeys > 0:
        if out.shape[1] != nkeys:
            raise ValueError("Output doesn't have nkeys columns")
    else:
        nkeys = out.shape[1]
    if out.shape[0] != nrows:
        raise ValueError("Output doesn't have the same number of rows as input")
    if keys.numel() != ncols:
        raise ValueError("Keys is not of size ncols")
    key_dt = _KEY_DTYPES.get(keys.dtype)
    if key_dt is None or data.dtype not in (torch.float32, torch.float64) or out.dtype != data.dtype:
        raise L.B2RError(L.ERR_UNSUPPORTED, "reduce_cols_by_key")
    ws_ptr, ws_bytes = (workspace.data_ptr(), workspace.numel() * workspace.element_size()) if workspace is not None \
        else (None, 0)
    with _on(data.device):
        st = L.load().b2r_reduce_cols_by_key(out.data_ptr(), data.data_ptr(), keys.data_ptr(), _DTYPES[data.dtype],
                                             key_dt, nrows, ncols, nkeys, 1 if reset_sums else 0, ws_ptr, ws_bytes,
                                             _stream_ptr(data.device))
    L.check(st, "b2r_reduce_cols_by_key")
    return out


def reduce_cols_by_key_workspace_bytes(data, nkeys):
    nrows, ncols = data.shape
    with _on(data.device):
        return L.load().b2r_reduce_cols_by_key_workspace_bytes(data.data_ptr(), _DTYPES[data.dtype], nrows, ncols,
                                                               nkeys)


_VOCAB_DTYPES = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
_TOKEN_DTYPES = {torch.int32: L.I32, torch.int64: L.I64}


def _on_device_of(t, name, other):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.device != other.device:
        raise ValueError(f"{name} must be on {other.device}")


def _row_stride(t, name):
    """Row stride of a row-major matrix (rows may be further apart than they are long)."""
    n_rows, n_cols = t.shape
    s0, s1 = t.stride()
    if n_cols > 1 and s1 != 1:
        raise ValueError(f"{name} must be row-major")
    if n_rows <= 1:
        return n_cols
    if s0 < n_cols:
        raise ValueError(f"{name} must be row-major")
    return s0


def _overlap(a, b):
    """Whether two tensors share memory. Rows of a matrix may lie between rows of another (column blocks of one buffer);
    of layouts that are not matrices of contiguous rows apart from one another, the memory that they span counts."""
    def rows(t):  # (address of the first row, bytes of a row, distance of rows, number of rows)
        size = t.element_size()
        if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) > t.shape[1]:
            return t.data_ptr(), t.shape[1] * size, t.stride(0) * size, t.shape[0]
        return t.data_ptr(), (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * size, 0, 1
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, la, sa, na), (b0, lb, sb, nb) = rows(a), rows(b)
    if a0 >= b0 + (nb - 1) * sb + lb or b0 >= a0 + (na - 1) * sa + la:
        return False
    if na < nb:
        (a0, la, sa, na), (b0, lb, sb, nb) = (b0, lb, sb, nb), (a0, la, sa, na)
    if na == 1:
        return True
    # for every row of b: is there an i such that row a0 + i sa begins before its end and ends behind its beginning?
    begin = b0 - a0 + torch.arange(nb, dtype=torch.int64) * sb
    first = torch.div(begin - la, sa, rounding_mode="floor") + 1
    last = torch.div(begin + lb - 1, sa, rounding_mode="floor")
    return bool((first.clamp(min=0) <= last.clamp(max=na - 1)).any())


def _workspace(workspace, like):
    if workspace is None:
        return None, 0
    _on_device_of(workspace, "workspace", like)
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def embedding_lookup(table, tokens, scale=1.0, out=None):
    """out[i, :] = scale * table[tokens[i], :], the rows of an embedding table by token.

    table: [vocab x n_cols] row-major (rows may be strided), float32 / float16 / bfloat16; tokens: int32 / int64 of
    any shape, contiguous; out: [tokens.numel() x n_cols] of the table's type (default: a new tensor of shape
    tokens.shape + (n_cols,)). A token outside [0, vocab) - the -1 of padded positions - gives a row of zeros.
    Outside autograd (embedding_grad is the gradient). Returns out."""
    _require_cuda(table, "table")
    if table.dim() != 2:
        raise ValueError("table must be a matrix")
    _on_device_of(tokens, "tokens", table)
    dt, tt = _VOCAB_DTYPES.get(table.dtype), _TOKEN_DTYPES.get(tokens.dtype)
    if dt is None or tt is None:
        raise L.B2RError(L.ERR_UNSUPPORTED, "embedding_lookup")
    if not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous")
    vocab, n_cols = table.shape
    n = tokens.numel()
    ldt = _row_stride(table, "table")
    if out is None:
        out = torch.empty(tokens.shape + (n_cols,), dtype=table.dtype, device=table.device)
        ldo = n_cols
    else:
        _on_device_of(out, "out", table)
        if out.dtype != table.dtype:
            raise ValueError("out and table must have the same element type")
        rows = _as_rows(out, n, n_cols, "out")
        ldo = _row_stride(rows, "out")
        if _overlap(out, table) or _overlap(out, tokens):
            raise ValueError("out must not overlap table or tokens")
    with _on(table.device):
        st = L.load().b2r_embedding_lookup(out.data_ptr(), ldo, table.data_ptr(), ldt, tokens.data_ptr(), dt, tt, n,
                                           n_cols, vocab, float(scale), _stream_ptr(table.device))
    L.check(st, "b2r_embedding_lookup")
    return out


def _as_rows(t, n, n_cols, name):
    """`t` as a matrix of n rows of n_cols, without a copy."""
    if t.dim() < 1 or t.shape[-1] != n_cols or t.numel() != n * n_cols:
        raise ValueError(f"{name} must have {n} rows of {n_cols}")
    if t.dim() == 2:
        return t
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous or a row-major matrix")
    return t.reshape(n, n_cols)


def embedding_grad(grad_out, tokens, vocab, scale=1.0, grad_table=None, accumulate=False, out_dtype=None,
                   workspace=None):
    """Gradient of embedding_lookup with respect to its table:
    grad_table[v, :] = scale * sum of grad_out[i, :] over the positions i with tokens[i] == v.

    grad_out: [tokens.numel() x n_cols] (or tokens.shape + (n_cols,), contiguous), float32 / float16 / bfloat16;
    grad_table: [vocab x n_cols] of the same type or float32 (default: a new tensor of type `out_dtype`, else
    grad_out's). With `accumulate` the sums are added to what grad_table holds; without, rows that no token names
    are set to zero. Tokens outside [0, vocab) add nothing. Sums are in float32 in an order that the positions alone
    determine: results repeat bit for bit. `workspace` (uint8, see embedding_grad_workspace_bytes) keeps the call
    allocation-free. Returns grad_table."""
    _require_cuda(grad_out, "grad_out")
    _on_device_of(tokens, "tokens", grad_out)
    dt, tt = _VOCAB_DTYPES.get(grad_out.dtype), _TOKEN_DTYPES.get(tokens.dtype)
    if dt is None or tt is None:
        raise L.B2RError(L.ERR_UNSUPPORTED, "embedding_grad")
    if not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous")
    if grad_out.dim() < 1:
        raise ValueError("grad_out must be a matrix")
    vocab, n, n_cols = int(vocab), tokens.numel(), grad_out.shape[-1]
    if vocab < 0:
        raise ValueError("vocab must not be negative")
    ldo = _row_stride(_as_rows(grad_out, n, n_cols, "grad_out"), "grad_out")
    if grad_table is None:
        if accumulate:
            raise ValueError("accumulate needs a grad_table")
        grad_table = torch.empty((vocab, n_cols), dtype=out_dtype or grad_out.dtype, device=grad_out.device)
        ldg = n_cols
    else:
        _on_device_of(grad_table, "grad_table", grad_out)
        if tuple(grad_table.shape) != (vocab, n_cols):
            raise ValueError("grad_table is not of size vocab * n_cols")
        if out_dtype is not None and out_dtype != grad_table.dtype:
            raise ValueError("grad_table is not of type out_dtype")
        ldg = _row_stride(grad_table, "grad_table")
        if _overlap(grad_table, grad_out) or _overlap(grad_table, tokens):
            raise ValueError("grad_table must not overlap grad_out or tokens")
    if grad_table.dtype not in (grad_out.dtype, torch.float32):
        raise L.B2RError(L.ERR_UNSUPPORTED, "embedding_grad")
    ws_ptr, ws_bytes = _workspace(workspace, grad_out)
    with _on(grad_out.device):
        st = L.load().b2r_embedding_grad(
            grad_table.data_ptr(), ldg, _VOCAB_DTYPES[grad_table.dtype], grad_out.data_ptr(), ldo, dt,
            tokens.data_ptr(), tt, n, n_cols, vocab, float(scale), 1 if accumulate else 0, ws_ptr, ws_bytes,
            _stream_ptr(grad_out.device))
    L.check(st, "b2r_embedding_grad")
    return grad_table


def embedding_grad_workspace_bytes(grad_out, vocab):
    """Bytes of workspace that embedding_grad takes for rows of grad_out's shape."""
    n_cols = grad_out.shape[-1]
    n = grad_out.numel() // n_cols if n_cols else 0
    with _on(grad_out.device):
        return L.load().b2r_embedding_grad_workspace_bytes(n, n_cols, int(vocab))


def _distill_args(logits, teacher_ids, teacher_logits, temperature, where):
    """The checks the distillation calls share: (dtype, id dtype, teacher dtype, row strides, rows, vocab, k)."""
    _require_cuda(logits, "logits")
    _on_device_of(teacher_ids, "teacher_ids", logits)
    _on_device_of(teacher_logits, "teacher_logits", logits)
    if logits.dim() != 2 or teacher_ids.dim() != 2 or teacher_logits.dim() != 2:
        raise ValueError("logits, teacher_ids and teacher_logits must be matrices")
    dt, it, tt = (_VOCAB_DTYPES.get(logits.dtype), _TOKEN_DTYPES.get(teacher_ids.dtype),
                  _VOCAB_DTYPES.get(teacher_logits.dtype))
    if dt is None or it is None or tt is None:
        raise L.B2RError(L.ERR_UNSUPPORTED, where)
    n, vocab = logits.shape
    if teacher_ids.shape[0] != n or teacher_ids.shape != teacher_logits.shape:
        raise ValueError("teacher_ids and teacher_logits must have a row of the same length for every row of logits")
    if not 1e-30 <= float(temperature) <= 1e30:
        raise ValueError("temperature must be positive and finite (1e-30 to 1e30)")
    return (dt, it, tt, _row_stride(logits, "logits"), _row_stride(teacher_ids, "teacher_ids"),
            _row_stride(teacher_logits, "teacher_logits"), n, vocab, teacher_ids.shape[1])


def _per_row(t, name, n, logits):
    """A contiguous float32 vector with an element per row of logits."""
    _on_device_of(t, name, logits)
    if t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 of size n_rows")
    return t


def _grad_like(grad, logits, ldl):
    """`grad`, checked, or a new matrix whose row stride differs from logits' by a multiple of 16 bytes (so that rows of
    both have the same alignment) and is as short as that allows: logits may be rows far apart, the last positions of
    sequences, say."""
    if grad is None:
        n, vocab = logits.shape
        ldg = vocab + (ldl - vocab) % (16 // logits.element_size())
        grad = torch.empty_strided((n, vocab), (max(ldg, 1), 1), dtype=logits.dtype, device=logits.device)
        return grad, ldg
    _on_device_of(grad, "grad", logits)
    if grad.dtype != logits.dtype or grad.shape != logits.shape:
        raise ValueError("grad must have the shape and element type of logits")
    ldg = _row_stride(grad, "grad")
    if _overlap(grad, logits) and (grad.data_ptr() != logits.data_ptr() or ldg != ldl):
        raise ValueError("grad must be logits or not overlap them")
    return grad, ldg


def _apart(outputs, inputs):
    """Refuses given outputs (name, tensor or None) that overlap an input or one another."""
    for i, (name, out) in enumerate(outputs):
        if out is None:
            continue
        for other_name, other in inputs + outputs[:i]:
            if other is not None and _overlap(out, other):
                raise ValueError(f"{name} must not overlap {other_name}")


def _distill(where, logits, teacher_ids, teacher_logits, grad_loss, temperature, loss, lse, grad, want_grad):
    dt, it, tt, ldl, ldi, ldt, n, vocab, k = _distill_args(logits, teacher_ids, teacher_logits, temperature, where)
    if loss is not None or lse is not None or grad is not None:
        lists = [("teacher_ids", teacher_ids), ("teacher_logits", teacher_logits), ("grad_loss", grad_loss)]
        _apart([("loss", loss), ("lse", lse)], lists + [("logits", logits)])
        _apart([("grad", grad)], lists + [("loss", loss), ("lse", lse)])
    loss = torch.empty(n, dtype=torch.float32, device=logits.device) if loss is None else \
        _per_row(loss, "loss", n, logits)
    lse = torch.empty(n, dtype=torch.float32, device=logits.device) if lse is None else _per_row(lse, "lse", n, logits)
    g_ptr, ldg, gl_ptr = None, 0, None
    if want_grad:
        gl_ptr = _per_row(grad_loss, "grad_loss", n, logits).data_ptr()
        grad, ldg = _grad_like(grad, logits, ldl)
        g_ptr = grad.data_ptr() or None
    with _on(logits.device):
        st = L.load().b2r_topk_distill(
            loss.data_ptr(), lse.data_ptr(), g_ptr, ldg, gl_ptr, logits.data_ptr(), ldl, dt, teacher_ids.data_ptr(),
            ldi, it, teacher_logits.data_ptr(), ldt, tt, n, vocab, k, float(temperature),
            _stream_ptr(logits.device))
    L.check(st, "b2r_topk_distill")
    return loss, lse, grad


def topk_distill(logits, teacher_ids, teacher_logits, temperature=1.0, loss=None, lse=None):
    """Distillation loss of every row of student logits against a teacher's top logits:

      p = softmax(teacher_logits / T) over the entries whose token lies in [0, vocab)
      loss = T^2 * sum_k p_k (log p_k - log softmax(logits / T)[teacher_ids_k]),  lse = log sum exp(logits / T)

    logits: [n_rows x vocab] row-major (rows may be strided), float32 / float16 / bfloat16; teacher_ids: [n_rows x k]
    int32 / int64, -1 where a list is shorter than k; teacher_logits: [n_rows x k], any of the three types; k <= 1024.
    A row without a valid entry has loss 0. Outside autograd (topk_distill_grad is the gradient, topk_distill_step
    returns both). Returns (loss, lse), float32 vectors."""
    loss, lse, _ = _distill("topk_distill", logits, teacher_ids, teacher_logits, None, temperature, loss, lse, None,
                            False)
    return loss, lse


def topk_distill_step(logits, teacher_ids, teacher_logits, grad_loss, temperature=1.0, loss=None, lse=None,
                      grad=None):
    """topk_distill and its gradient in one pass over the logits: grad = grad_loss[:, None] * d loss / d logits for
    a given weight of every row (float32 [n_rows], 1 / n_rows for a mean). `grad` may be `logits`. Returns
    (loss, lse, grad)."""
    return _distill("topk_distill_step", logits, teacher_ids, teacher_logits, grad_loss, temperature, loss, lse, grad,
                    True)


def topk_distill_grad(logits, teacher_ids, teacher_logits, lse, grad_loss, temperature=1.0, grad=None):
    """The gradient of topk_distill alone, from the lse that it returned:
    grad[r, v] = grad_loss[r] * T * (softmax(logits / T)[r, v] - sum of p_k with teacher_ids[r, k] == v).
    The softmax carries the rounding of the float32 lse, a factor of 1 +- |lse| 2^-24; where that is too much (low
    temperatures, large logits) topk_distill_step has the gradient without it. `grad` may be `logits`. Returns grad."""
    dt, it, tt, ldl, ldi, ldt, n, vocab, k = _distill_args(logits, teacher_ids, teacher_logits, temperature,
                                                           "topk_distill_grad")
    _per_row(lse, "lse", n, logits)
    _per_row(grad_loss, "grad_loss", n, logits)
    _apart([("grad", grad)], [("teacher_ids", teacher_ids), ("teacher_logits", teacher_logits), ("lse", lse),
                              ("grad_loss", grad_loss)])
    grad, ldg = _grad_like(grad, logits, ldl)
    with _on(logits.device):
        st = L.load().b2r_topk_distill_grad(
            grad.data_ptr(), ldg, lse.data_ptr(), grad_loss.data_ptr(), logits.data_ptr(), ldl, dt,
            teacher_ids.data_ptr(), ldi, it, teacher_logits.data_ptr(), ldt, tt, n, vocab, k, float(temperature),
            _stream_ptr(logits.device))
    L.check(st, "b2r_topk_distill_grad")
    return grad


def _sample_param(value, name, dtype, n, logits):
    """(tensor or None, value for all rows) of a sampling parameter given as a number or as a tensor."""
    if isinstance(value, torch.Tensor):
        _on_device_of(value, name, logits)
        if value.dtype != dtype or value.numel() != n or not value.is_contiguous():
            raise ValueError(f"{name} must be a number or contiguous {dtype} of size n_rows")
        return value.data_ptr(), 0
    return None, value


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, logprobs=None,
                  index_dtype=torch.int32):
    """One token for every row of logits, from a uniform number in [0, 1) for each row. In the order of falling logits
    (equal ones by rising token) the first `top_k` are kept (0: all), of those the tokens whose probability is at
    least `min_p` of the largest, of those the shortest beginning of the order that holds at least `top_p` of their
    probability; the drawn token is the first kept one, by token number, at which the running probability under
    `temperature` exceeds uniform times the kept one. temperature <= 0 takes the largest logit.

    logits: [n_rows x vocab] row-major (rows may be strided), float32 / float16 / bfloat16; uniform: float32 [n_rows];
    the parameters are numbers or vectors of n_rows (int32 for top_k, float32 for the others). NaN logits count as
    -inf; a row of -inf alone gives -1; vocab is at most 16777216. Returns (tokens, logprobs): int32 or int64, and the
    float32 log of the probability with which each token was drawn."""
    _require_cuda(logits, "logits")
    if logits.dim() != 2:
        raise ValueError("logits must be a matrix")
    dt = _VOCAB_DTYPES.get(logits.dtype)
    if dt is None:
        raise L.B2RError(L.ERR_UNSUPPORTED, "sample_tokens")
    n, vocab = logits.shape
    ldl = _row_stride(logits, "logits")
    _per_row(uniform, "uniform", n, logits)
    if out is not None or logprobs is not None:
        _apart([("out", out), ("logprobs", logprobs)], [("logits", logits), ("uniform", uniform)] + [
            (name, v) for name, v in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p),
                                      ("min_p", min_p)) if isinstance(v, torch.Tensor)])
    if out is None:
        out = torch.empty(n, dtype=index_dtype, device=logits.device)
    _on_device_of(out, "out", logits)
    if out.numel() != n or not out.is_contiguous():
        raise ValueError("out must be contiguous, of size n_rows")
    ot = _TOKEN_DTYPES.get(out.dtype)
    if ot is None:
        raise L.B2RError(L.ERR_UNSUPPORTED, "sample_tokens")
    logprobs = torch.empty(n, dtype=torch.float32, device=logits.device) if logprobs is None else \
        _per_row(logprobs, "logprobs", n, logits)
    temp_ptr, temp = _sample_param(temperature, "temperature", torch.float32, n, logits)
    k_ptr, k = _sample_param(top_k, "top_k", torch.int32, n, logits)
    p_ptr, p = _sample_param(top_p, "top_p", torch.float32, n, logits)
    m_ptr, m = _sample_param(min_p, "min_p", torch.float32, n, logits)
    desc = L.SampleDesc(dt, ot, n, vocab, ldl, temp_ptr, k_ptr, p_ptr, m_ptr, temp,
                        max(0, min(int(k), 0x7fffffff)), p, m)
    with _on(logits.device):
        st = L.load().b2r_sample_tokens(desc, out.data_ptr(), logprobs.data_ptr(), logits.data_ptr(),
                                        uniform.data_ptr(), _stream_ptr(logits.device))
    L.check(st, "b2r_sample_tokens")
    return out, logprobs


def last_kernel_status(device, clear=True):
    """Synchronises `device` and returns L.OK, or L.ERR_TIMEOUT if a bounded wait inside a kernel of any
    earlier call on that device ran out (that call's unfinished floating-point outputs are NaN)."""
    import ctypes
    torch.cuda.synchronize(device)
    out = ctypes.c_int32(0)
    with _on(device):
        L.check(L.load().b2r_last_kernel_status(ctypes.byref(out), 1 if clear else 0), "b2r_last_kernel_status")
    return out.value


def set_wait_limit_ms(ms):
    """Bound of every wait inside the kernels that stage tiles through shared memory; 0 = the default."""
    L.check(L.load().b2r_set_wait_limit_ms(int(ms)), "b2r_set_wait_limit_ms")


def _matrix_arg(fn_name, data, out, index_dtype):
    _require_cuda(data, "in")
    if data.dim() != 2 or not data.is_contiguous():
        raise ValueError("in must be a row-major matrix")
    n_rows, n_cols = data.shape
    if out is None:
        out = torch.empty(n_rows, dtype=index_dtype, device=data.device)
    if out.numel() != n_rows:
        raise ValueError("Size of output vector must equal number of rows in input matrix.")
    if data.dtype not in (torch.float32, torch.float64) or out.dtype not in (torch.int32, torch.int64):
        raise L.B2RError(L.ERR_UNSUPPORTED, fn_name)
    with _on(data.device):
        st = getattr(L.load(), fn_name)(out.data_ptr(), _DTYPES[out.dtype], data.data_ptr(), _DTYPES[data.dtype],
                                        n_rows, n_cols, _stream_ptr(data.device))
    L.check(st, fn_name)
    return out


def argmin(data, out=None, index_dtype=torch.int32):
    """raft::matrix::argmin (matrix/argmin.cuh:27-39): index of the smallest element of every row
    of a row-major matrix, lowest index on ties."""
    return _matrix_arg("b2r_matrix_argmin", data, out, index_dtype)


def argmax(data, out=None, index_dtype=torch.int32):
    """raft::matrix::argmax (matrix/argmax.cuh:27-39): index of the largest element of every row,
    lowest index on ties."""
    return _matrix_arg("b2r_matrix_argmax", data, out, index_dtype)


def map_reduce(data, map_op="identity", reduce_op="add", neutral=0.0, out=None, out_dtype=None, workspace=None):
    """raft::linalg::mapReduce / mapThenSumReduce for the named map functors
    (linalg/map_reduce.cuh:43-103, linalg/map_then_reduce.cuh:37-53):
    out[0] = reduce_op over i of map_op(data[i]); `neutral` is the identity of reduce_op.
    `data` is any contiguous tensor, read as a flat array. Returns a one-element tensor."""
    _require_cuda(data, "data")
    if not data.is_contiguous():
        raise ValueError("Input must be contiguous")
    flat = data.reshape(1, -1)
    if out is None:
        out = torch.empty(1, dtype=out_dtype or data.dtype, device=data.device)
    return reduce(flat, ALONG_ROWS, out, init=neutral, main_op=map_op, reduce_op=reduce_op, workspace=workspace)


def row_normalize(data, norm_type="L2", out=None, eps=1e-8):
    """raft::linalg::row_normalize<norm_type> (linalg/normalize.cuh:88-107): every row of a
    row-major matrix divided by its L1 / L2 / Linf norm. A row whose norm is <= eps is not
    written: `out` keeps what it held there (the reference's behaviour), so pass an initialised
    `out` if such rows can occur. `out` may be `data`."""
    _require_cuda(data, "data")
    if data.dim() != 2 or not data.is_contiguous():
        raise ValueError("Input must be contiguous")
    if out is None:
        out = torch.zeros_like(data)
    _require_cuda(out, "out")
    if not out.is_contiguous():
        raise ValueError("Output must be contiguous")
    if out.shape[0] != data.shape[0]:
        raise ValueError("The number of rows of the input and output should be equal")
    if out.shape[1] != data.shape[1]:
        raise ValueError("The number of columns of the input and output should be equal")
    if out.dtype != data.dtype:
        raise ValueError("input and output must have the same element type")
    if norm_type not in ("L1", "L2", "Linf"):
        raise ValueError("Unsupported norm type: %s" % norm_type)
    n_rows, n_cols = data.shape
    with _on(data.device):
        st = L.load().b2r_row_normalize(out.data_ptr(), data.data_ptr(), _DTYPES[data.dtype], n_rows, n_cols,
                                        _NORM[norm_type], float(eps), _stream_ptr(data.device))
    L.check(st, "b2r_row_normalize")
    return out


def probe_empty_launch(device):
    """One empty kernel on the device's current stream (the cost floor of an event pair around a launch)."""
    with _on(device):
        L.check(L.load().b2r_probe_empty_launch(_stream_ptr(device)), "b2r_probe_empty_launch")


def probe_stream_read(data):
    """Reads `data` once with plain streaming loads and does nothing else (the read floor of its size)."""
    _require_cuda(data, "data")
    with _on(data.device):
        L.check(L.load().b2r_probe_stream_read(data.data_ptr(), data.numel() * data.element_size(), None,
                                               _stream_ptr(data.device)), "b2r_probe_stream_read")


def reload_tuning():
    """Makes the library read its B2R_* environment knobs again (they are otherwise read once, at the
    first call). For tests and sweeps that change them within one process."""
    L.check(L.load().b2r_reload_tuning(), "b2r_reload_tuning")


def apply_final(v, final_op, final_scalar=1.0):
    """v[i] = final_op(v[i]) in place (the deferred final step of a sharded reduction)."""
    _require_cuda(v, "v")
    with _on(v.device):
        st = L.load().b2r_apply_final(v.data_ptr(), _DTYPES[v.dtype], v.numel(), _FINAL[final_op],
                                      float(final_scalar), _stream_ptr(v.device))
    L.check(st, "b2r_apply_final")
    return v


def synth_fill(dst, seed, kind, lo=0.0, hi=1.0, first_index=0):
    """Fills `dst` (any shape, contiguous) with the counter-based synthetic data of
    b2r_synth_fill: kind "uniform", "normal" or "int"."""
    _require_cuda(dst, "dst")
    if not dst.is_contiguous():
        raise ValueError("dst must be contiguous")
    k = {"uniform": 0, "normal": 1, "int": 2}[kind]
    with _on(dst.device):
        st = L.load().b2r_synth_fill(dst.data_ptr(), _DTYPES[dst.dtype], dst.numel(), first_index, seed, k,
                                     float(lo), float(hi), _stream_ptr(dst.device))
    L.check(st, "b2r_synth_fill")
    return dst
