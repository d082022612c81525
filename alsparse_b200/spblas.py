"""Host-side mirror of the reference's operator interface for the CSR mv / mm path.

Same names, argument order and status codes as the C API (include/alphasparse/spapi.h); the
functions take numpy arrays (host pointers) or torch CUDA tensors (device pointers) where the
C API takes pointers and return the ``alphasparse_status_t`` as an int, so a test written
against the reference's C entry points reads the same here:

    st, A = create_coo('s', BASE_ZERO, rows, cols, nnz, ri, ci, v)
    st, B = convert_csr(A, NON_TRANSPOSE)
    st = mv('s', NON_TRANSPOSE, 2.0, B, descr(GENERAL), x, 2.0, y)      # y updated in place
"""
import ctypes as C

import numpy as np

from . import capi
from .capi import (BASE_ONE, BASE_ZERO, COLUMN_MAJOR, GENERAL, NON_TRANSPOSE, ROW_MAJOR, SUCCESS,  # noqa: F401
                   TRANSPOSE, MatInfo, MatrixDescr)

_NP = {"s": np.float32, "d": np.float64}


def descr(type_=capi.GENERAL, mode=0, diag=0):
    return MatrixDescr(type_, mode, diag)


def _ptr(a):
    """Raw address of a numpy array, a torch tensor, an int address or None."""
    if a is None:
        return None
    if isinstance(a, int):
        return a
    if isinstance(a, np.ndarray):
        return a.ctypes.data
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    raise TypeError(f"cannot take the address of {type(a)!r}")


def _i32(a):
    return None if a is None else np.ascontiguousarray(a, dtype=np.int32)


def create_csr(kind, indexing, rows, cols, rows_start, rows_end, col_indx, values):
    """alphasparse_{s,d}_create_csr.  Returns (status, handle)."""
    lib = capi.load()
    rs, re_, ci = _i32(rows_start), _i32(rows_end), _i32(col_indx)
    v = None if values is None else np.ascontiguousarray(values, dtype=_NP.get(kind, np.float32))
    h = C.c_void_p()
    st = getattr(lib, f"alphasparse_{kind}_create_csr")(C.byref(h), indexing, rows, cols, _ptr(rs), _ptr(re_),
                                                         _ptr(ci), _ptr(v))
    return st, h


def create_coo(kind, indexing, rows, cols, nnz, row_indx, col_indx, values):
    """alphasparse_{s,d}_create_coo.  Returns (status, handle)."""
    lib = capi.load()
    ri, ci = _i32(row_indx), _i32(col_indx)
    v = None if values is None else np.ascontiguousarray(values, dtype=_NP.get(kind, np.float32))
    h = C.c_void_p()
    st = getattr(lib, f"alphasparse_{kind}_create_coo")(C.byref(h), indexing, rows, cols, nnz, _ptr(ri), _ptr(ci),
                                                         _ptr(v))
    return st, h


def convert_csr(source, operation=capi.NON_TRANSPOSE):
    """alphasparse_convert_csr.  Returns (status, handle)."""
    h = C.c_void_p()
    st = capi.load().alphasparse_convert_csr(source, operation, C.byref(h))
    return st, h


def export_csr(kind, source):
    """alphasparse_{s,d}_export_csr.  Returns (status, base, rows, cols, rows_start, rows_end, col_indx,
    values); the arrays are numpy views of the handle's own storage (borrowed, like the C pointers)."""
    lib = capi.load()
    base, rows, cols = C.c_int(), C.c_int32(), C.c_int32()
    rs, re_, ci, v = C.c_void_p(), C.c_void_p(), C.c_void_p(), C.c_void_p()
    st = getattr(lib, f"alphasparse_{kind}_export_csr")(source, C.byref(base), C.byref(rows), C.byref(cols),
                                                         C.byref(rs), C.byref(re_), C.byref(ci), C.byref(v))
    if st != SUCCESS:
        return (st,) + (None,) * 7
    m = rows.value

    def view(p, n, ct):
        if n == 0 or not p.value:
            return np.zeros(0, dtype=np.dtype(ct))
        return np.ctypeslib.as_array(C.cast(p, C.POINTER(ct)), shape=(n,))

    ptr = view(rs, m + 1, C.c_int32)
    nnz = int(ptr[m] - ptr[0]) if m > 0 else 0
    ct = C.c_float if kind == "s" else C.c_double
    return (st, base.value, m, cols.value, ptr[:m], ptr[1:m + 1] if m > 0 else ptr[:0], view(ci, nnz, C.c_int32),
            view(v, nnz, ct))


def create_csc(kind, indexing, rows, cols, cols_start, cols_end, row_indx, values):
    """alphasparse_{s,d}_create_csc.  Returns (status, handle)."""
    lib = capi.load()
    cs, ce, ri = _i32(cols_start), _i32(cols_end), _i32(row_indx)
    v = None if values is None else np.ascontiguousarray(values, dtype=_NP.get(kind, np.float32))
    h = C.c_void_p()
    st = getattr(lib, f"alphasparse_{kind}_create_csc")(C.byref(h), indexing, rows, cols, _ptr(cs), _ptr(ce),
                                                         _ptr(ri), _ptr(v))
    return st, h


def convert_csc(source, operation=capi.NON_TRANSPOSE):
    """alphasparse_convert_csc (COO source).  Returns (status, handle)."""
    h = C.c_void_p()
    st = capi.load().alphasparse_convert_csc(source, operation, C.byref(h))
    return st, h


def export_csc(kind, source):
    """alphasparse_{s,d}_export_csc.  Returns (status, base, rows, cols, cols_start, cols_end, row_indx, values)
    as borrowed numpy views, like export_csr."""
    lib = capi.load()
    base, rows, cols = C.c_int(), C.c_int32(), C.c_int32()
    cs, ce, ri, v = C.c_void_p(), C.c_void_p(), C.c_void_p(), C.c_void_p()
    st = getattr(lib, f"alphasparse_{kind}_export_csc")(source, C.byref(base), C.byref(rows), C.byref(cols),
                                                         C.byref(cs), C.byref(ce), C.byref(ri), C.byref(v))
    if st != SUCCESS:
        return (st,) + (None,) * 7
    n = cols.value

    def view(p, k, ct):
        if k == 0 or not p.value:
            return np.zeros(0, dtype=np.dtype(ct))
        return np.ctypeslib.as_array(C.cast(p, C.POINTER(ct)), shape=(k,))

    ptr = view(cs, n + 1, C.c_int32)
    nnz = int(ptr[n] - ptr[0]) if n > 0 else 0
    ct = C.c_float if kind == "s" else C.c_double
    return (st, base.value, rows.value, n, ptr[:n], ptr[1:n + 1] if n > 0 else ptr[:0], view(ri, nnz, C.c_int32),
            view(v, nnz, ct))


def destroy(handle):
    return capi.load().alphasparse_destroy(handle)


def mv(kind, operation, alpha, A, descr_, x, beta, y):
    """alphasparse_{s,d}_mv: y = alpha*op(A)*x + beta*y, y updated in place.  Returns the status."""
    return getattr(capi.load(), f"alphasparse_{kind}_mv")(operation, alpha, A, descr_, _ptr(x), beta, _ptr(y))


def mm(kind, operation, alpha, A, descr_, layout, x, columns, ldx, beta, y, ldy):
    """alphasparse_{s,d}_mm: Y = alpha*op(A)*X + beta*Y, Y updated in place.  Returns the status."""
    return getattr(capi.load(), f"alphasparse_{kind}_mm")(operation, alpha, A, descr_, layout, _ptr(x), columns, ldx,
                                                           beta, _ptr(y), ldy)


def optimize(A):
    """alphasparse_optimize: re-runs the analysis of the handle."""
    return capi.load().alphasparse_optimize(A)


def mat_info(A):
    info = MatInfo()
    st = capi.load().alphasparse_cuda_get_mat_info(A, C.byref(info))
    return st, info


def device_csr(A):
    """(status, d_row_ptr, d_col_indx, d_values) as integer device addresses."""
    a, b, c = C.c_void_p(), C.c_void_p(), C.c_void_p()
    st = capi.load().alphasparse_cuda_get_device_csr(A, C.byref(a), C.byref(b), C.byref(c))
    return st, a.value, b.value, c.value


def set_stream(stream_ptr):
    return capi.load().alphasparse_cuda_set_stream(stream_ptr)


def set_algorithm(alg):
    return capi.load().alphasparse_cuda_set_algorithm(alg)


def set_option(name, value):
    """alphasparse_cuda_set_option: a tuning value of the analysis (negative restores the default)."""
    return capi.load().alphasparse_cuda_set_option(name.encode(), int(value))


def get_option(name):
    v = C.c_int64()
    st = capi.load().alphasparse_cuda_get_option(name.encode(), C.byref(v))
    assert st == SUCCESS, capi.STATUS_NAMES[st]
    return v.value


def launch_count():
    return capi.load().alphasparse_cuda_launch_count()


def last_error():
    return capi.load().alphasparse_cuda_last_error().decode()


def partition_rows_by_nnz(rows_end, parts):
    """balanced_partition_row_by_nnz: nnz-balanced contiguous row split, parts+1 boundaries."""
    acc = _i32(rows_end)
    out = np.zeros(parts + 1, dtype=np.int32)
    capi.load().balanced_partition_row_by_nnz(_ptr(acc), len(acc), parts, _ptr(out))
    return out


def kernel_status(A, clear=False):
    """alphasparse_cuda_kernel_status: (status, code) -- the error word of the handle's kernels (0 = fine)."""
    code = C.c_int()
    st = capi.load().alphasparse_cuda_kernel_status(A, C.byref(code), 1 if clear else 0)
    return st, code.value


def profile_kernel(A, enable=True):
    return capi.load().alphasparse_cuda_profile_kernel(A, 1 if enable else 0)


def kernel_ms(A):
    """Duration in ms of the dominant kernel of the last mv / mm call on A (profiling enabled)."""
    ms = C.c_float()
    st = capi.load().alphasparse_cuda_kernel_ms(A, C.byref(ms))
    assert st == SUCCESS, capi.STATUS_NAMES[st]
    return ms.value


def release_cached_memory():
    """alphasparse_cuda_release_cached_memory: what the library keeps for later calls goes back to CUDA."""
    return capi.load().alphasparse_cuda_release_cached_memory()


def csrmv_noalloc(rows, cols, nnz, alpha, d_row_ptr, d_col_indx, d_values, d_x, beta, d_y):
    """alphasparse_cuda_d_csrmv_noalloc: double-precision SpMV on device arrays that never allocates
    (scratch lives in a fixed 4 MiB array inside the library; rows + nnz <= 375,802,112)."""
    return capi.load().alphasparse_cuda_d_csrmv_noalloc(rows, cols, nnz, alpha, _ptr(d_row_ptr), _ptr(d_col_indx),
                                                         _ptr(d_values), _ptr(d_x), beta, _ptr(d_y))


def read_coo(kind, path):
    """alpha_read_coo / alpha_read_coo_d: (rows, cols, row_indx, col_indx, values) as numpy copies (zero-based)."""
    lib = capi.load()
    m, n, nnz = C.c_int32(), C.c_int32(), C.c_int32()
    ri, ci, v = C.c_void_p(), C.c_void_p(), C.c_void_p()
    getattr(lib, "alpha_read_coo" if kind == "s" else "alpha_read_coo_d")(path.encode(), C.byref(m), C.byref(n),
                                                                          C.byref(nnz), C.byref(ri), C.byref(ci),
                                                                          C.byref(v))
    if nnz.value < 0:
        raise OSError(f"cannot read {path}")
    k = nnz.value

    def take(p, ct):
        a = np.ctypeslib.as_array(C.cast(p, C.POINTER(ct)), shape=(max(k, 1),))[:k].copy()
        lib.alpha_free(p)
        return a
    return m.value, n.value, take(ri, C.c_int32), take(ci, C.c_int32), take(v, C.c_float if kind == "s" else C.c_double)


# ---- products of matrices that are made at run time (device tensors) ------------------------------------------
# Calls of a few microseconds: each operand's properties are read once.

_TYPES = {"float32": capi.TYPE_F32, "float16": capi.TYPE_F16, "bfloat16": capi.TYPE_BF16}
_INDICES = {"int32": capi.INDEX_I32, "int64": capi.INDEX_I64}
_NONE = -1                # element type that the library has no name for: it refuses the value
_KINDS = {}               # element type of torch or numpy -> (enum of a value, enum of an index), -1 for none


def _kind(a):
    kind = _KINDS.get(a.dtype)
    if kind is None:
        name = str(a.dtype).replace("torch.", "")
        kind = _KINDS[a.dtype] = (_TYPES.get(name, _NONE), _INDICES.get(name, _NONE))
    return kind


def _type(a):
    return _kind(a)[0]


def _f32(a):
    return _kind(a)[0] == capi.TYPE_F32


def _i32s(a):
    return _kind(a)[1] == capi.INDEX_I32


def _np_strides(a):
    return tuple(s // a.itemsize for s in a.strides)


def _matrix(a):
    """(rows, columns, leading dimension, address) of a row-major numpy array or torch tensor whose rows are contiguous, None if it
    is not one (the caller's view has to be copied first)."""
    try:
        rows, width = a.shape
    except ValueError:
        return None
    if isinstance(a, np.ndarray):
        (ld, step), at = _np_strides(a), a.ctypes.data
    else:
        (ld, step), at = a.stride(), a.data_ptr()
    if step != 1 and width > 1:
        return None
    return rows, width, ld if rows > 1 or ld > width else width, at


def _vector(a):
    """(elements, distance, address) of an array of one dimension, None if it has another number of them."""
    try:
        n, = a.shape
    except ValueError:
        return None
    if isinstance(a, np.ndarray):
        (step,), at = _np_strides(a), a.ctypes.data
    else:
        (step,), at = a.stride(), a.data_ptr()
    return n, step if n > 1 else 1, at


def _matrices(a):
    """(matrices, rows, columns, leading dimension, distance of the matrices, address) of an array of three dimensions."""
    try:
        n, rows, width = a.shape
    except ValueError:
        return None
    if isinstance(a, np.ndarray):
        (apart, ld, step), at = _np_strides(a), a.ctypes.data
    else:
        (apart, ld, step), at = a.stride(), a.data_ptr()
    if step != 1 and width > 1:
        return None
    ld = ld if rows > 1 or ld > width else width
    return n, rows, width, ld, apart if n > 1 or apart > ld * rows else ld * rows, at


def _buffer(b):
    """Address and bytes of a workspace: a contiguous array, or None; (None, -1) if its elements are apart."""
    if b is None:
        return None, 0
    if not (b.flags.c_contiguous if isinstance(b, np.ndarray) else b.is_contiguous()):
        return None, -1
    return _ptr(b), b.nbytes


def embedding(tokens, table, scale, y):
    """alphasparse_cuda_embedding: y[i] = scale * table[tokens[i]].  tokens: one dimension of int32 or int64, at any distance above 0;
    table (vocab, width) and y (tokens, width) of one type, rows contiguous.  Returns the status."""
    t, e, o = _vector(tokens), _matrix(table), _matrix(y)
    if t is None or e is None or o is None or y.dtype != table.dtype or o[0] != t[0] or o[1] != e[1]:
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_embedding(_kind(tokens)[1], _kind(table)[0], t[0], t[2], t[1], e[0], e[1], scale, e[3], e[2], o[3], o[2])


def embedding_grad_buffer_size(tokens, vocab, width):
    """(status, bytes of the workspace) of embedding_grad."""
    n = C.c_size_t()
    st = capi.load().alphasparse_cuda_embedding_grad_buffer_size(tokens, vocab, width, C.byref(n))
    return st, n.value


def embedding_grad(tokens, dy, alpha, beta, dtable, buffer):
    """alphasparse_cuda_embedding_grad: dtable[v] = alpha * (sum of dy[i] where tokens[i] == v) + beta * dtable[v].
    Returns the status."""
    t, d, o = _vector(tokens), _matrix(dy), _matrix(dtable)
    if t is None or d is None or o is None or d[0] != t[0] or d[1] != o[1]:
        return capi.INVALID_VALUE
    at, size = _buffer(buffer)
    if size < 0:
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_embedding_grad(_kind(tokens)[1], _kind(dy)[0], _kind(dtable)[0], t[0], t[2], t[1], o[0], o[1], alpha,
                                                       d[3], d[2], beta, o[3], o[2], at, size)


def route(score, logits, bias, groups, top_groups, renormalize, scale, index, weight):
    """alphasparse_cuda_route: the experts index (tokens, k; int32) of each row of logits (tokens, experts) and their
    weights (tokens, k; float32); bias: (experts,) float32 or None.  Returns the status."""
    x, i, w = _matrix(logits), _matrix(index), _matrix(weight)
    if x is None or i is None or w is None or not _i32s(index) or not _f32(weight) or i[:2] != w[:2] or i[0] != x[0]:
        return capi.INVALID_VALUE
    b = None
    if bias is not None:
        b = _vector(bias)
        if b is None or not _f32(bias) or b[:2] != (x[1], 1):
            return capi.INVALID_VALUE
        b = b[2]
    return capi.load().alphasparse_cuda_route(score, _kind(logits)[0], x[0], x[1], x[3], x[2], b, groups, top_groups, i[1],
                                              1 if renormalize else 0, scale, i[3], i[2], w[3], w[2])


def route_grad(score, logits, index, renormalize, scale, dweight, dlogits):
    """alphasparse_cuda_route_grad: dlogits from the gradient dweight of the weights of index.  Returns the status."""
    x, i, w, d = _matrix(logits), _matrix(index), _matrix(dweight), _matrix(dlogits)
    if x is None or i is None or w is None or d is None or not _i32s(index) or not _f32(dweight) or dlogits.dtype != logits.dtype \
            or d[:2] != x[:2] or i[:2] != w[:2] or i[0] != x[0]:
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_route_grad(score, _kind(logits)[0], x[0], x[1], x[3], x[2], i[1], i[3], i[2], 1 if renormalize else 0,
                                                   scale, w[3], w[2], d[3], d[2])


def expert_plan_buffer_size(tokens, k, experts):
    """(status, bytes of the workspace) of expert_plan; 0 for a few thousand pairs."""
    n = C.c_size_t()
    st = capi.load().alphasparse_cuda_expert_plan_buffer_size(tokens, k, experts, C.byref(n))
    return st, n.value


def expert_plan(index, offsets, slot, buffer):
    """alphasparse_cuda_expert_plan: offsets (experts + 1) and slot (tokens, k) of index (tokens, k), all int32.  Returns
    the status."""
    i, s, o = _matrix(index), _matrix(slot), _vector(offsets)
    if i is None or s is None or o is None or i[:2] != s[:2] or o[1] != 1 or not _i32s(index) or not _i32s(offsets) or not _i32s(slot):
        return capi.INVALID_VALUE
    at, size = _buffer(buffer)
    if size < 0:
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_expert_plan(i[0], i[1], o[0] - 1, i[3], i[2], o[2], s[3], s[2], at, size)


def expert_dispatch(x, slot, xs):
    """alphasparse_cuda_expert_dispatch: xs[slot[t, j]] = x[t].  Returns the status."""
    a, s, o = _matrix(x), _matrix(slot), _matrix(xs)
    if a is None or s is None or o is None or not _i32s(slot) or xs.dtype != x.dtype or s[0] != a[0] or o[1] != a[1]:
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_expert_dispatch(_kind(x)[0], a[0], s[1], a[1], a[3], a[2], s[3], s[2], o[0], o[3], o[2])


def _weights(weight, slot):
    """(leading dimension, address) of the weights of the slots (0, None for None), or None if they do not fit them."""
    if weight is None:
        return 0, None
    w = _matrix(weight)
    return (w[2], w[3]) if w is not None and _f32(weight) and w[:2] == slot[:2] else None


def expert_combine(y, slot, weight, beta, out):
    """alphasparse_cuda_expert_combine: out[t] = sum over j of weight[t, j] * y[slot[t, j]] + beta * out[t]; weight None: ones.
    Returns the status."""
    a, s, o = _matrix(y), _matrix(slot), _matrix(out)
    if a is None or s is None or o is None or not _i32s(slot) or out.dtype != y.dtype or o[0] != s[0] or o[1] != a[1]:
        return capi.INVALID_VALUE
    w = _weights(weight, s)
    if w is None:
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_expert_combine(_kind(y)[0], s[0], s[1], a[1], a[0], a[3], a[2], s[3], s[2], w[1], w[0], beta, o[3], o[2])


def expert_combine_grad(dout, y, slot, weight, dy, dweight):
    """alphasparse_cuda_expert_combine_grad: dy[slot[t, j]] = weight[t, j] * dout[t], dweight[t, j] = <dout[t], y[slot[t, j]]>.
    Returns the status."""
    o, a, s, d, g = _matrix(dout), _matrix(y), _matrix(slot), _matrix(dy), _matrix(dweight)
    if o is None or a is None or s is None or d is None or g is None or not _i32s(slot) or not _f32(dweight) or dout.dtype != y.dtype \
            or dy.dtype != y.dtype or d[:2] != a[:2] or o[:2] != (s[0], a[1]) or g[:2] != s[:2]:
        return capi.INVALID_VALUE
    w = _weights(weight, s)
    if w is None:
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_expert_combine_grad(_kind(y)[0], s[0], s[1], a[1], a[0], o[3], o[2], a[3], a[2], s[3], s[2], w[1], w[0],
                                                            d[3], d[2], g[3], g[2])


def expert_mm(operation, offsets, x, w, y):
    """alphasparse_cuda_expert_mm: y[r] = x[r] * op(w[e]) for the rows r from offsets[e] to offsets[e + 1]; w (experts, out, in).
    Returns the status."""
    o, a, m, b = _vector(offsets), _matrix(x), _matrices(w), _matrix(y)
    if o is None or a is None or m is None or b is None or x.dtype != w.dtype or y.dtype != w.dtype or a[0] != b[0] or not _i32s(offsets) \
            or o[:2] != (m[0] + 1, 1) or (a[1], b[1]) != ((m[2], m[1]) if operation == TRANSPOSE else (m[1], m[2])):
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_expert_mm(operation, _kind(w)[0], m[0], a[0], o[2], m[1], m[2], a[3], a[2], m[5], m[3], m[4], b[3], b[2])


def expert_mm_grad(offsets, dy, x, beta, dw):
    """alphasparse_cuda_expert_mm_grad: dw[e] = dy[rows of e]^T x[rows of e] + beta * dw[e].  Returns the status."""
    o, d, a, m = _vector(offsets), _matrix(dy), _matrix(x), _matrices(dw)
    if o is None or d is None or a is None or m is None or x.dtype != dy.dtype or d[0] != a[0] or m[1:3] != (d[1], a[1]) or not _i32s(offsets) \
            or o[:2] != (m[0] + 1, 1):
        return capi.INVALID_VALUE
    return capi.load().alphasparse_cuda_expert_mm_grad(_kind(x)[0], _kind(dw)[0], m[0], a[0], o[2], m[1], m[2], d[3], d[2], a[3], a[2], beta, m[5],
                                                       m[3], m[4])


def expert_mm_status(clear=False):
    """alphasparse_cuda_expert_mm_status: (status, 1 if a wait of any product on the current device ran out since it was last cleared)."""
    v = C.c_int()
    st = capi.load().alphasparse_cuda_expert_mm_status(C.byref(v), 1 if clear else 0)
    return st, v.value
