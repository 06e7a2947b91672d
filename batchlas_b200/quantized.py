"""8-bit integer products with a scale for each token and channel, over torch tensors (device memory and
streams only): :func:`quantize_i8` makes the operands, :func:`gemm_i8` multiplies them.

Tensors use the convention of :mod:`batchlas_b200.gemm`: a column-major ``rows x cols`` matrix is a tensor
of shape ``(batch, cols, rows)`` (or ``(cols, rows)``) with unit stride along ``rows``.  For a linear layer
that is the usual storage: weights ``(out, in)`` are a ``k x m`` matrix with one column per output channel,
activations ``(tokens, in)`` a ``k x n`` matrix with one column per token, and the product ``C`` comes out as
``(tokens, out)``::

    Wq, sw = quantize_i8(W)                      # once
    Xq, sx = quantize_i8(X)                      # every call
    gemm_i8(Wq, Xq, Y, sw, sx)                   # Y = X W^T up to the quantisation
"""
from __future__ import annotations

import torch

from ._lib import GemmI8Desc, QuantizeDesc, check, load
from .gemm import Transpose

FTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


# These calls are short, so their host side is kept short too: plain integers instead of views, no device guard or stream
# object where the current ones are the right ones (builds of torch without the short way to the current stream, CPU builds
# among them, take the public one).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _same_device(where, index, *ts):
    """Raises unless every tensor is on CUDA device `index`, the first operand's."""
    if index < 0 or any(t.get_device() < 0 for t in ts):
        raise RuntimeError(f"{where} needs CUDA tensors; there is no CPU path")
    if any(t.get_device() != index for t in ts):
        raise RuntimeError(f"{where}: operands are on different devices")


def _launch(index, stream, fn, desc):
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return _launch(index, stream, fn, desc)
    status = fn(desc, _raw_stream(index) if stream is None else stream)
    if status:
        check(status)


def _empty(shape, dtype, device, stream, returned=True):
    """Memory that a call on `stream` (None: the current one) is the first to write.  It comes from that stream's pool: a block of
    the current stream's may still be read by what is queued there.  The caller goes on to use what is `returned` on the
    current stream, so the allocator waits for both streams before it hands the block out again."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    current = torch.cuda.current_stream(device)
    if current.cuda_stream == stream:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device)):
        t = torch.empty(shape, dtype=dtype, device=device)
    if returned:
        t.record_stream(current)
    return t


def _matrix(t):
    """(batch, cols, rows, ld, stride) of a column-major tensor."""
    st = t.stride()
    if len(st) == 2:
        cols, rows = t.shape
        ld, inner = st
        if inner == 1 and cols > 1:
            return 1, cols, rows, ld, 0
        batch, stride = 1, 0
    elif len(st) == 3:
        batch, cols, rows = t.shape
        stride, ld, inner = st
        if batch <= 1:
            stride = 0
    else:
        raise ValueError("expected a (batch, cols, rows) or (cols, rows) tensor")
    if rows > 1 and inner != 1:
        raise ValueError("rows must be contiguous (column-major storage)")
    return batch, cols, rows, ld if cols > 1 else max(rows, 1, ld), stride


def _scales(where, s, batch, size, shared=True):
    """Batch stride of a float scale vector per item, or of one vector for the whole batch."""
    if s.dtype is not torch.float32:
        raise TypeError(f"{where}: scales must be float32")
    st = s.stride()
    if len(st) == 1:
        items, given, inner = 1, s.shape[0], st[0]
    elif len(st) == 2:
        items, given = s.shape
        inner = st[1]
    else:
        given = -1
    if given != size or (items != batch and not (shared and items == 1)):
        raise RuntimeError(f"{where}: incompatible scale dimensions")
    if inner != 1 and size > 1:
        raise ValueError(f"{where}: scales must be contiguous along the columns")
    return st[0] if items > 1 else 0


def quantize_i8(X, Q=None, scale=None, stream=None):
    """Quantises every column of X: ``scale = max|x| * float32(1 / 127)``, ``Q = round(x / scale)``, halves to
    even.  Q (int8, the shape of X) and scale (float32, one per column) are made when they are not given; returns both.
    Asynchronous."""
    index = X.get_device()
    if index < 0:
        _same_device("batchlas_b200.quantize_i8", index)
    if Q is None:
        Q = _empty(X.shape, torch.int8, X.device, stream)
    if scale is None:
        scale = _empty(X.shape[:-1], torch.float32, X.device, stream)
    if Q.get_device() != index or scale.get_device() != index:
        _same_device("batchlas_b200.quantize_i8", index, Q, scale)
    ftype = FTYPE_CODES.get(X.dtype)
    if ftype is None:
        raise TypeError("quantize_i8: X must be float32, float16 or bfloat16")
    if Q.dtype is not torch.int8:
        raise TypeError("quantize_i8: Q must be int8")
    batch, cols, k, ldx, stride_x = _matrix(X)
    q_batch, q_cols, q_k, ldq, stride_q = _matrix(Q)
    if (batch, cols, k) != (q_batch, q_cols, q_k):
        raise RuntimeError("QUANTIZE_I8: incompatible matrix dimensions")
    stride_s = _scales("QUANTIZE_I8", scale, batch, cols, shared=False)
    d = QuantizeDesc(X.data_ptr(), Q.data_ptr(), scale.data_ptr(), k, cols, batch, ldx, stride_x, ldq, stride_q, stride_s, ftype)
    _launch(index, stream, load().blb200_quantize_i8, d)
    return Q, scale


def gemm_i8(A, B, C, scale_a=None, scale_b=None, alpha=1.0, beta=0.0, transA: Transpose = Transpose.Trans,
            transB: Transpose = Transpose.NoTrans, stream=None):
    """C <- alpha * diag(scale_a) * A^T * B * diag(scale_b) + beta * C for every batch item; returns C.  Asynchronous.

    A (k x m) and B (k x n) are int8 with k fastest, so the op pair is always (Trans, NoTrans); C (m x n) is float32,
    float16 or bfloat16.  scale_a has one float per row of C (channel), scale_b one per column (token); one vector may
    serve the whole batch, None stands for ones.  A or B of batch 1 likewise serve every item of C."""
    index = C.get_device()
    _same_device("batchlas_b200.gemm_i8", index, A, B, *(t for t in (scale_a, scale_b) if t is not None))
    if A.dtype is not torch.int8 or B.dtype is not torch.int8:
        raise TypeError("gemm_i8: A and B must be int8")
    ftype = FTYPE_CODES.get(C.dtype)
    if ftype is None:
        raise TypeError("gemm_i8: C must be float32, float16 or bfloat16")
    if transA == Transpose.NoTrans or transB != Transpose.NoTrans:
        raise ValueError("gemm_i8: only the op pair (Trans, NoTrans) exists: both operands are stored with k fastest")
    if isinstance(alpha, complex) or isinstance(beta, complex):
        raise TypeError("gemm_i8: alpha and beta are real")
    batch, n, m, ldc, stride_c = _matrix(C)
    a_batch, a_cols, k, lda, stride_a = _matrix(A)
    b_batch, b_cols, b_k, ldb, stride_b = _matrix(B)
    if (a_batch != 1 and a_batch != batch) or (b_batch != 1 and b_batch != batch) or b_k != k or a_cols != m or b_cols != n:
        raise RuntimeError("GEMM_I8: incompatible matrix dimensions")
    stride_sa = stride_sb = 0
    ptr_sa = ptr_sb = None
    if scale_a is not None:
        stride_sa, ptr_sa = _scales("GEMM_I8", scale_a, batch, m), scale_a.data_ptr()
    if scale_b is not None:
        stride_sb, ptr_sb = _scales("GEMM_I8", scale_b, batch, n), scale_b.data_ptr()
    d = GemmI8Desc(A.data_ptr(), B.data_ptr(), C.data_ptr(), ptr_sa, ptr_sb, m, n, k, batch, lda, ldb, ldc, stride_a, stride_b,
                   stride_c, stride_sa, stride_sb, float(alpha), float(beta), ftype)
    _launch(index, stream, load().blb200_gemm_i8, d)
    return C
