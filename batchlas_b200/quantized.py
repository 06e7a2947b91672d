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

import ctypes

import torch

from ._lib import GemmI8Desc, QuantizeDesc, check, load
from .gemm import Transpose, _as3

FTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _ld(t):
    return t.stride(1) if t.shape[1] > 1 else max(t.shape[2], 1, t.stride(1))


def _st(t):
    return t.stride(0) if t.shape[0] > 1 else 0


def _same_device(where, *ts):
    if any(not t.is_cuda for t in ts):
        raise RuntimeError(f"{where} needs CUDA tensors; there is no CPU path")
    if len({t.device for t in ts}) != 1:
        raise RuntimeError(f"{where}: operands are on different devices")


def _stream(stream):
    return torch.cuda.current_stream().cuda_stream if stream is None else stream


def _scales(where, s, batch, size):
    """(batch, size) view of a float scale vector per item, or of one vector for the whole batch."""
    if s.dtype != torch.float32:
        raise TypeError(f"{where}: scales must be float32")
    if s.dim() == 1:
        s = s.unsqueeze(0)
    if s.dim() != 2 or s.shape[0] not in (1, batch) or s.shape[1] != size:
        raise RuntimeError(f"{where}: incompatible scale dimensions")
    if size > 1 and s.stride(1) != 1:
        raise ValueError(f"{where}: scales must be contiguous along the columns")
    return s


def quantize_i8(X, Q=None, scale=None, stream=None):
    """Quantises every column of X: ``scale = max|x| / 127``, ``Q = round(x / scale)``, halves to even.  Q (int8, the
    shape of X) and scale (float32, one per column) are made when they are not given; returns both.  Asynchronous."""
    _same_device("batchlas_b200.quantize_i8", *(t for t in (X, Q, scale) if t is not None))
    if X.dtype not in FTYPE_CODES:
        raise TypeError("quantize_i8: X must be float32, float16 or bfloat16")
    if Q is None:
        Q = torch.empty(X.shape, dtype=torch.int8, device=X.device)
    if scale is None:
        scale = torch.empty(X.shape[:-1], dtype=torch.float32, device=X.device)
    if Q.dtype != torch.int8:
        raise TypeError("quantize_i8: Q must be int8")
    X3, Q3 = _as3(X), _as3(Q)
    if X3.shape != Q3.shape:
        raise RuntimeError("QUANTIZE_I8: incompatible matrix dimensions")
    batch, cols, k = X3.shape
    s = _scales("QUANTIZE_I8", scale, batch, cols)
    if s.shape[0] != batch:
        raise RuntimeError("QUANTIZE_I8: incompatible scale dimensions")
    d = QuantizeDesc()
    d.x, d.q, d.scale = X3.data_ptr(), Q3.data_ptr(), s.data_ptr()
    d.k, d.cols, d.batch = k, cols, batch
    d.ldx, d.stride_x, d.ldq, d.stride_q, d.stride_scale = _ld(X3), _st(X3), _ld(Q3), _st(Q3), _st(s)
    d.ftype = FTYPE_CODES[X.dtype]
    with torch.cuda.device(X.device):
        check(load().blb200_quantize_i8(d, _stream(stream)))
    return Q, scale


def gemm_i8(A, B, C, scale_a=None, scale_b=None, alpha=1.0, beta=0.0, transA: Transpose = Transpose.Trans,
            transB: Transpose = Transpose.NoTrans, stream=None):
    """C <- alpha * diag(scale_a) * A^T * B * diag(scale_b) + beta * C for every batch item; returns C.  Asynchronous.

    A (k x m) and B (k x n) are int8 with k fastest, so the op pair is always (Trans, NoTrans); C (m x n) is float32,
    float16 or bfloat16.  scale_a has one float per row of C (channel), scale_b one per column (token); one vector may
    serve the whole batch, None stands for ones.  A or B of batch 1 likewise serve every item of C."""
    _same_device("batchlas_b200.gemm_i8", *(t for t in (A, B, C, scale_a, scale_b) if t is not None))
    if A.dtype != torch.int8 or B.dtype != torch.int8:
        raise TypeError("gemm_i8: A and B must be int8")
    if C.dtype not in FTYPE_CODES:
        raise TypeError("gemm_i8: C must be float32, float16 or bfloat16")
    if Transpose(transA) == Transpose.NoTrans or Transpose(transB) != Transpose.NoTrans:
        raise ValueError("gemm_i8: only the op pair (Trans, NoTrans) exists: both operands are stored with k fastest")
    if isinstance(alpha, complex) or isinstance(beta, complex):
        raise TypeError("gemm_i8: alpha and beta are real")
    A, B, C3 = _as3(A), _as3(B), _as3(C)
    batch, n, m = C3.shape
    k = A.shape[2]
    if A.shape[0] not in (1, batch) or B.shape[0] not in (1, batch) or B.shape[2] != k or A.shape[1] != m or B.shape[1] != n:
        raise RuntimeError("GEMM_I8: incompatible matrix dimensions")
    d = GemmI8Desc()
    d.a, d.b, d.c = A.data_ptr(), B.data_ptr(), C3.data_ptr()
    if scale_a is not None:
        s = _scales("GEMM_I8", scale_a, batch, m)
        d.scale_a, d.stride_scale_a = s.data_ptr(), _st(s)
    if scale_b is not None:
        s = _scales("GEMM_I8", scale_b, batch, n)
        d.scale_b, d.stride_scale_b = s.data_ptr(), _st(s)
    d.m, d.n, d.k, d.batch = m, n, k, batch
    d.lda, d.ldb, d.ldc = _ld(A), _ld(B), _ld(C3)
    d.stride_a, d.stride_b, d.stride_c = _st(A), _st(B), _st(C3)
    d.alpha, d.beta = float(alpha), float(beta)
    d.ftype_c = FTYPE_CODES[C.dtype]
    with torch.cuda.device(C.device):
        check(load().blb200_gemm_i8(d, _stream(stream)))
    return C
