"""Orthogonalisation of update matrices by Newton-Schulz products, over torch tensors (device memory and streams
only).  Matrices use the convention of :mod:`batchlas_b200.gemm`; since the iteration commutes with transposition, a
row-major matrix can be passed as it is."""
from __future__ import annotations

import ctypes
import numbers

import torch

from ._lib import NewtonSchulzDesc, load
from .quantized import FTYPE_CODES, _empty, _launch, _matrix, _same_device

QUINTIC = (3.4445, -4.7750, 2.0315)


def _desc(X, Y, steps, coefficients, eps, half_intermediates):
    if X.dtype not in FTYPE_CODES or Y.dtype != X.dtype:
        raise TypeError("newton_schulz: X and Y must share one of float32/float16/bfloat16")
    batch, cols, rows, ldx, stride_x = _matrix(X)
    y_batch, y_cols, y_rows, ldy, stride_y = _matrix(Y)
    if (batch, cols, rows) != (y_batch, y_cols, y_rows):
        raise RuntimeError("NEWTON_SCHULZ: incompatible matrix dimensions")
    sets = list(coefficients)
    if len(sets) == 3 and isinstance(sets[0], numbers.Real):
        sets = [sets]
    if len(sets) not in (1, steps) or any(len(s) != 3 for s in sets):
        raise ValueError("newton_schulz: coefficients are one triple (a, b, c), or one for each step")
    flat = [float(v) for s in sets for v in s]
    return NewtonSchulzDesc(X.data_ptr(), Y.data_ptr(), rows, cols, batch, ldx, ldy, stride_x, stride_y, FTYPE_CODES[X.dtype], int(steps),
                            len(sets), int(bool(half_intermediates)), (ctypes.c_double * len(flat))(*flat), float(eps))


def newton_schulz_workspace_bytes(X, half_intermediates=False) -> int:
    """Scratch bytes that :func:`newton_schulz` needs for a tensor of X's shape and type."""
    return int(load().blb200_newton_schulz_workspace_bytes(_desc(X, X, 1, QUINTIC, 0.0, half_intermediates)))


def newton_schulz(X, Y=None, steps=5, coefficients=QUINTIC, eps=1e-7, *, half_intermediates=False, workspace=None, stream=None):
    """Y <- X / (||X||_F + eps), then `steps` times Y <- (a I + b Y Y^T + c (Y Y^T)^2) Y, for every batch item; returns Y.

    Y is made when it is not given and may be X.  Every intermediate matrix is a pair of float16 matrices times a power of
    two, which keeps float accuracy throughout; Y is rounded once.  ``half_intermediates`` (bfloat16 only) keeps one float16
    matrix of each: large calls take 0.3 of the time, and the error grows from 1.65e-3 of the result (rounding Y) to 1.9 to
    2.2e-3.  The scratch comes from torch's caching allocator unless `workspace` (a CUDA uint8 tensor, 256-byte aligned, of at
    least :func:`newton_schulz_workspace_bytes` bytes) is given.  Asynchronous."""
    index = X.get_device()
    _same_device("batchlas_b200.newton_schulz", index, *(() if Y is None else (Y,)))
    if Y is None:
        Y = _empty(X.shape, X.dtype, X.device, stream)
    d = _desc(X, Y, steps, coefficients, eps, half_intermediates)
    need = int(load().blb200_newton_schulz_workspace_bytes(d))
    if workspace is None:
        workspace = _empty((max(need, 256),), torch.uint8, X.device, stream, returned=False)
    elif workspace.get_device() != index or workspace.dtype is not torch.uint8 or workspace.numel() < need \
            or not workspace.is_contiguous() or workspace.data_ptr() % 256:
        raise ValueError(f"workspace must be a contiguous uint8 tensor of at least {need} bytes on {X.device}, 256-byte aligned")
    _launch(index, stream, lambda desc, on: load().blb200_newton_schulz(desc, workspace.data_ptr(), workspace.numel(), on), d)
    return Y
