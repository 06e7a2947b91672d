"""CPU-side checks of the 8-bit product, its quantiser and the Newton-Schulz call: descriptor layouts, refusals and
empty calls of the C ABI, argument checks of the Python layer.  Nothing here reaches a device."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from batchlas_b200 import _lib  # noqa: E402

QUINTIC = (3.4445, -4.7750, 2.0315)


def fill(desc, **kw):
    for k, v in kw.items():
        setattr(desc, k, v)
    return desc


def quantize_desc(**kw):
    base = dict(x=0x1000, q=0x2000, scale=0x3000, k=8, cols=4, batch=2, ldx=8, stride_x=32, ldq=8, stride_q=32,
                stride_scale=4, ftype=0)
    return fill(_lib.QuantizeDesc(), **{**base, **kw})


def gemm_desc(**kw):
    base = dict(a=0x1000, b=0x2000, c=0x3000, scale_a=0x4000, scale_b=0x5000, m=4, n=4, k=8, batch=1, lda=8, ldb=8, ldc=4,
                stride_a=0, stride_b=0, stride_c=0, stride_scale_a=0, stride_scale_b=0, alpha=1.0, beta=0.0, ftype_c=0)
    return fill(_lib.GemmI8Desc(), **{**base, **kw})


def ns_desc(coefficients=QUINTIC, sets=None, **kw):
    flat = (ctypes.c_double * len(coefficients))(*coefficients)
    base = dict(x=0x1000, y=0x2000, rows=4, cols=4, batch=1, ldx=4, ldy=4, stride_x=0, stride_y=0, ftype=0, steps=5,
                coefficient_sets=len(coefficients) // 3 if sets is None else sets, eps=1e-7)
    d = fill(_lib.NewtonSchulzDesc(), **{**base, **kw})
    d.coefficients = flat
    return d


def test_descriptor_layouts_match_the_header():
    assert ctypes.sizeof(_lib.QuantizeDesc) == 3 * 8 + 3 * 4 + 4 + 5 * 8 + 4 + 4
    assert ctypes.sizeof(_lib.GemmI8Desc) == 5 * 8 + 4 * 4 + 8 * 8 + 2 * 8 + 4 + 4
    assert ctypes.sizeof(_lib.NewtonSchulzDesc) == 2 * 8 + 3 * 4 + 4 + 4 * 8 + 3 * 4 + 4 + 8 + 8


@pytest.mark.parametrize("kw,status", [
    (dict(ftype=3), _lib.E_DTYPE), (dict(ftype=-1), _lib.E_DTYPE), (dict(k=-1), _lib.E_SHAPE), (dict(cols=-1), _lib.E_SHAPE),
    (dict(batch=-1), _lib.E_SHAPE), (dict(ldx=7), _lib.E_SHAPE), (dict(ldq=7), _lib.E_SHAPE), (dict(stride_x=-1), _lib.E_SHAPE),
    (dict(stride_q=0), _lib.E_SHAPE), (dict(stride_q=31), _lib.E_SHAPE), (dict(stride_scale=3), _lib.E_SHAPE),
    (dict(x=0), _lib.E_NULL), (dict(q=0), _lib.E_NULL), (dict(scale=0), _lib.E_NULL),
    (dict(cols=0, x=0, q=0, scale=0), 0), (dict(batch=0), 0),
    (dict(k=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31, stride_x=1 << 34, stride_q=1 << 34), _lib.E_TOO_LARGE)])
def test_quantize_refusals(lib, kw, status):
    assert lib.blb200_quantize_i8(quantize_desc(**kw), None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(ftype_c=3), _lib.E_DTYPE), (dict(m=-1), _lib.E_SHAPE), (dict(n=-1), _lib.E_SHAPE), (dict(k=-1), _lib.E_SHAPE),
    (dict(k=131072, lda=131072, ldb=131072), _lib.E_TOO_LARGE), (dict(lda=7), _lib.E_SHAPE), (dict(ldb=7), _lib.E_SHAPE),
    (dict(ldc=3), _lib.E_SHAPE), (dict(batch=2), _lib.E_SHAPE), (dict(batch=2, stride_c=15), _lib.E_SHAPE),
    (dict(batch=2, stride_c=4, ldc=7), _lib.E_SHAPE), (dict(stride_scale_a=-1), _lib.E_SHAPE),
    (dict(a=0), _lib.E_NULL), (dict(b=0), _lib.E_NULL), (dict(c=0), _lib.E_NULL),
    (dict(m=0, a=0, b=0, c=0), 0), (dict(n=0), 0), (dict(batch=0), 0),
    (dict(m=(1 << 30) + 1, ldc=1 << 31), _lib.E_TOO_LARGE), (dict(n=(1 << 30) + 1), _lib.E_TOO_LARGE)])
def test_gemm_i8_refusals(lib, kw, status):
    assert lib.blb200_gemm_i8(gemm_desc(**kw), None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(ftype=7), _lib.E_DTYPE), (dict(rows=-1), _lib.E_SHAPE), (dict(ldx=3), _lib.E_SHAPE), (dict(ldy=3), _lib.E_SHAPE),
    (dict(batch=2), _lib.E_SHAPE), (dict(batch=2, stride_y=15), _lib.E_SHAPE), (dict(batch=70000, stride_y=16), _lib.E_TOO_LARGE),
    (dict(steps=0), _lib.E_UNSUPPORTED), (dict(steps=65), _lib.E_UNSUPPORTED), (dict(eps=-1.0), _lib.E_UNSUPPORTED),
    (dict(eps=float("nan")), _lib.E_UNSUPPORTED), (dict(sets=2), _lib.E_UNSUPPORTED),
    (dict(coefficients=(float("inf"), 0.0, 0.0)), _lib.E_UNSUPPORTED), (dict(coefficients=(65.0, 0.0, 0.0)), _lib.E_TOO_LARGE),
    (dict(coefficients=(3.0, 0.0, 0.0)), _lib.E_TOO_LARGE),          # 3^5 > 64
    (dict(coefficients=(1.0, 20000.0, -20000.0)), _lib.E_TOO_LARGE),
    (dict(x=0), _lib.E_NULL), (dict(y=0), _lib.E_NULL), (dict(rows=0), 0), (dict(cols=0), 0), (dict(batch=0), 0),
    (dict(rows=(1 << 30) + 1, ldx=1 << 31, ldy=1 << 31), _lib.E_TOO_LARGE)])
def test_newton_schulz_refusals(lib, kw, status):
    assert lib.blb200_newton_schulz(ns_desc(**kw), None, 0, None) == status


def test_newton_schulz_workspace_is_checked_before_any_launch(lib):
    d = ns_desc()
    need = lib.blb200_newton_schulz_workspace_bytes(d)
    assert need > 0
    assert lib.blb200_newton_schulz(d, None, need, None) == _lib.E_NULL
    assert lib.blb200_newton_schulz(d, 0x10000, need - 1, None) == _lib.E_SHAPE
    assert lib.blb200_newton_schulz(d, 0x10010, need, None) == _lib.E_SHAPE
    assert lib.blb200_newton_schulz_workspace_bytes(ns_desc(rows=0)) == 0
    big = dict(rows=1024, cols=1024, ldx=1024, ldy=1024, batch=3, stride_x=1 << 20, stride_y=1 << 20)
    assert lib.blb200_newton_schulz_workspace_bytes(ns_desc(steps=1, **big)) == \
        lib.blb200_newton_schulz_workspace_bytes(ns_desc(steps=64, **big))   # one scratch serves every number of steps
    d.coefficients = None
    assert lib.blb200_newton_schulz(d, 0x10000, need, None) == _lib.E_NULL


def test_python_layer_refuses_host_tensors_and_wrong_arguments(lib):
    import batchlas_b200 as bl
    x = torch.zeros(2, 3, 4)
    q = x.to(torch.int8)
    with pytest.raises(RuntimeError, match="CUDA"):
        bl.quantize_i8(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        bl.gemm_i8(q, q, torch.zeros(2, 3, 3))
    with pytest.raises(RuntimeError, match="CUDA"):
        bl.newton_schulz(x)
    with pytest.raises(TypeError):
        bl.newton_schulz_workspace_bytes(x.double())
    assert bl.newton_schulz_workspace_bytes(x) > 0
