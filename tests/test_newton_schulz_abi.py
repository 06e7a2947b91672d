"""CPU-side checks of newton_schulz's arguments through the C ABI: nothing here reaches a device."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from batchlas_b200 import _lib  # noqa: E402

QUINTIC = (3.4445, -4.7750, 2.0315)


def desc(coefficients=QUINTIC, **kw):
    d = _lib.NewtonSchulzDesc()
    base = dict(x=0x1000, y=0x2000, rows=300, cols=300, batch=1, ldx=300, ldy=300, stride_x=0, stride_y=0, ftype=2, steps=len(coefficients) // 3,
                coefficient_sets=len(coefficients) // 3, eps=1e-7)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    d.coefficients = (ctypes.c_double * len(coefficients))(*coefficients)
    return d


@pytest.mark.parametrize("ftype,flag,status", [(2, 0, _lib.E_NULL), (2, 1, _lib.E_NULL), (2, 2, _lib.E_UNSUPPORTED), (2, -1, _lib.E_UNSUPPORTED),
                                               (0, 1, _lib.E_UNSUPPORTED), (1, 1, _lib.E_UNSUPPORTED), (0, 0, _lib.E_NULL)])
def test_half_intermediates_is_a_flag_for_bfloat16(lib, ftype, flag, status):
    assert lib.blb200_newton_schulz(desc(ftype=ftype, half_intermediates=flag), None, 0, None) == status   # no workspace: E_NULL


def test_half_intermediates_need_half_the_scratch(lib):
    import batchlas_b200 as bl
    x = torch.zeros(3, 1024, 2048, dtype=torch.bfloat16)
    pairs, halves = bl.newton_schulz_workspace_bytes(x), bl.newton_schulz_workspace_bytes(x, half_intermediates=True)
    matrices = 3 * 2 * (2 * 1024 * 2048 + 2 * 1024 * 1024)          # bytes of X twice, S and B in one half each
    assert pairs - halves == matrices
