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


# |a s + b s^3 + c s^5| over 0 <= s <= 1 has its maximum inside: 0.3849 a for b = -a, 0.535 a for c = -a.  With one of the coefficients
# next to zero it still has.
@pytest.mark.parametrize("tiny", [0.0, 1e-20, -1e-20, 1e-17, -1e-17, 1e-13, -1e-13, 1e-300])
def test_bound_with_a_coefficient_next_to_zero(lib, tiny):
    status = lambda *q: lib.blb200_newton_schulz(desc(q), None, 0, None)  # noqa: E731
    assert status(200.0, -200.0, tiny) == _lib.E_TOO_LARGE        # 76.98
    assert status(150.0, -150.0, tiny) == _lib.E_NULL             # 57.7, accepted (and then no workspace)
    assert status(150.0, tiny, -150.0) == _lib.E_TOO_LARGE        # 80.2
    assert status(100.0, tiny, -100.0) == _lib.E_NULL             # 53.5
    assert status(tiny, 200.0, -200.0) == _lib.E_NULL             # 200 (s^3 - s^5): 37.2
    assert status(tiny, 400.0, -400.0) == _lib.E_TOO_LARGE        # 74.4


@pytest.mark.parametrize("small", [0.5, 0.1, 0.02])
def test_bound_of_small_matrices_with_large_coefficients(lib, small):
    """s of a second step goes up to 1.01 small; in u = s / small its polynomial is 200 (u - u^3), then 150 (u - u^3)."""
    second = lambda a: lib.blb200_newton_schulz(desc((small, 0.0, 0.0, a / small, -a / small / small / small, 1e-20)), None, 0, None)  # noqa: E731
    assert second(200.0) == _lib.E_TOO_LARGE
    assert second(150.0) == _lib.E_NULL


@pytest.mark.parametrize("coefficients", [QUINTIC, list(QUINTIC), (3, -4, 2)], ids=str)
@pytest.mark.parametrize("form", ["as is", "float32 array", "one per step"])
def test_forms_of_the_coefficients(lib, coefficients, form):
    import numpy as np

    from batchlas_b200.orthogonal import _desc
    given = {"as is": coefficients, "float32 array": np.array(coefficients, np.float32), "one per step": [coefficients] * 4}[form]
    x = torch.zeros(2, 3, 4)
    d = _desc(x, x, 4, given, 1e-7, False)
    sets = 4 if form == "one per step" else 1
    want = [float(np.float32(v)) if form == "float32 array" else float(v) for v in coefficients] * sets
    assert d.coefficient_sets == sets and d.coefficients[:3 * sets] == want
