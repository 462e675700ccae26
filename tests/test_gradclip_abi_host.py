"""CPU tests of what the entry points of the gradient norms and clipping refuse
before anything is launched (a pointer that is not aligned to its type would
fault the GPU)."""

import ctypes

import pytest

import ilqr_native as nat
from test_gradclip_host import A, _norm


def _clip(**kw):
    arr = [(ctypes.c_uint64 * 1)(A), (ctypes.c_uint64 * 1)(2 * A), (ctypes.c_int64 * 1)(5), (ctypes.c_int32 * 1)(0)]
    n = kw.get("n", 1)
    return nat.lib().ilqr_b200_grad_clip(*(arr if n else [None] * 4), n, 0, 1.0, 1e-6, kw.get("total"), kw.get("norm"),
                                         3 * A, 1 << 20, None)


def _elements(layout=(1, 10, 0, 10, 0, 10), norms=None, dtype=0, B=4):
    arr = [(ctypes.c_uint64 * 1)(A), (ctypes.c_uint64 * 1)(2 * A), (ctypes.c_int32 * 1)(dtype), (ctypes.c_int64 * 6)(*layout)]
    return nat.lib().ilqr_b200_grad_clip_elements(*arr, 1, B, 1.0, 1e-6, 0, norms, None)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_norms_are_refused(off):
    for n in (0, 2):  # an empty list's norm is written too
        assert _norm(norm=A + off, n=n) == 2
        assert _norm(norm=None, norms=A + off, n=n) == 2
    for n in (0, 1):
        assert _clip(norm=4 * A + off, n=n) == 2
    assert _elements(norms=4 * A + off) == 2


@pytest.mark.parametrize("off", [1, 2, 4, 6])
def test_misaligned_totals_are_refused(off):
    for n in (0, 2):
        assert _norm(total=A + off, n=n) == 2
        assert _norm(norm=None, total=A + off, n=n) == 2
    for n in (0, 1):
        assert _clip(total=4 * A + off, n=n) == 2


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("k", [2, 3, 4, 5])
def test_the_lowest_stride_is_refused(k, dtype):
    """-2^63, whose magnitude is no 64-bit integer; its bytes wrap to stride 0."""
    for lowest in (-2**63, -2**63 + 1, 2**63 - 1, -2**62):
        layout = [2, 10, 10, 20, 10, 20]
        layout[k] = lowest
        assert _elements(layout, dtype=dtype) == 1
        assert _elements([1, *layout[1:]], dtype=dtype, B=1) == 1
