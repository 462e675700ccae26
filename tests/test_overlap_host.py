"""CPU tests of the check for memory that two tensors of a clipping call share:
the arithmetic against sets of addresses, and what the entry points refuse and
take by it."""

import ctypes
import itertools
import os
import random
import subprocess

import pytest
import torch

import ilqr_native as nat
from test_gradclip_host import A, _elements

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "ilqr_overlap.h"
extern "C" int meet(uint64_t a, int64_t la, const int64_t* da, int na, uint64_t b, int64_t lb, const int64_t* db, int nb) {
  static_assert(sizeof(ilqr::Every) == 16, "count and stride");
  return ilqr::Meeting::of({(uintptr_t)a, la, reinterpret_cast<const ilqr::Every*>(da), na},
                           {(uintptr_t)b, lb, reinterpret_cast<const ilqr::Every*>(db), nb});
}
"""


@pytest.fixture(scope="module")
def meet(tmp_path_factory):
    at = tmp_path_factory.mktemp("overlap")
    (at / "meet.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", str(at / "meet.cpp"), "-I",
                    os.path.join(ROOT, "ca-ac-mpc_b200", "csrc"), "-o", str(at / "meet.so")], check=True)
    f = ctypes.CDLL(str(at / "meet.so")).meet

    def call(a, b):
        given = []
        for base, length, dims in (a, b):
            flat = [v for d in dims for v in d] or [0]
            given += [ctypes.c_uint64(base), ctypes.c_int64(length), (ctypes.c_int64 * len(flat))(*flat), len(dims)]
        return bool(f(*given))
    return call


def _bytes(s):
    base, length, dims = s
    return {base + sum(i * d[1] for i, d in zip(at, dims)) + k
            for at in itertools.product(*(range(d[0]) for d in dims)) for k in range(length)}


def test_small_sets_against_their_addresses(meet):
    """Every answer is right: two or three strides, equal or not, zero ones,
    empty sets, runs that touch and runs that meet in one byte."""
    rng = random.Random(5)
    seen = [0, 0]
    for turn in range(20_000):
        sets = []
        strides = [rng.choice([0, 1, 2, 3, 4, 6, 7, 10, 12, 20, 21, 40, 60]) for _ in range(3)]
        for _ in range(2):
            own = strides if rng.random() < 0.7 else [rng.randint(0, 50) for _ in range(3)]
            dims = [(rng.choice([0] * (turn % 50 == 0) + [1, 2, 3, 5]), s) for s in own[:rng.randint(0, 3)]]
            sets.append((1000 + rng.randint(0, 120), rng.randint(1, 9), dims))
        want = bool(_bytes(sets[0]) & _bytes(sets[1]))
        assert meet(*sets) == want and meet(*reversed(sets)) == want, sets
        seen[want] += 1
    assert min(seen) > 1000


def test_long_sets(meet):
    """Columns of arrays with far more values than could be gone through."""
    for B, T in ((2**31 - 1, 500), (70_000, 50), (3, 1)):
        for row, seg in ((840, 840 * B), (840 * T, 840)):
            C = (1 << 20, 784, [(B, row), (T, seg)])
            c = ((1 << 20) + 784, 56, [(B, row), (T, seg)])
            assert not meet(C, c) and not meet(c, C)
            assert meet(C, ((1 << 20) + 783, 57, c[2])) and meet(C, (c[0] + 840 + 55, 2, []))
            assert not meet(C, (c[0], 56, [(T, seg)])) and meet(C, (c[0] + 1, 56, [(T, seg)]))
            last = (1 << 20) + (B - 1) * row + (T - 1) * seg
            assert meet(C, (last, 784, [])) and not meet(C, (last + 784, 56, []))


# ---- what the entry point takes and refuses ------------------------------------
# Layouts of C and c as columns 0..195 and 196..209 of one [T, B, 210] or
# [B, T, 210] array of float32.

def _packed(T, B, time_major, at=196, width=14):
    row, seg = (210, 210 * B) if time_major else (210 * T, 210)
    lay = [(T, w, seg, row, seg, row) for w in (196, width)]
    return dict(grads=(A, A + 4 * at), out=(A, A + 4 * at), dtypes=(0, 0), layout=lay, B=B)


@pytest.mark.parametrize("T,B", [(5, 16), (1, 16), (5, 1), (50, 3), (1, 1)])
@pytest.mark.parametrize("time_major", [False, True])
def test_overlapping_columns_are_refused(T, B, time_major):
    assert _elements(**_packed(T, B, time_major, at=195)) == 7
    assert _elements(**_packed(T, B, time_major, at=197 - 2, width=1)) == 7
    if T * B > 1:
        assert _elements(**_packed(T, B, time_major, at=196, width=15)) == 7   # the next one's first value
    row, seg = (210, 210 * B) if time_major else (210 * T, 210)
    # in place within one tensor, one value on
    assert _elements(grads=(A,), out=(A + 4,), layout=((T, 100, seg, row, seg, row),), B=B) == 7


# The calls that pass every check end in a launch, which fails without a GPU (status 4).
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses stand for memory that is not there")


@no_gpu
@pytest.mark.parametrize("T,B", [(5, 16), (1, 16), (5, 1), (50, 3), (1, 1)])
@pytest.mark.parametrize("time_major", [False, True])
def test_columns_of_one_array_are_taken(T, B, time_major):
    assert _elements(**_packed(T, B, time_major)) == 4
    row, seg = (210, 210 * B) if time_major else (210 * T, 210)
    # the other half of each step of the same array
    assert _elements(grads=(A,), out=(A + 420,), layout=((T, 105, seg, row, seg, row),), B=B) == 4
    # x0 before the steps of each element of one [B, 10 + 210 T] array
    R = 10 + 210 * T
    lay = ((1, 10, 0, R, 0, R), (T, 196, 210, R, 210, R), (T, 14, 210, R, 210, R))
    at = (A, A + 40, A + 40 + 784)
    assert _elements(grads=at, out=at, dtypes=(0, 0, 0), layout=lay, B=B) == 4


# ---- what a call writes or reads beside the gradients ----------------------------

def _raw_clip(total=None, norm=None, grads=(A, 2 * A), out=(3 * A, 4 * A), numel=(50, 70)):
    arr = [(ctypes.c_uint64 * 2)(*grads), (ctypes.c_uint64 * 2)(*out), (ctypes.c_int64 * 2)(*numel), (ctypes.c_int32 * 2)(0, 0)]
    return nat.lib().ilqr_b200_grad_clip(*arr, 2, 0, 1.0, 1e-6, total, norm, 8 * A, 1 << 20, None)


def _raw_elements(norms, in_place=True, B=16, T=5):
    arr = [(ctypes.c_uint64 * 1)(A), (ctypes.c_uint64 * 1)(A if in_place else 4 * A), (ctypes.c_int32 * 1)(0),
           (ctypes.c_int64 * 6)(T, 14, 210, 210 * T, 210, 210 * T)]
    return nat.lib().ilqr_b200_grad_clip_elements(*arr, 1, B, 1.0, 1e-6, 0, norms, None)


def test_total_and_norm_that_share_memory_are_refused():
    assert _raw_clip(total=3 * A) == 7 and _raw_clip(total=4 * A + 272) == 7       # within an output, at its end
    assert _raw_clip(total=A, out=(A, 4 * A)) == 7                                 # and in place
    assert _raw_clip(norm=3 * A + 196) == 7 and _raw_clip(norm=A + 196) == 7       # an output, an input
    assert _raw_clip(total=6 * A, norm=6 * A) == 7 and _raw_clip(total=6 * A, norm=6 * A + 4) == 7
    for in_place in (True, False):
        assert _raw_elements(A, in_place) == 7                                     # over the first element
        assert _raw_elements(A + 4 * (210 * 79 + 13), in_place) == 7               # from the last value on
        assert _raw_elements(A + 780, in_place) == 7                               # from a gap into the next run
    assert _raw_elements(4 * A, False) == 7


@no_gpu
def test_total_and_norm_beside_the_tensors_are_taken():
    assert _raw_clip(total=3 * A + 200, norm=3 * A + 208) == 4                     # behind an output
    assert _raw_clip(total=A) == 4                                                 # an input that is only read
    for in_place in (True, False):
        assert _raw_elements(A + 4 * (210 * 79 + 14), in_place) == 4
        assert _raw_elements(A + 776, in_place) == 4                               # within a gap


def test_long_sets_with_strides_of_their_own(meet):
    """Every second row of a column beside all rows of another, and the like:
    found for any number of rows."""
    for N in (100, 20_000, 5_000_000, 2**40):
        a = (1 << 20, 128, [(N, 256)])
        for step in (2, 3, 17):
            b = ((1 << 20) + 128, 128, [(N // step, 256 * step)])
            assert not meet(a, b) and not meet(b, a)
            assert meet(a, (b[0] + 1, 128, b[2])) and meet((b[0] - 1, 128, b[2]), a)
        # blocks of rows, columns of each
        c = (1 << 20, 64, [(N, 1024), (5, 192)])
        d = ((1 << 20) + 64, 128, [(N // 3, 3072), (4, 192)])
        assert not meet(c, d) and not meet(d, c) and meet(c, (d[0], 129, d[2]))
    # strides without a common measure: the first two runs that meet are far on
    for s, t, n in ((1009, 1013, 1013), (10_007, 10_009, 10_009)):
        a, b = (0, 1, [(n, s)]), (5, 1, [(n, t)])
        # i s = 5 + j t with 0 <= i, j < n
        j = next((j for j in range(n) if (5 + j * t) % s == 0 and (5 + j * t) // s < n), None)
        assert j is not None and meet(a, b)
        assert not meet((0, 1, [((5 + j * t) // s, s)]), (5, 1, [(j + 1, t)]))


def test_larger_sets_against_their_addresses(meet):
    rng = random.Random(11)
    seen = [0, 0]
    for _ in range(1500):
        sets = []
        unit = rng.choice([1, 1, 2, 7, 16])
        for _ in range(2):
            dims = [(rng.randint(1, 40), rng.randint(1, 60) * unit) for _ in range(rng.randint(1, 2))]
            sets.append((5000 + rng.randint(0, 700), rng.randint(1, 3), dims))
        want = bool(_bytes(sets[0]) & _bytes(sets[1]))
        assert meet(*sets) == want and meet(*reversed(sets)) == want, sets
        seen[want] += 1
    assert min(seen) > 100
