"""Gradients that lie between one another in one array, clipped in place and
into each other's gaps, against the definition in 64 bits (tolerances as in
test_gpu_gradclip.py)."""

import math

import pytest
import torch

from test_gpu_gradclip import DEV, F32, TYPES, _check_elements, _values

pytestmark = pytest.mark.gpu


def _columns(T, B, n, dtype, time_major, seed):
    """x0, C and c of B elements as columns of one array each step, some
    columns left over; and the array."""
    wide = n * n + n + 3
    lead = (T, B) if time_major else (B, T)
    p = _values((*lead, wide), dtype, seed)
    b = int(time_major)
    p *= torch.linspace(0.1, 2.0, B, device=DEV).to(dtype).view((1, B, 1) if time_major else (B, 1, 1))
    return [p[..., :n * n].unflatten(-1, (n, n)), p[..., n * n:n * n + n]], [b, b], p


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("time_major", [False, True])
@pytest.mark.parametrize("B,T,n", [(1, 1, 14), (16, 5, 14), (33, 20, 14), (7, 3, 17), (5, 1, 14), (2, 300, 14), (1, 900, 17)])
def test_columns_of_one_array_in_place(B, T, n, dtype, time_major):
    grads, dims, p = _columns(T, B, n, dtype, time_major, seed=B + T)
    left = p[..., n * n + n:].clone()
    m = math.sqrt(T * (n * n + n))
    # the order of a sum goes by how its tensors lie, so new outputs may differ in bits
    _check_elements(grads, dims, m)
    _check_elements(grads, dims, m, out=grads)
    assert torch.equal(p[..., n * n + n:], left)


@pytest.mark.parametrize("time_major", [False, True])
def test_into_the_other_half_of_each_step(time_major):
    for dtype in TYPES:
        for n in (4, 7, 128, 700):
            p = _values((6, 9, 2 * n), dtype, n)
            before = p[..., :n].clone()
            _check_elements([p[..., :n]], [int(time_major)], math.sqrt(6 * n) * 0.8, out=[p[..., n:]])
            assert torch.equal(p[..., :n], before)


def test_one_array_of_whole_elements_in_place():
    """[B, 10 + 210 T]: x0, then the steps."""
    B, T = 19, 8
    p = _values((B, 10 + 210 * T), F32, 3)
    steps = p[:, 10:].unflatten(1, (T, 210))
    grads = [p[:, :10], steps[..., :196].unflatten(-1, (14, 14)), steps[..., 196:]]
    _check_elements(grads, [0, 0, 0], 20.0, out=grads)
