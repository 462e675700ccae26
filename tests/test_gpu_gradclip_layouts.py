"""Gradients that lie between one another in one array, clipped in place and
into each other's gaps, against the definition in 64 bits (tolerances as in
test_gpu_gradclip.py)."""

import math

import pytest
import torch

import ilqr_native as nat
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


# ---- outputs with gaps -----------------------------------------------------------

def _refused(call, *tensors):
    """The call is refused and writes nothing."""
    kept = [t.clone() for t in tensors]
    with pytest.raises(RuntimeError, match="shares memory"):
        call()
    assert all(torch.equal(t, k) for t, k in zip(tensors, kept))


def test_outputs_with_gaps_that_share_memory_are_refused():
    for dtype in TYPES:
        g, h, y = (_values((s,), dtype, k) for k, s in enumerate((50, 50, 200)))
        other = _values((100,), dtype, 9)
        strided = _values((100,), dtype, 8)[::2]
        for form in (nat.clip_grad_norm, nat.clip_grad_elements):
            # an output's gaps hold another output's values, or not
            _refused(lambda: form([g, h], 0.5, out=[y[:100:2], y[:50]]), y)
            _refused(lambda: form([h, g], 0.5, out=[y[:50], y[:100:2]]), y)
            _refused(lambda: form([g, h], 0.5, out=[y[:100:2], y[98:198:2]]), y)
            # the same gradient twice, in place
            _refused(lambda: form([strided, strided], 0.5, out=[strided, strided]), strided)
            # another tensor's input, and its own shifted
            _refused(lambda: form([other[::2], y[:50]], 0.5, out=[y[1:100:2], h]), y, h)
            _refused(lambda: form([y[:50], other[::2]], 0.5, out=[h, y[1:100:2]]), y, h)
            _refused(lambda: form([y[:100:2]], 0.5, out=[y[2:102:2]]), y)
        # elements whose values have two strides
        q, out = _values((6, 8, 10), dtype, 3), torch.empty(3, 4, 5, dtype=dtype, device=DEV)
        a, b = q[:3, :4, ::2], q[3:, 4:, ::2]
        _refused(lambda: nat.clip_grad_elements([a, b], 0.5, out=[b, a]), q)
        _refused(lambda: nat.clip_grad_elements([out, a], 0.5, out=[b, q[3:, 4:, :5]]), q)
        _refused(lambda: nat.clip_grad_elements([a, out], 0.5, out=[out, q[2:5, :4, :5]]), q, out)
        # outputs that the kernels write as they lie, over another's gathered input
        _refused(lambda: nat.clip_grad_norm([y[:100:2], g], 0.5, out=[other[::2], y[50:100]]), y, other)


def test_outputs_in_each_others_gaps_are_taken():
    for dtype in TYPES:
        for form, dims in ((nat.clip_grad_norm, ()), (nat.clip_grad_elements, (0,))):
            g, h = _values((50,), dtype, 1), _values((50,), dtype, 2)
            want = [t.clone() for t in form([g, h], 3.0, *dims)[0]]
            y = torch.full((100,), 7.0, dtype=dtype, device=DEV)
            form([g, h], 3.0, *dims, out=[y[::2], y[1::2]])
            assert torch.equal(y[::2], want[0]) and torch.equal(y[1::2], want[1])
            p = torch.stack([g, h], 1)
            form([p[:, 0], p[:, 1]], 3.0, *dims, out=[p[:, 0], p[:, 1]])
            assert torch.equal(p[:, 0], want[0]) and torch.equal(p[:, 1], want[1])
            p = torch.stack([g, torch.full_like(g, 7.0)], 1)
            form([p[:, 0], h], 3.0, *dims, out=[p[:, 1], h])
            assert torch.equal(p[:, 1], want[0]) and torch.equal(p[:, 0], g) and torch.equal(h, want[1])
            # three strides, blocks of one array
            q = _values((6, 8, 10), dtype, 3)
            parts = [q[:3, :4, ::2], q[:3, :4, 1::2], q[3:, 4:, :5], q[3:, :4, 5:]]
            kept = q[:3, 4:].clone()
            want = [t.clone() for t in form(parts, 2.0, *dims)[0]]
            form(parts, 2.0, *dims, out=parts)
            assert all(torch.equal(a, b) for a, b in zip(parts, want)) and torch.equal(q[:3, 4:], kept)


def test_in_place_through_another_view():
    """The same values seen through strides that differ where there is one step."""
    for form in (nat.clip_grad_norm, nat.clip_grad_elements):
        y = _values((20,), F32, 4)
        want = form([y.as_strided((10, 1), (2, 1))], 0.1)[0][0]
        form([y.as_strided((10, 1), (2, 1))], 0.1, out=[y.as_strided((10, 1), (2, 7))])
        assert torch.equal(y[::2], want[:, 0])


def test_a_total_within_an_output_is_refused():
    g = _values((400,), F32, 1)
    y = torch.zeros(800, device=DEV)
    total = y.view(torch.float64)[30]                # values 60 and 61
    total.copy_(nat.grad_norm_total([g]))
    _refused(lambda: nat.clip_grad_norm([g], 0.5, total=total, out=[y[:400]]), y)
    _refused(lambda: nat.clip_grad_norm([g], 0.5, total=total, out=[y[::2]]), y)
    got, n = nat.clip_grad_norm([g], 0.5, total=total, out=[y[62:462]])
    want, m = nat.clip_grad_norm([g], 0.5, total=total.clone(), out=[torch.zeros(800, device=DEV)[62:462]])
    assert torch.equal(n, m) and torch.equal(got[0], want[0])
    # one that is part of a gradient that is only read
    both, n = nat.clip_grad_norm([y[60:62]], 0.5, total=total)
    assert torch.equal(n, m)


def test_empty_tensors_of_every_shape():
    """An element has no values in them, whatever their strides and batch dimension."""
    import itertools
    full = [_values((4, 6, 8), F32, k)[..., 1:] for k in range(8)]
    for shape in itertools.product((0, 1, 3), repeat=4):
        if 0 not in shape:
            continue
        wide = torch.zeros([2 * s + 1 for s in shape], device=DEV)
        gaps = wide[tuple(slice(0, 2 * s, 2) for s in shape)]
        assert gaps.shape == shape
        for dim, B in enumerate(shape):
            x = _values((B, 7), F32, dim)
            for empty in (torch.zeros(shape, device=DEV), gaps, gaps.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0)):
                for out in (None, [empty, x]):
                    # right after a call whose layouts have values everywhere
                    nat.clip_grad_elements(full, 1.0, out=full)
                    _, n = nat.clip_grad_elements([empty], 1.0, batch_dims=dim, out=out and [empty])
                    assert n.tolist() == [0.0] * B
                    _check_elements([empty, x], [dim, 0], 1.5, out=out)


def test_every_second_row_beside_all_rows():
    base = _values((30_000, 64), F32, 2)
    grads = [base[:, :32].t(), base[::2, 32:], base[1::2, 40:]]
    left = base[1::2, 32:40].clone()
    want = [t.clone() for t in nat.clip_grad_norm(grads, 3.0)[0]]
    nat.clip_grad_norm(grads, 3.0, out=grads)
    assert all(torch.equal(a, b) for a, b in zip(grads, want)) and torch.equal(base[1::2, 32:40], left)
    _refused(lambda: nat.clip_grad_norm(grads, 3.0, out=[grads[0], grads[1], base[::2, 40:]]), base)
