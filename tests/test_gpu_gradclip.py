"""Gradient norms and clipping against their definitions in 64 bits.

Tolerances, before any run: a sum of squares is off by at most eight roundings
of 2^-24 (the groups that are added in 32 bits) and what 64-bit sums add, under
2^-45; its root by half of that, the norm as a float by 2^-24 more: 2^-22 +
2^-24 < 2^-21. A coefficient is as far off as the norm it comes from and its
own rounding, a value another rounding to float and one to its own type: 2^-21
relative and eps/2 of the type, and half of the type's smallest step where
values are denormal."""

import math

import numpy as np
import pytest
import torch

import ilqr_native as nat

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
NORM_TOL = 2.0**-21


def _values(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _wide(t):
    return t.detach().double().cpu().numpy()


def _norm64(arrays, p=2.0):
    flat = np.concatenate([a.reshape(-1) for a in arrays]) if arrays else np.zeros(0)
    if flat.size == 0:
        return 0.0
    return float(np.sqrt(np.square(flat).sum())) if p == 2.0 else float(np.abs(flat).max())


def _close_norm(got, want):
    got = float(got)
    if math.isnan(want):
        assert math.isnan(got)
    elif want == 0.0 or want > 3.4028236e38:  # rounds to no float: infinity
        assert got == (math.inf if want else 0.0)
    else:
        # half a step of a denormal float, should the norm be one
        assert abs(got - want) <= NORM_TOL * want + 2.0**-150, (got, want)


def _close_values(got, want):
    """got: a tensor; want: its 64-bit values."""
    t = got.dtype
    g = _wide(got)
    both = np.isnan(want)
    assert np.array_equal(np.isnan(g), both)
    with np.errstate(invalid="ignore"):
        step = torch.finfo(t).smallest_normal * torch.finfo(t).eps
        bar = np.abs(want) * (NORM_TOL + torch.finfo(t).eps / 2) + 0.5 * step
        ok = (np.abs(g - want) <= bar) | both | (g == want)
    assert ok.all(), np.abs(g - want)[~ok].max()


def _coef64(norm, m, eps=1e-6):
    if math.isinf(m):
        return 1.0
    if math.isnan(norm):
        return math.nan
    return 0.0 if math.isinf(norm) else min(1.0, m / (norm + eps))


def _lists(dtype, seed=0):
    """Lists of gradients of every kind of layout."""
    v = lambda *s, k=0: _values(s, dtype, seed + k)
    base = v(1000, k=9)
    return {
        "one value": [v(1)],
        "scalar": [_values((), dtype, seed)],
        "empty ones among others": [v(0), v(5), v(3, 0, 2), v(7)],
        "only empty": [v(0), v(2, 0)],
        "odd": [v(17, k=1), v(3, 5, 7, k=2), v(1, k=3), v(4097, k=4)],
        "long": [v(150_001, k=5)],
        "views at odd offsets": [base[1:18], base[18:19], base[21:400], base[403:]],
        "permuted": [v(6, 5, 4, k=6).permute(2, 0, 1), v(31, 9, k=7).t()],
        "gaps": [v(40, 50, k=8)[:, ::3], base[::7], v(8, 9, k=1)[2:5, 1:4]],
        "expanded": [v(5, k=2).expand(3, 5), v(1, k=3).expand(100)],
    }


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [2.0, math.inf])
def test_norm_of_every_layout(dtype, p):
    for kind, grads in _lists(dtype).items():
        want = _norm64([_wide(g) for g in grads], p)
        _close_norm(nat.grad_norm(grads, p), want)
        norm, norms = nat.grad_norm(grads, p, per_tensor=True)
        assert norm.dtype == F32 and norm.shape == () and norms.shape == (len(grads),), kind
        _close_norm(norm, want)
        for g, n in zip(grads, norms):
            _close_norm(n, _norm64([_wide(g)], p))
        total = nat.grad_norm_total(grads, p)
        assert total.dtype == torch.float64
        _close_norm(math.sqrt(float(total)) if p == 2.0 else float(total), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("part", [0.25, 0.9, 3.0])
def test_clip_of_every_layout(dtype, p, part):
    for kind, grads in _lists(dtype).items():
        before = [_wide(g) for g in grads]
        norm = _norm64(before, p)
        m = part * norm
        c = _coef64(norm, m)
        got, n = nat.clip_grad_norm(grads, m, norm_type=p)
        _close_norm(n, norm)
        for g, o, b in zip(grads, got, before):
            assert o.shape == g.shape and o.dtype == g.dtype and np.array_equal(_wide(g), b), kind
            if part > 1.0:
                assert torch.equal(o, g)
            else:
                _close_values(o, b * c)
        if kind == "expanded":
            with pytest.raises(RuntimeError, match="place"):
                nat.clip_grad_norm(grads, m, norm_type=p, out=grads)
            continue
        # into given outputs of another layout, and in place: the same values
        given = [torch.full((*g.shape, 2), 7.0, dtype=dtype, device=DEV)[..., 0] for g in grads]
        same, _ = nat.clip_grad_norm(grads, m, norm_type=p, out=given)
        assert all(s is o for s, o in zip(same, given)) and all(torch.equal(s, o) for s, o in zip(given, got))
        versions = [g._version for g in grads]
        nat.clip_grad_norm(grads, m, norm_type=p, out=grads)
        assert all(torch.equal(g, o) for g, o in zip(grads, got)), kind
        assert all(g._version > v for g, v in zip(grads, versions))


def test_gaps_keep_what_lies_between():
    base = _values((60, 7), F32, 3)
    kept = base.clone()
    nat.clip_grad_norm([base[::2, 1:4]], 0.5, out=[base[::2, 1:4]])
    mask = torch.ones_like(base, dtype=torch.bool)
    mask[::2, 1:4] = False
    assert torch.equal(base[mask], kept[mask]) and not torch.equal(base, kept)


@pytest.mark.parametrize("dtype,scale", [(F32, 1e30), (F32, 1e-30), (F32, 3e37), (F32, 1e-40), (BF16, 1e30),
                                         (BF16, 1e-30), (BF16, 1e-39), (F16, 1e4), (F16, 1e-7)])
def test_magnitudes_at_the_ends_of_the_range(dtype, scale):
    """Squares that a float cannot hold, coefficients that it cannot either."""
    grads = [_values((777,), dtype, 1, scale), _values((3, 5), dtype, 2, scale), torch.zeros(40, dtype=dtype, device=DEV)]
    before = [_wide(g) for g in grads]
    norm = _norm64(before)
    assert 0.0 < norm < 3.4e38 * 0.99 or scale == 3e37
    if norm < 3.4e38:
        _close_norm(nat.grad_norm(grads), norm)
    for m in (1.0, norm * 0.1, 1e-3):
        got, _ = nat.clip_grad_norm(grads, m, eps=0.0)
        c = min(1.0, m / norm)
        for o, b in zip(got, before):
            _close_values(o, b * c)


def test_norm_beyond_the_floats():
    big = torch.full((100,), 3e38, device=DEV)
    assert float(nat.grad_norm([big])) == math.inf     # 3e39 is no float
    got, _ = nat.clip_grad_norm([big], 10.0, eps=0.0)     # and yet the values are right
    _close_values(got[0], np.full(100, 1.0))


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_infinities_and_nan(p, bad):
    for where in (0, 5, 300, 8191):
        g = [_values((9000,), F32, 4), _values((11,), BF16, 5), _values((3,), F16, 6)]
        g[0][where] = bad
        n, each = nat.grad_norm(g, p, per_tensor=True)
        want = math.nan if math.isnan(bad) else math.inf
        _close_norm(n, want)
        _close_norm(each[0], want)
        _close_norm(each[1], _norm64([_wide(g[1])], p))
        got, _ = nat.clip_grad_norm(g, 1.0, norm_type=p)
        for o, x in zip(got, g):
            with np.errstate(invalid="ignore"):
                assert np.array_equal(_wide(o), _wide(x) * (math.nan if math.isnan(bad) else 0.0), equal_nan=True)
        got, _ = nat.clip_grad_norm(g, math.inf, norm_type=p)
        assert all(np.array_equal(_wide(o), _wide(x), equal_nan=True) for o, x in zip(got, g))
    for order in ([math.nan, math.inf], [math.inf, math.nan]):
        g = [torch.tensor([v], device=DEV) for v in order]
        assert math.isnan(float(nat.grad_norm(g, p)))


def test_bounds_at_their_ends():
    g = [_values((33,), F32, 1)]
    zero, n = nat.clip_grad_norm(g, 0.0)
    assert torch.count_nonzero(zero[0]) == 0
    nothing = [torch.zeros(9, device=DEV)]
    got, n = nat.clip_grad_norm(nothing, 0.0)
    assert float(n) == 0.0 and torch.equal(got[0], nothing[0])
    got, n = nat.clip_grad_norm(nothing, 0.0, eps=0.0)  # 0 / 0, as written
    assert torch.isnan(got[0]).all()


@pytest.mark.parametrize("count", [59, 60, 61, 240, 241, 1000, 1001, 5003])
def test_many_tensors(count):
    """Lists beyond what one launch takes, of mixed types and sizes."""
    rng = np.random.default_rng(count)
    sizes = rng.integers(0, 90, count)
    sizes[rng.integers(0, count, 5)] = 20_011
    grads = [_values((int(s),), TYPES[i % 3], i) for i, s in enumerate(sizes)]
    before = [_wide(g) for g in grads]
    for p in (2.0, math.inf):
        norm, norms = nat.grad_norm(grads, p, per_tensor=True)
        want = _norm64(before, p)
        _close_norm(norm, want)
        _close_norm(nat.grad_norm(grads, p), want)
        each = norms.cpu().numpy()
        for b, e in zip(before, each):
            _close_norm(e, _norm64([b], p))
    want = _norm64(before)
    nat.clip_grad_norm(grads, 0.3 * want, out=grads)
    c = _coef64(want, 0.3 * want)
    for g, b in zip(grads, before):
        _close_values(g, b * c)


def test_long_lists_of_long_tensors():
    """Enough blocks in several launches that their sums are joined first."""
    grads = [_values((30_000,), BF16, i % 7) for i in range(4100)]
    want = _norm64([_wide(g) for g in grads])
    _close_norm(nat.grad_norm(grads), want)
    norm, norms = nat.grad_norm(grads, per_tensor=True)
    _close_norm(norm, want)
    for i in (0, 999, 1000, 4099):
        _close_norm(norms[i], _norm64([_wide(grads[i])]))
    got, n = nat.clip_grad_norm(grads, 0.5 * want)
    _close_norm(n, want)
    for i in (0, 999, 1000, 4099):
        _close_values(got[i], _wide(grads[i]) * _coef64(want, 0.5 * want))


def test_offsets_beyond_32_bits():
    n = 2**31 + 77
    x = torch.full((n,), 0.5, dtype=BF16, device=DEV)
    x[-3:] = 300.0
    want = math.sqrt((n - 3) * 0.25 + 3 * 9e4)
    _close_norm(nat.grad_norm([x]), want)
    assert float(nat.grad_norm([x], math.inf)) == 300.0
    nat.clip_grad_norm([x], want / 2, eps=0.0, out=[x])
    assert float(x[0]) == 0.25 and float(x[2**31 - 1]) == 0.25 and float(x[-1]) == 150.0 and float(x[-4]) == 0.25


def test_total_from_elsewhere():
    a, b = [_values((100,), F32, 1)], [_values((7, 3), BF16, 2), _values((0,), F32, 3)]
    total = nat.grad_norm_total(a) + nat.grad_norm_total(b)
    want = _norm64([_wide(t) for t in a + b])
    got, n = nat.clip_grad_norm(a, 0.5 * want, total=total)
    _close_norm(n, want)
    _close_values(got[0], _wide(a[0]) * _coef64(want, 0.5 * want))
    top = torch.maximum(nat.grad_norm_total(a, math.inf), nat.grad_norm_total(b, math.inf))
    _, n = nat.clip_grad_norm(b, 1.0, norm_type=math.inf, total=top)
    _close_norm(n, _norm64([_wide(t) for t in a + b], math.inf))
    with pytest.raises(RuntimeError, match="total"):
        nat.clip_grad_norm(a, 1.0, total=torch.zeros((), device=DEV))


def test_same_bits_each_time_and_in_every_form():
    grads = [_values((123_457,), F32, 1), _values((99_999,), BF16, 2)]
    first, n0 = nat.clip_grad_norm(grads, 3.0)
    for _ in range(3):
        again, n1 = nat.clip_grad_norm(grads, 3.0)
        assert torch.equal(n0, n1) and all(torch.equal(a, b) for a, b in zip(first, again))
    assert torch.equal(nat.grad_norm(grads), n0)


def test_gpu_refusals():
    x, y = _values((10,), F32, 1), _values((10,), F32, 2)
    with pytest.raises(RuntimeError, match="float32"):
        nat.grad_norm([x.double()])
    with pytest.raises(RuntimeError, match="one device|CUDA"):
        nat.grad_norm([x, y.cpu()])
    with pytest.raises(RuntimeError, match="shares memory"):
        nat.clip_grad_norm([x, x], 1.0, out=[x, x])
    with pytest.raises(RuntimeError, match="shares memory"):
        nat.clip_grad_norm([x[:8]], 1.0, out=[x[1:9]])
    with pytest.raises(RuntimeError, match="out must"):
        nat.clip_grad_norm([x], 1.0, out=[y[:9]])
    with pytest.raises(RuntimeError, match="out must hold 1"):
        nat.clip_grad_norm([x], 1.0, out=[y, y])
    with pytest.raises(RuntimeError, match="require grad"):
        nat.clip_grad_norm([x], 1.0, out=[torch.zeros(10, device=DEV, requires_grad=True)])
    with pytest.raises(RuntimeError, match="sparse|dense"):
        nat.grad_norm([torch.eye(3, device=DEV).to_sparse()])
    with pytest.raises(RuntimeError, match="batch size"):
        nat.clip_grad_elements([x, y[:9]], 1.0)
    with pytest.raises(RuntimeError, match="batch dimension"):
        nat.clip_grad_elements([x], 1.0, batch_dims=1)
    with pytest.raises(RuntimeError, match="1 to 8"):
        nat.clip_grad_elements([x] * 9, 1.0)
    # reading a tensor twice is no conflict
    _close_norm(nat.grad_norm([x, x]), math.sqrt(2.0) * _norm64([_wide(x)]))


# ---- batch elements ---------------------------------------------------------

def _rows64(grads, dims):
    B = grads[0].shape[dims[0]]
    if B == 0:
        return np.zeros(0)
    rows = [np.moveaxis(_wide(g), d, 0).reshape(B, -1) for g, d in zip(grads, dims)]
    return np.sqrt(sum(np.square(r).sum(1) for r in rows))


def _check_elements(grads, dims, m, out=None, zero=False):
    before = [_wide(g) for g in grads]
    with np.errstate(invalid="ignore"):
        norms = _rows64(grads, dims)
    got, n = nat.clip_grad_elements(grads, m, batch_dims=dims, zero_nonfinite=zero, out=out)
    assert n.shape == norms.shape and n.dtype == F32
    for a, b in zip(n.cpu().tolist(), norms.tolist()):
        _close_norm(a, b)
    c = np.array([_coef64(float(v), m) for v in norms])
    for o, b, d in zip(got, before, dims):
        view = [1] * b.ndim
        view[d] = -1
        with np.errstate(invalid="ignore"):
            want = b * c.reshape(view)
            if zero:
                want = np.where(np.isfinite(norms).reshape(view), want, 0.0)
        _close_values(o, want)
        same = np.moveaxis(_wide(o), d, 0)[c == 1.0]
        assert np.array_equal(same, np.moveaxis(b, d, 0)[c == 1.0], equal_nan=True)
    return got, n


def _solver(B, T, n, dtype, time_major, seed=0):
    """x0, C, c gradients whose elements differ widely in size."""
    g = torch.Generator().manual_seed(seed)
    scale = torch.exp(1.5 * torch.randn(B, generator=g)) / math.sqrt(max(1, T) * n * n)
    lead = (T, B) if time_major else (B, T)
    out, dims = [], [0, int(time_major), int(time_major)]
    for shape, d in zip(((B, n - 4), lead + (n, n), lead + (n,)), dims):
        view = [1] * len(shape)
        view[d] = -1
        out.append((torch.randn(shape, generator=g) * scale.view(view)).to(dtype).to(DEV))
    return out, dims


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("time_major", [False, True])
@pytest.mark.parametrize("B,T,n", [(1, 1, 14), (16, 5, 14), (37, 3, 17), (5, 20, 14), (3, 50, 17), (300, 2, 14),
                                   (2, 0, 14), (0, 4, 14), (1, 700, 14)])
def test_elements_of_the_solvers_gradients(B, T, n, dtype, time_major):
    grads, dims = _solver(B, T, n, dtype, time_major, seed=B + T)
    _check_elements(grads, dims, 1.0)
    got, _ = nat.clip_grad_elements(grads, 1.0, batch_dims=dims)
    nat.clip_grad_elements(grads, 1.0, batch_dims=dims, out=grads)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))


@pytest.mark.parametrize("width", [1, 2, 3, 7, 56, 127, 128, 560, 1023, 1024, 1025, 1400, 4097, 30_001])
def test_elements_of_every_width(width):
    B = 11
    for dtype in TYPES:
        x = _values((B, width), dtype, width)
        x *= torch.linspace(0.1, 3.0, B, device=DEV).to(dtype).unsqueeze(1)
        _check_elements([x], [0], math.sqrt(width))
    odd = _values((B, width + 1), F32, width)
    _check_elements([odd[:, 1:], odd[:, :1]], [0, 0], math.sqrt(width))  # columns of one array
    _check_elements([odd[:, 1:], odd[:, :1]], [0, 0], math.sqrt(width), out=[odd[:, 1:], odd[:, :1]])


def test_elements_longer_than_shared_memory():
    """Elements that a cluster's blocks share, and those that no block can hold."""
    for shape, d in (((3, 90_001), 0), ((2, 500_003), 0), ((2, 3, 300_001), 1), ((61, 3, 5003), 1), ((9, 2, 30_000), 1),
                     ((5, 1, 70_000), 1), ((1, 300_000), 0)):
        for dtype in TYPES:
            x = _values(shape, dtype, 3)
            y = _values((shape[d], 77), F32, 4)
            width = x.numel() // shape[d]
            x.select(d, 0).mul_(0.2)
            _check_elements([y, x], [0, d], math.sqrt(width) * 0.7)
            _check_elements([y, x], [0, d], math.sqrt(width) * 0.7, out=[y, x])
    x = _values((2, 100_000), F32, 5)
    x[1, 70_000] = math.inf
    for zero in (False, True):
        _check_elements([x], [0], 3.0, zero=zero)
    _check_elements([x[:1]], [0], 1e-36)             # a coefficient below the floats' range


def test_elements_of_other_layouts():
    B = 9
    x = _values((4, B, 3, 5), F32, 1)
    _check_elements([x.permute(1, 0, 2, 3)], [0], 4.0)                      # time-major seen batch first
    _check_elements([x.permute(1, 0, 2, 3)], [0], 4.0, out=[torch.empty(B, 4, 3, 5, device=DEV)])
    _check_elements([_values((6, B), BF16, 2)], [1], 2.0)                    # batch last
    _check_elements([_values((B, 6, 8, 10), F32, 3)[:, ::2, ::2, 1:]], [0], 5.0)
    _check_elements([_values((1,), F32, 4).expand(B, 4)], [0], 0.5)
    _check_elements([_values((2 * B, 12), F16, 5)[::2]], [0], 2.0)           # every other element
    _check_elements([_values((B,), F32, 6), _values((3, B), BF16, 7)], [0, 1], 0.7)
    mixed = [_values((B, 40), d, k) for k, d in enumerate(TYPES)]
    _check_elements(mixed, [0, 0, 0], 6.0)
    eight = [_values((B, k + 1), TYPES[k % 3], k) for k in range(8)]
    _check_elements(eight, [0] * 8, 3.0)
    with pytest.raises(RuntimeError, match="place"):
        e = _values((1,), F32, 4).expand(B, 4)
        nat.clip_grad_elements([e], 0.5, out=[e])


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("time_major", [False, True])
def test_elements_that_diverged_leave_the_others(zero, time_major):
    B = 24
    grads, dims = _solver(B, 6, 14, F32, time_major, seed=5)
    grads[0][3, 2] = math.inf
    grads[1].select(dims[1], 7).fill_(math.nan)
    grads[2].select(dims[2], 11)[1] = -math.inf
    grads[0][20] = 3e38                              # finite, however large
    for inplace in (False, True):
        use = [g.clone() for g in grads]
        got, n = _check_elements(use, dims, 0.5, out=use if inplace else None, zero=zero)
        fine = [b for b in range(B) if b not in (3, 7, 11)]
        for o, d in zip(got, dims):
            assert torch.isfinite(o.movedim(d, 0)[fine]).all()
            if zero:
                assert torch.count_nonzero(o.movedim(d, 0)[[3, 7, 11]]) == 0


@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-42])
def test_elements_at_the_ends_of_the_range(scale):
    x = _values((6, 130), F32, 8, scale)
    _check_elements([x], [0], 1.0 if scale > 1 else float(scale))


def test_elements_equal_the_list_form_for_one_element():
    x = [_values((1, 500), F32, 1), _values((1, 77), BF16, 2)]
    a, n = nat.clip_grad_elements(x, 2.0)
    b, m = nat.clip_grad_norm(x, 2.0)
    _close_norm(float(n[0]), float(m))
    for u, v in zip(a, b):
        _close_values(u, _wide(v))


# ---- streams and graphs ------------------------------------------------------

def test_on_another_stream():
    x = [_values((50_000,), F32, 1), _values((301,), BF16, 2)]
    want, n0 = nat.clip_grad_norm(x, 1.0)
    rows = [_values((64, 900), F32, 3)]
    want_rows, r0 = nat.clip_grad_elements(rows, 1.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, n1 = nat.clip_grad_norm(x, 1.0)
        got_rows, r1 = nat.clip_grad_elements(rows, 1.0)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(n0, n1) and torch.equal(r0, r1) and torch.equal(want_rows[0], got_rows[0])
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_two_graphs_replayed_with_new_values():
    shapes = [(30_000,), (17,), (40, 41)]
    graphs = []
    for k in range(2):
        x = [_values(s, F32, 10 * k + i) for i, s in enumerate(shapes)]
        rows = [_values((33, 700), F32, 50 + k)]
        nat.clip_grad_norm(x, 2.0), nat.grad_norm(x, per_tensor=True), nat.clip_grad_elements(rows, 3.0)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, n = nat.clip_grad_norm(x, 2.0)
            m, each = nat.grad_norm(x, per_tensor=True)
            ro, rn = nat.clip_grad_elements(rows, 3.0)
        graphs.append((g, x, rows, out, n, m, each, ro, rn))
    for turn in range(3):
        for k, (g, x, rows, *_) in enumerate(graphs):
            for i, t in enumerate(x + rows):
                t.copy_(_values(tuple(t.shape), F32, 100 * turn + 10 * k + i, 1.0 + turn))
        for k in (0, 1) if turn % 2 == 0 else (1, 0):
            graphs[k][0].replay()
        torch.cuda.synchronize()
        for g, x, rows, out, n, m, each, ro, rn in graphs:
            want, n0 = nat.clip_grad_norm(x, 2.0)
            assert torch.equal(n, n0)
            m0, each0 = nat.grad_norm(x, per_tensor=True)
            assert torch.equal(m, m0) and torch.equal(each, each0)
            assert all(torch.equal(a, b) for a, b in zip(want, out))
            wr, w0 = nat.clip_grad_elements(rows, 3.0)
            assert torch.equal(w0, rn) and torch.equal(wr[0], ro[0])


# ---- what lies around, and the first call --------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [5, 56, 131, 700, 2900, 40_003])
def test_elements_leave_what_lies_around_them(dtype, width):
    """Slices at every offset within 16 bytes of a wider array, in place and into
    another array at the same and at another offset: nothing else is written."""
    B, room = 6, 16
    for at in range(0, 9, 1 if width < 200 else 3):
        for d in (0, 1):
            shape = (B, width + room) if d == 0 else (3, B, width + room)
            base = torch.full(shape, 7.0, dtype=dtype, device=DEV)
            x = base[..., at:at + width]
            x.copy_(_values(tuple(x.shape), dtype, width + at))
            start = base.clone()
            other = torch.full_like(base, 5.0)
            for to in (at, at + 1):
                y = other[..., to:to + width]
                want, n = _check_elements([x], [d], math.sqrt(width) * 0.9, out=[y])
                kept = other.clone()
                kept[..., to:to + width] = 5.0
                assert torch.equal(kept, torch.full_like(kept, 5.0)) and torch.equal(base, start)
                if to == at:  # the same words, so the same order of the sums
                    done = y.clone()
                other.fill_(5.0)
            _check_elements([x], [d], math.sqrt(width) * 0.9, out=[x])
            assert torch.equal(x, done)
            start[..., at:at + width] = x
            assert torch.equal(base, start)


def test_elements_without_values():
    for dims, x in (([0], [torch.zeros(4, 0, device=DEV)]), ([1], [torch.zeros(0, 4, 3, device=DEV)])):
        got, n = nat.clip_grad_elements(x, 1.0, batch_dims=dims)
        assert n.tolist() == [0.0] * 4 and got[0].shape == x[0].shape
    got, n = nat.clip_grad_elements([torch.zeros(0, 9, device=DEV)], 1.0)
    assert n.shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
def test_list_leaves_what_lies_around_it(dtype):
    """Views at every offset, small and long lists, in place and into outputs
    that lie otherwise in their 16-byte words."""
    for n in (3, 100, 5000, 70_001):
        for at in (0, 1, 3, 7):
            base = torch.full((n + 20,), 7.0, dtype=dtype, device=DEV)
            x = base[at:at + n]
            x.copy_(_values((n,), dtype, n))
            other = torch.full_like(base, 5.0)
            m = 0.5 * _norm64([_wide(x)])
            c = _coef64(_norm64([_wide(x)]), m)
            want = _wide(x) * c
            for to in (at, at + 1, at + 4):
                y = other[to:to + n]
                nat.clip_grad_norm([x], m, out=[y])
                _close_values(y, want)
                y.fill_(5.0)
                assert torch.equal(other, torch.full_like(other, 5.0))
            nat.clip_grad_norm([x], m, out=[x])
            _close_values(x, want)
            rest = torch.cat([base[:at], base[at + n:]])
            assert torch.equal(rest, torch.full_like(rest, 7.0))


@pytest.mark.parametrize("dtype,n", [(F32, 20_000_001), (BF16, 40_000_003)])
def test_lists_beyond_l2(dtype, n):
    """The form for lists that do not stay in L2, out of place, in place, below
    the bound, and with a total from elsewhere."""
    flat = _values((n,), dtype, 1)
    sizes = [n // 3, 1, n // 2, 17]
    sizes.append(n - sum(sizes))
    x = list(flat.split(sizes))
    before = _wide(flat)
    norm = float(np.sqrt(np.square(before).sum()))
    c = _coef64(norm, 0.3 * norm)
    got, nn = nat.clip_grad_norm(x, 0.3 * norm)
    _close_norm(nn, norm)
    _close_values(torch.cat(got), before * c)
    again, _ = nat.clip_grad_norm(x, 0.3 * norm, total=nat.grad_norm_total(x))
    _close_values(torch.cat(again), before * c)
    nat.clip_grad_norm(x, 2.0 * norm, out=x)
    assert np.array_equal(_wide(flat), before)
    top = float(np.abs(before).max())
    got, nn = nat.clip_grad_norm(x, 0.5 * top, norm_type=math.inf)
    assert float(nn) == np.float32(top)
    _close_values(torch.cat(got), before * _coef64(top, 0.5 * top))
    nat.clip_grad_norm(x, 0.3 * norm, out=x)
    _close_values(flat, before * c)


PROGRAM = """
import sys
sys.path[:0] = [{root!r}, {pkg!r}]
import torch
import ilqr_native as nat
x = [torch.ones(100_000, device="cuda"), torch.ones(3, device="cuda")]
y = [torch.ones(5, 700, device="cuda"), torch.ones(5, 40_000, device="cuda")]
s = torch.cuda.Stream()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    a, n = nat.clip_grad_norm(x, 1.0)
    b, m = nat.clip_grad_elements(y, 1.0)
    k = nat.grad_norm(x, per_tensor=True)
g.replay()
torch.cuda.synchronize()
assert abs(float(n) - 100_003 ** 0.5) < 1e-3 and abs(float(m[3]) - 40_700 ** 0.5) < 1e-3
assert abs(float(a[0][5]) * float(n) - 1) < 1e-5 and abs(float(b[1][4, 9]) * float(m[4]) - 1) < 1e-5
"""


def test_first_calls_of_a_process_are_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM.format(root=root, pkg=os.path.join(root, "ca-ac-mpc_b200"))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_threads_at_once():
    """Calls from two Python threads on streams of their own."""
    import threading
    data = [[_values((60_000,), F32, k), _values((40, 3000), BF16, 9 + k)] for k in range(2)]
    want = [(nat.clip_grad_norm(d, 2.0), nat.clip_grad_elements(d[1:], 2.0)) for d in data]
    torch.cuda.synchronize()
    fails = []

    def work(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(50):
                (a, n), (b, m) = nat.clip_grad_norm(data[k], 2.0), nat.clip_grad_elements(data[k][1:], 2.0)
                s.synchronize()
                (a0, n0), (b0, m0) = want[k]
                same = torch.equal(n, n0) and torch.equal(m, m0) and all(map(torch.equal, a + b, a0 + b0))
                if not same:
                    fails.append(k)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not fails
