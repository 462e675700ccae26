"""The paths that clip gradients: the MPC operator's backward, the policy
actor, the trainer's parameter gradients and a sharded batch, against the same
backward without clipping and the formula in 64 bits. Tolerances as in
test_gpu_gradclip.py (2^-21 of a value and half a step of its type), and where
clipped gradients run on through a network's float32 products, the error that
those can make of it: the products' length times 2^-24 of the sums of
magnitudes."""

import math
import os
import socket

import numpy as np
import pytest
import torch

import ilqr_native as nat
import ilqr_shard
import ilqr_workload as wl
import mpc_compat
import policy_mpc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DX = type("Dx", (), {"dt": wl.DT})()
TOL = 2.0**-21 + 2.0**-24


def _t(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def _sigmoid(B, T, seed):
    rng = np.random.default_rng(seed)
    return _t((1 / (1 + np.exp(-rng.normal(0, 1.5, (B, 28 * T))))).astype(np.float32))


def _grads(kind, B, T, seed=0, spoil=None, backprop=True, **clip):
    """Gradients (batch first, 64 bits) of x_init and the costs through the
    operator, its outputs and the operator; spoil: elements whose incoming
    gradient is infinite."""
    n = 13 if kind == "rotor13" else 10
    inp = wl.make_rotor13_inputs(B, T, seed=seed) if n == 13 else wl.make_inputs(B, T, seed=seed)
    gX, gU = (_t(g) for g in wl.make_backward_seeds(B, T, nx=n))
    if spoil is not None:
        gU[spoil, 0, 0] = math.inf
    lo, hi = (wl.U_MIN13, wl.U_MAX13) if n == 13 else (wl.U_MIN, wl.U_MAX)
    box = lambda v: _t(np.broadcast_to(v, (T, 1, 4)))
    numerics = "fastmpc" if kind.startswith("fastmpc") else "diffmpc"
    mpc = mpc_compat.MPC(n, 4, T, u_lower=box(lo), u_upper=box(hi), lqr_iter=2, eps=1e-6, numerics=numerics, **clip)
    x0 = _t(inp["x0"]).requires_grad_(True)
    leaves = [x0]
    if kind.endswith("sigmoid"):
        sc = _sigmoid(B, T, seed + 1).requires_grad_(True)
        leaves.append(sc)
        cost = mpc_compat.SigmoidQuadCost(sc, range_q=10.0, range_p=10.0)
    else:
        C = _t(np.transpose(inp["C"], (1, 0, 2, 3))).requires_grad_(True)
        c = _t(np.transpose(inp["c"], (1, 0, 2))).requires_grad_(True)
        leaves += [C, c]
        cost = mpc_compat.QuadCost(C, c)
    x, u, _ = mpc(x0, cost, DX)
    torch.autograd.backward([x, u], [gX.permute(1, 0, 2), gU.permute(1, 0, 2)])
    got = [(v.grad if v.dim() < 3 else v.grad.transpose(0, 1)).double().cpu().numpy() for v in leaves]
    return got, (x.detach(), u.detach()), mpc


def _row_norms(grads):
    return np.sqrt(sum(np.square(g.reshape(g.shape[0], -1)).sum(1) for g in grads))


def _assert_close(got, want):
    bar = TOL * np.abs(want) + 2.0**-150
    assert (np.abs(got - want) <= bar).all(), (np.abs(got - want) - bar).max()


KINDS = ["dense", "sigmoid", "rotor13", "fastmpc", "fastmpc_sigmoid"]


@pytest.mark.parametrize("kind", KINDS)
def test_operator_clips_each_element(kind):
    B, T = 23, 6
    free, out0, _ = _grads(kind, B, T)
    norms = _row_norms(free)
    m = float(np.median(norms))
    got, out1, mpc = _grads(kind, B, T, max_grad_norm=m)
    assert all(torch.equal(a, b) for a, b in zip(out0, out1))
    assert mpc.grad_norms.shape == (B,)
    _assert_close(mpc.grad_norms.double().cpu().numpy(), norms)
    c = np.minimum(1.0, m / (norms + 1e-6))
    assert 0 < (c < 1).sum() < B
    for g, f in zip(got, free):
        _assert_close(g, f * c.reshape(-1, *[1] * (f.ndim - 1)))
        assert np.array_equal(g[norms < 0.999 * m], f[norms < 0.999 * m])


@pytest.mark.parametrize("kind", KINDS)
def test_operator_clips_the_batch(kind):
    B, T = 23, 6
    free, _, _ = _grads(kind, B, T)
    norm = float(np.sqrt(sum(np.square(g).sum() for g in free)))
    got, _, mpc = _grads(kind, B, T, max_grad_norm=0.3 * norm, grad_clip="batch")
    assert mpc.grad_norms.shape == ()
    assert abs(float(mpc.grad_norms) - norm) <= TOL * norm
    for g, f in zip(got, free):
        _assert_close(g, f * (0.3 * norm / (norm + 1e-6)))
    got, _, _ = _grads(kind, B, T, max_grad_norm=3.0 * norm, grad_clip="batch")
    assert all(np.array_equal(g, f) for g, f in zip(got, free))


@pytest.mark.parametrize("kind", KINDS)
def test_operator_sets_diverged_elements_to_zero(kind):
    B, T = 12, 5
    free, _, _ = _grads(kind, B, T)
    got, _, mpc = _grads(kind, B, T, spoil=[4, 9], zero_nonfinite_grad=True)
    rest = [b for b in range(B) if b not in (4, 9)]
    for g, f in zip(got, free):
        assert np.array_equal(g[rest], f[rest]) and not g[[4, 9]].any()
    assert not torch.isfinite(mpc.grad_norms[[4, 9]]).any() and torch.isfinite(mpc.grad_norms[rest]).all()


def test_no_clipping_is_what_it_was_and_refusals():
    got, _, mpc = _grads("dense", 5, 3)
    assert mpc.grad_clip is None and mpc.grad_norms is None
    again, _, _ = _grads("dense", 5, 3, max_grad_norm=math.inf)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))
    none, _, mpc = _grads("dense", 0, 3, max_grad_norm=1.0)
    assert mpc.grad_norms.shape == (0,)


def test_only_the_gradients_asked_for_count():
    B, T = 7, 4
    inp = wl.make_inputs(B, T, seed=3)
    C, c = _t(np.transpose(inp["C"], (1, 0, 2, 3))), _t(np.transpose(inp["c"], (1, 0, 2)))
    grads = []
    for m in (None, 1e-3):
        mpc = mpc_compat.MPC(10, 4, T, lqr_iter=2, max_grad_norm=m)
        x0 = _t(inp["x0"]).requires_grad_(True)
        x, u, _ = mpc(x0, mpc_compat.QuadCost(C, c), DX)
        u.sum().backward()
        grads.append(x0.grad.double().cpu().numpy())
    norms = _row_norms(grads[:1])
    _assert_close(grads[1], grads[0] * np.minimum(1.0, 1e-3 / (norms + 1e-6))[:, None])


def test_broadcast_cost_sums_the_clipped_elements():
    """A cost [14, 14] for the whole batch: its gradient is the sum over
    elements and steps of what each clipped element contributes."""
    B, T = 9, 3
    inp = wl.make_inputs(B, T, seed=3)
    one = torch.diag(torch.linspace(0.5, 2.0, 14)).to(DEV)
    full = one.expand(T, B, 14, 14)
    c = _t(np.transpose(inp["c"], (1, 0, 2)))
    res = []
    for C in (one.clone().requires_grad_(True), full.clone().requires_grad_(True)):
        mpc = mpc_compat.MPC(10, 4, T, lqr_iter=2, max_grad_norm=0.01)
        x, u, _ = mpc(_t(inp["x0"]), mpc_compat.QuadCost(C, c), DX)
        (x.sum() + u.sum()).backward()
        res.append(C.grad.double().cpu().numpy())
        assert (mpc.grad_norms > 0.01).any()
    want, mags = res[1].sum((0, 1)), np.abs(res[1]).sum((0, 1))
    assert (np.abs(res[0] - want) <= B * T * 2.0**-24 * mags + 1e-30).all()


# ---- the trainer's side ------------------------------------------------------

def _net(seed, out):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(10, 33), torch.nn.Tanh(), torch.nn.Linear(33, out), torch.nn.Sigmoid()).to(DEV)


def test_parameter_clipping_matches_torch():
    for part in (0.2, 5.0):
        for p in (2.0, math.inf):
            a, b = _net(1, 56), _net(1, 56)
            x = torch.randn(20, 10, device=DEV)
            for net in (a, b):
                (net(x).square().sum() * 3.0).backward()
            bound = part * float(torch.nn.utils.get_total_norm([q.grad for q in a.parameters()], p))
            na = torch.nn.utils.clip_grad_norm_(a.parameters(), bound, norm_type=p)
            nb = policy_mpc.clip_grad_norm_(b.parameters(), bound, norm_type=p)
            # both sides are within their own roundings of the exact ones
            assert abs(float(na) - float(nb)) <= 2.0**-18 * float(na)
            for u, v in zip(a.parameters(), b.parameters()):
                assert torch.allclose(u.grad, v.grad, rtol=2.0**-18, atol=0.0)


def test_parameter_clipping_takes_what_torch_takes():
    lone = torch.zeros(3, device=DEV, requires_grad=True)
    assert float(policy_mpc.clip_grad_norm_([lone], 1.0)) == 0.0       # no gradient yet
    assert float(policy_mpc.clip_grad_norm_([], 1.0)) == 0.0
    lone.grad = torch.tensor([3.0, 0.0, 4.0], device=DEV)
    assert float(policy_mpc.clip_grad_norm_(lone, 1.0)) == 5.0          # one tensor, not a list
    assert torch.allclose(lone.grad, torch.tensor([0.6, 0.0, 0.8], device=DEV), rtol=1e-6)
    half = torch.zeros(2, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    half.grad = torch.tensor([math.inf, 1.0], device=DEV, dtype=torch.bfloat16)
    kept = lone.grad.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        policy_mpc.clip_grad_norm_(iter([lone, half]), 1.0, error_if_nonfinite=True)
    assert torch.equal(lone.grad, kept)
    assert math.isinf(float(policy_mpc.clip_grad_norm_([lone, half], 1.0)))
    assert torch.count_nonzero(lone.grad) == 0


def test_a_training_step_from_actor_to_update():
    """Backward through the actor with elements clipped, then the network's
    gradients clipped together: against the unclipped backward, the formula
    and the network's own backward."""
    B, T, m_el = 31, 2, 0.05
    inp = wl.make_inputs(B, T, seed=7)
    states = _t(inp["x0"])

    def step(**clip):
        net = _net(3, 28 * T)
        pm = policy_mpc.PolicyMPC(T, 0.05, lqr_iter=2, eps=0.1, device=DEV, **clip)
        sc = net(states)
        sc.retain_grad()
        pm.actor(sc, states).square().sum().backward()
        return net, pm, sc

    _, _, free = step()
    net, pm, sc = step(max_grad_norm=m_el * 1e-3, zero_nonfinite_grad=True)
    g = free.grad.double().cpu().numpy()
    norms = np.sqrt(np.square(g).sum(1))
    c = np.minimum(1.0, m_el * 1e-3 / (norms + 1e-6))
    assert (c < 1).any()
    _assert_close(pm.solver.grad_norms.double().cpu().numpy(), norms)
    _assert_close(sc.grad.double().cpu().numpy(), g * c[:, None])
    # what the network makes of the clipped rows
    other = _net(3, 28 * T)
    want = torch.autograd.grad(other(states), list(other.parameters()), sc.grad)
    for p, w in zip(net.parameters(), want):
        assert torch.equal(p.grad, w)
    total = math.sqrt(sum(float(w.double().square().sum()) for w in want))
    n = policy_mpc.clip_grad_norm_(net.parameters(), 0.5 * total)
    assert abs(float(n) - total) <= TOL * total
    scale = 0.5 * total / (total + 1e-6)
    for p, w in zip(net.parameters(), want):
        _assert_close(p.grad.double().cpu().numpy(), w.double().cpu().numpy() * scale)


def test_backward_and_clipping_in_one_graph():
    """The solver's backward and the clipping of its gradients, captured and
    replayed for other incoming gradients."""
    B, T = 19, 5
    inp = wl.make_inputs(B, T, seed=2)
    r = nat.solve(_t(inp["x0"]), _t(inp["U_init"]), _t(inp["C"]), _t(inp["c"]), None, None, None, None, _t(wl.U_MIN),
                  _t(wl.U_MAX), dt=wl.DT, max_iter=2)
    gX, gU = (_t(g) for g in wl.make_backward_seeds(B, T))

    def both():
        g = nat.backward(r["X"], r["U"], C, gX, gU, tight=r["tight"], dt=wl.DT)
        held = [g[k] for k in ("x0", "C", "c")]
        _, norms = nat.clip_grad_elements(held, 0.5, out=held)
        total = nat.grad_norm(held)
        return held, norms, total

    C = _t(inp["C"])
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for seed in (4, 5):
        for dst, src in zip((gX, gU), wl.make_backward_seeds(B, T, seed=seed)):
            dst.copy_(_t(src))
        graph.replay()
        want = both()
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
        assert all(torch.equal(a, b) for a, b in zip(got[0], want[0]))


def test_sharded_clipping_with_one_rank():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    import torch.distributed as dist
    dist.init_process_group("gloo", rank=0, world_size=1)
    try:
        for p in (2.0, math.inf):
            g = {"x0": torch.randn(6, 10, device=DEV), "C": torch.randn(6, 3, 14, 14, device=DEV)}
            want, n0 = nat.clip_grad_norm(list(g.values()), 0.7, norm_type=p)
            n = ilqr_shard.clip_gradients(g, 0.7, norm_type=p)
            assert abs(float(n) - float(n0)) <= TOL * float(n0)
            for a, b in zip(g.values(), want):
                assert torch.allclose(a, b, rtol=2.0**-21, atol=0.0)
    finally:
        dist.destroy_process_group()
