"""CPU tests of the clipping of a policy's parameters, with plain stand-ins for
the two native calls that it makes."""

import inspect
import math

import pytest
import torch

import policy_mpc


class _Plain:
    """The native calls in plain form, and what they were given."""

    def __init__(self):
        self.calls = []

    def grad_norm_total(self, grads, norm_type=2.0):
        assert not torch.is_grad_enabled() and isinstance(norm_type, float)
        self.calls.append(("total", list(grads)))
        flat = torch.cat([g.detach().reshape(-1).double() for g in grads])
        return flat.square().sum() if norm_type == 2.0 else flat.abs().max()

    def clip_grad_norm(self, grads, max_norm, norm_type=2.0, eps=1e-6, total=None, out=None):
        assert not torch.is_grad_enabled() and isinstance(norm_type, float) and out is grads
        if total is None:
            total = self.grad_norm_total(grads, norm_type)
            self.calls.pop()
        self.calls.append(("clip", list(grads)))
        norm = total.sqrt() if norm_type == 2.0 else total
        for g in out:
            g.mul_((max_norm / (norm + eps)).clamp(max=1.0).to(g.dtype))
        return out, norm.float()


@pytest.fixture
def plain(monkeypatch):
    p = _Plain()
    monkeypatch.setattr(policy_mpc._nat, "grad_norm_total", p.grad_norm_total)
    monkeypatch.setattr(policy_mpc._nat, "clip_grad_norm", p.clip_grad_norm)
    return p


def _net():
    torch.manual_seed(3)
    net = torch.nn.Sequential(torch.nn.Linear(4, 9), torch.nn.Tanh(), torch.nn.Linear(9, 2))
    net(torch.randn(7, 4)).square().sum().backward()
    return net


def test_arguments_are_torchs():
    ours = inspect.signature(policy_mpc.clip_grad_norm_).parameters
    theirs = inspect.signature(torch.nn.utils.clip_grad_norm_).parameters
    assert list(ours) == [p for p in theirs if p != "foreach"]
    assert all(ours[p].default == theirs[p].default for p in ours)


@pytest.mark.filterwarnings("ignore:Using backward")
def test_gradients_with_history_are_clipped(plain):
    """Those of a backward with create_graph=True (a gradient penalty's)."""
    w = torch.randn(5, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
    (w.pow(3).sum()).backward(create_graph=True)
    assert w.grad.requires_grad
    before, version = w.grad.detach().clone(), w.grad._version
    n = policy_mpc.clip_grad_norm_([w], 0.5)
    assert torch.is_grad_enabled() and not n.requires_grad and w.grad._version > version
    assert torch.allclose(w.grad.detach(), before * 0.5 / (before.norm() + 1e-6))
    w.grad = None


def test_norm_types_that_torch_takes(plain):
    for given, want in (("inf", math.inf), (math.inf, math.inf), ("2", 2.0), (2, 2.0), (torch.tensor(2.0), 2.0)):
        a, b = _net(), _net()
        bound = 0.3 * float(torch.nn.utils.get_total_norm([q.grad for q in a.parameters()], want))
        na = torch.nn.utils.clip_grad_norm_(a.parameters(), bound, norm_type=given)
        nb = policy_mpc.clip_grad_norm_(b.parameters(), bound, norm_type=given)
        assert math.isclose(float(na), float(nb), rel_tol=2.0**-18)
        for u, v in zip(a.parameters(), b.parameters()):
            assert torch.allclose(u.grad, v.grad, rtol=2.0**-18, atol=0.0)
    with pytest.raises(ValueError):
        policy_mpc.clip_grad_norm_(_net().parameters(), 1.0, norm_type="two")


class _On(torch.Tensor):
    """A CPU tensor that says it is on another device."""

    @staticmethod
    def of(t, index):
        x = t.detach().as_subclass(_On)
        x.index = index
        return x

    @property
    def device(self):
        return torch.device("cuda", getattr(self, "index", 0))

    def to(self, device):
        return _On.of(self.as_subclass(torch.Tensor).clone(), torch.device(device).index)


class _Param:
    def __init__(self, grad):
        self.grad = grad


def _spread(seed=5):
    """Gradients on three devices in turn, one on its own, and parameters without any."""
    gen = torch.Generator().manual_seed(seed)
    at = [1, 0, 1, 2, 0, 1]
    grads = [_On.of(torch.randn(k + 1, generator=gen), d) for k, d in enumerate(at)]
    return [_Param(None), *map(_Param, grads), _Param(None)], grads, at


@pytest.mark.parametrize("p", [2.0, math.inf, "inf"])
@pytest.mark.parametrize("check", [False, True])
def test_parameters_on_several_devices(plain, monkeypatch, p, check):
    """Each device's gradients are one list, scaled by the norm of them all."""
    params, grads, at = _spread()
    flat = torch.cat([g.as_subclass(torch.Tensor).double() for g in grads])
    norm = float(flat.norm() if p == 2.0 else flat.abs().max())
    before = [g.as_subclass(torch.Tensor).clone() for g in grads]
    # totals lie on their list's device and are joined on the first gradient's
    given = []
    total, clip = plain.grad_norm_total, plain.clip_grad_norm

    def total_there(held, norm_type=2.0):
        assert len({g.device for g in held}) == 1
        return _On.of(total(held, norm_type), held[0].device.index)

    def clip_there(held, max_norm, norm_type=2.0, total=None, out=None):
        assert total.device == held[0].device
        given.append(float(total))
        return clip(held, max_norm, norm_type=norm_type, total=total.as_subclass(torch.Tensor), out=out)
    monkeypatch.setattr(policy_mpc._nat, "grad_norm_total", total_there)
    monkeypatch.setattr(policy_mpc._nat, "clip_grad_norm", clip_there)
    n = policy_mpc.clip_grad_norm_(params, 0.5, norm_type=p, error_if_nonfinite=check)
    assert math.isclose(float(n), norm, rel_tol=2.0**-23)
    assert len(given) == 3 and len(set(given)) == 1
    lists = [held for kind, held in plain.calls if kind == "clip"]
    for held, device in zip(lists, (1, 0, 2)):
        assert [id(g) for g in held] == [id(g) for g, d in zip(grads, at) if d == device]
    for g, b in zip(grads, before):
        assert torch.allclose(g.as_subclass(torch.Tensor), b * 0.5 / (norm + 1e-6), rtol=1e-6)


@pytest.mark.parametrize("p", [2.0, math.inf])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_norm_that_is_not_finite_is_reported_before_anything_is_written(plain, monkeypatch, p, bad):
    params, grads, _ = _spread()
    grads[3][1] = bad
    before = [g.as_subclass(torch.Tensor).clone() for g in grads]
    total = plain.grad_norm_total
    monkeypatch.setattr(policy_mpc._nat, "grad_norm_total",
                        lambda held, norm_type: _On.of(total(held, norm_type), held[0].device.index))
    with pytest.raises(RuntimeError, match="non-finite"):
        policy_mpc.clip_grad_norm_(params, 0.5, norm_type=p, error_if_nonfinite=True)
    assert all(torch.equal(g.as_subclass(torch.Tensor).nan_to_num(7.0), b.nan_to_num(7.0)) for g, b in zip(grads, before))
    assert not any(kind == "clip" for kind, _ in plain.calls)


def test_grad_mode_is_left_as_it_was(plain):
    for enabled in (True, False):
        with torch.set_grad_enabled(enabled):
            w = torch.nn.Parameter(torch.ones(3))
            w.grad = torch.ones(3)
            policy_mpc.clip_grad_norm_([w], 1.0)
            assert torch.is_grad_enabled() == enabled
            with pytest.raises(ValueError):
                policy_mpc.clip_grad_norm_([], 1.0, norm_type="two")
            assert torch.is_grad_enabled() == enabled
